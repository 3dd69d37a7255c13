// Attention over the 8-bit cache for up to 128 rows of queries to a key head (drafted tokens, chunks of prompts);
// what there is to both kernels is in attention_cached.cuh.
//
// A thread per row, four for its quarters of a tile of 128 tokens:
//   S = a K^T + b K^T   M = 128 rows, N = 128 tokens, K = 128, twice: the queries' terms from shared memory, into
//                       one sum, so b is not scaled up: its codes are 2^-9 apart and the row's largest element is
//                       between 2^7 and 2^8, which leaves 2^-17 of that in each element.  A score is off by
//                       scale 2^-17 max|q| sum|k| at worst
//   softmax             a row's scores, reference and sum are in registers of the four threads
//   O_a += a V, O_b += b V   M = 128 rows, N = 128 dimensions, K = 128 tokens: weights from TMEM, written over the
//                       scores; the values' tile is read along its rows
// A tile takes some 1000 MMA cycles and, by the softmax warps, some 800 issue slots of each scheduler, beside the
// 1400 cycles that the memory takes to bring one to an SM.  Scores are a tile ahead of the values.
//
// Measured, 48 sequences of 8192 tokens on average with up to 8 new rows each, 16 heads on each of 2 key heads: 104 us
// (201 MB: 1.9 TB/s).  A tile takes some 2900 cycles: the warps go through a tile's steps together (scores and
// maximum 600 cycles, exponentials and codes 1400, barriers between), so the special function unit and the issue slots
// are idle in turn.  With 8 softmax warps 119 us where 16 took 114; four pipelines of 128 rows and instructions for the
// conversions to codes, 162 where this form took 128.
#include "attention_cached.cuh"

namespace nmoe {
namespace {

struct Rows {
  static constexpr int kRows = kMaxRows;
  static constexpr int kKeySlots = 5, kValueSlots = 5;  // tiles in flight
  static constexpr int kSoftmaxWarps = 16;              // each four have a quarter of the tokens
  static constexpr int kBatch = 2;                      // rows of queries to a warp at a time
  // What a (sequence, key head, rows) costs a block beside its tiles, in tiles: its queries, and its results on their way
  // out.  Counted where tiles are shared.  (1: 101.5 us, 2: 100.3, 3: 100.0, 4: 99.6, 48 sequences of 8192 tokens)
  static constexpr int kUnitCost = 4;
  static constexpr int kThreads = 32 * (kSoftmaxWarps + 2);
  static constexpr int kValueReaders = 1, kSegmentReaders = kSoftmaxWarps + 1, kQueryWriters = kSoftmaxWarps;
  static constexpr uint32_t kQueryBytes = 2 * kRows * kHeadDim;
};
using S = Rows;

constexpr int kQuarter = kKeyTile / 4;
constexpr uint32_t kTermBytes = S::kRows * kHeadDim;  // of the queries
constexpr int kPart = 16;  // tokens that never lie in two pages
constexpr int kColumns = 512, kSums = 2 * kKeyTile;  // two buffers of S; then O_a, O_b

struct Control : WorkControl<S> {
  uint64_t s_full[2], p_full, o_full;
  float top[4][S::kRows], sum[4][S::kRows];  // by quarter
  int failed;
};

constexpr size_t kSharedBytes = 1024 + (S::kKeySlots + S::kValueSlots) * kKeyTileBytes + S::kQueryBytes + sizeof(Control);
static_assert(kSharedBytes <= kMaxSharedBytes);

__device__ bool mma_role(uint32_t keys_at, uint32_t values_at, uint32_t q_at, uint32_t tmem, Control* c) {
  constexpr uint32_t kScoresDesc = make_idesc_e4m3(kKeyTile, false, false), kValuesDesc = make_idesc_e4m3(kHeadDim, false, true);
  const uint64_t q_desc = make_smem_desc(q_at, 16, 1024, 2);
  uint32_t first_no = 0;  // of the segment's tiles among all
#pragma unroll 1
  for (uint32_t segments = 0;; ++segments) {
    const uint32_t place = segments % kSegments;
    if (!mbar_wait_warp(smem_u32(&c->segment_full[place]), (segments / kSegments) & 1)) return false;
    const int some = c->has_segment[place], tiles = warp_uniform(c->segment[place].tiles);
    __syncwarp();
    if (!some) return true;
    if (elect_one()) mbar_arrive(&c->segment_empty[place]);
    __syncwarp();
    if (!mbar_wait_warp(smem_u32(&c->q_full), segments & 1)) return false;
    tcgen05_fence_after();
#pragma unroll 1
    for (int j = 0; j <= tiles; ++j) {
      if (j < tiles) {  // (the weights that lay here have been multiplied, in order)
        const uint32_t no = first_no + j, slot = no % S::kKeySlots, buffer = no & 1;
        if (!mbar_wait_warp(smem_u32(&c->k_full[slot]), (no / S::kKeySlots) & 1)) return false;
        tcgen05_fence_after();
        if (elect_one()) {
          const uint64_t k_desc = make_smem_desc(keys_at + slot * kKeyTileBytes, 16, 1024, 2);
#pragma unroll
          for (int k = 0; k < 2 * kHeadDim / 32; ++k) {
            mma_e4m3(tmem + buffer * kKeyTile, advance_smem_desc(q_desc, k / 4 * kTermBytes + k % 4 * 32),
                     advance_smem_desc(k_desc, k % 4 * 32), kScoresDesc, k > 0);
          }
          tcgen05_commit(&c->s_full[buffer]);
          tcgen05_commit(&c->k_empty[slot]);
        }
        __syncwarp();
      }
      if (j > 0) {
        const uint32_t no = first_no + j - 1, slot = no % S::kValueSlots, buffer = no & 1;
        if (!mbar_wait_warp(smem_u32(&c->v_full[slot]), (no / S::kValueSlots) & 1)) return false;
        if (!mbar_wait_warp(smem_u32(&c->p_full), no & 1)) return false;
        tcgen05_fence_after();
        if (elect_one()) {
          // (eight tokens are 1024 bytes of values)
          const uint64_t v_desc = make_smem_desc(values_at + slot * kKeyTileBytes, 16, 1024, 2);
#pragma unroll
          for (int k = 0; k < 2 * kKeyTile / 32; ++k) {
            mma_e4m3_ts(tmem + kSums + k / 4 * kHeadDim, tmem + buffer * kKeyTile + k * 8,
                        advance_smem_desc(v_desc, k % 4 * 4096), kValuesDesc, j > 1 || k % 4 > 0);
          }
          tcgen05_commit(&c->o_full);
          tcgen05_commit(&c->v_empty[slot]);
        }
        __syncwarp();
      }
    }
    first_no += tiles;
  }
}

template <Part P>
__device__ bool softmax_role(const CachedArgs& args, const Split& split, uint8_t* values, uint8_t* q, uint32_t tmem, Control* c) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quarter = warp >> 2;
  const int row = threadIdx.x & (S::kRows - 1);
  const uint32_t lanes = tmem + (static_cast<uint32_t>(warp & 3) << 21);
  const int page_shift = args.cache.page_shift;
  volatile int* failed = &c->failed;
  int joins = 0;
  uint32_t no = 0;  // tiles so far
  bool ok = mbar_wait_warp(smem_u32(&c->segment_full[0]), 0);
  int some = ok && c->has_segment[0];
  uint2 queries[S::kBatch];
  if (some) load_queries<S>(args, c->segment[0], 0, queries);
#pragma unroll 1
  for (uint32_t segments = 0;; ++segments) {
    const Segment& s = c->segment[segments % kSegments];
    if (!ok) *failed = 1;
    softmax_sync<S>();
    if (*failed) return false;
    if (!some) break;
    if (threadIdx.x < kHeadDim) c->first_bad[threadIdx.x] = INT32_MAX;
    if (threadIdx.x == 0) c->found_bad = 0;
    prepare_queries<S, 1>(args, s, 0, queries, q, c);
    fence_proxy_async_smem();
    softmax_sync<S>();
    if (lane == 0) mbar_arrive(&c->q_full);
    const bool has_rows = s.row0 + (row & ~31) < s.rows * (args.heads / args.cache.kv_heads);  // the warp
    const int clear = P == Part::kShared ? s.length : s.length - s.rows;  // the last token that every row sees
    float factor = 0.0f, shift = 0.0f, sum = 0.0f;
    int limit = -1;
    if (has_rows) {
      factor = c->factor[0][row];
      limit = c->limit[0][row];
    }
#pragma unroll 1
    for (int j = 0; j < s.tiles; ++j, ++no) {
      const uint32_t slot = no % S::kValueSlots, buffer = no & 1;
      const int first = (s.tile + j) * kKeyTile, begin = first + quarter * kQuarter;
      const bool at_end = first + kKeyTile - 1 > clear, is_first = j == 0;
      ok = mbar_wait_warp(smem_u32(&c->v_full[slot]), (no / S::kValueSlots) & 1);
      if (at_end && quarter == 0) clean_values<S>(values + slot * kKeyTileBytes, row, first + row, s, c);
      ok = mbar_wait_warp(smem_u32(&c->s_full[buffer]), (no >> 1) & 1) && ok;
      tcgen05_fence_after();
      // exponents of the weights, tokens in pairs: score + power of the values - reference + kWeightBits
      const uint32_t s_at = lanes + buffer * kKeyTile;
      uint32_t y[kQuarter];
      float v_inverse[kQuarter / kPart], high = -INFINITY;
      auto exponents = [&] {
#pragma unroll
        for (int i = 0; i < kQuarter; i += 32) tmem_ld_x32_async(s_at + quarter * kQuarter + i, y + i);
        tmem_ld_wait();
        registers_loaded<kQuarter>(y);
#pragma unroll
        for (int p = 0; p < kQuarter / kPart; ++p) {
          // (places behind the sequence may lie in pages that it does not have)
          const int page = (quarter * kQuarter + p * kPart) >> page_shift;
          const bool there = begin + p * kPart < s.length;
          const int k_power = there ? c->powers[slot][0][page] : 0, v_power = there ? c->powers[slot][1][page] : 0;
          v_inverse[p] = power_of_two(-v_power);
          const float scale = factor * power_of_two(k_power), bias = static_cast<float>(v_power) + shift;
          const uint64_t scale2 = pack2(scale, scale), bias2 = pack2(bias, bias);
#pragma unroll
          for (int i = p * kPart; i < (p + 1) * kPart; i += 2) {
            float y0, y1;
            unpack2(fma2(pack2(__uint_as_float(y[i]), __uint_as_float(y[i + 1])), scale2, bias2), y0, y1);
            y[i] = __float_as_uint(y0);
            y[i + 1] = __float_as_uint(y1);
          }
        }
        if (at_end) {
#pragma unroll
          for (int i = 0; i < kQuarter; ++i) {
            if (begin + i > limit) y[i] = 0xff800000u;
          }
        }
        high = -INFINITY;
#pragma unroll
        for (int i = 0; i < kQuarter; ++i) high = fmaxf(high, __uint_as_float(y[i]));
      };
      if (has_rows) exponents();
      // (all scores are read behind this: weights may be written over them)
      if (!ok) *failed = 1;
      const bool rise = softmax_any<S>(is_first || high > kLargestBits);
      if (*failed) return false;
      if (rise) {
        c->top[quarter][row] = high;
        softmax_sync<S>();
        float top = fmaxf(fmaxf(c->top[0][row], c->top[1][row]), fmaxf(c->top[2][row], c->top[3][row]));
        const bool anew = has_rows && !is_first && top > kFarBits;
        if (!is_first && softmax_any<S>(anew)) {  // (hardly ever)
          if (anew) shift = 0.0f;
          if (has_rows) exponents();
          c->top[quarter][row] = high;
          softmax_sync<S>();
          top = fmaxf(fmaxf(c->top[0][row], c->top[1][row]), fmaxf(c->top[2][row], c->top[3][row]));
        }
        // a row's first tile sets its reference (unless it sees none of it), others may raise it
        const float by = has_rows && top > (is_first || anew ? -INFINITY : kLargestBits) ? top - kWeightBits : 0.0f;
        shift = is_first && top == -INFINITY ? -kNoReference : shift - by;
        if (__any_sync(0xffffffffu, by != 0.0f || anew)) {
#pragma unroll
          for (int i = 0; i < kQuarter; ++i) y[i] = __float_as_uint(__uint_as_float(y[i]) - by);
          if (!is_first) {
            const float fade = anew ? 0.0f : exp2_approx(-by);
            sum *= fade;
            // O of the tiles before is complete; each quarter takes half of one of its terms
            ok = mbar_wait_warp(smem_u32(&c->o_full), (no & 1) ^ 1);
            tcgen05_fence_after();
            if (!ok) *failed = 1;
            const uint32_t o_at = lanes + kSums + quarter * (kHeadDim / 2);
#pragma unroll 1
            for (int i = 0; i < kHeadDim / 2; i += 32) {
              uint32_t o[32];
              tmem_ld_x32_async(o_at + i, o);
              tmem_ld_wait();
              registers_loaded<32>(o);
#pragma unroll
              for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * fade);
              tmem_st_x32(o_at + i, o);
            }
          }
        }
        softmax_sync<S>();  // (top is read; O is scaled)
      }
      if (has_rows) {
        // four codes to a column: the first terms of the tile's 128 tokens, then the second terms
        uint32_t a[kQuarter / 4], b[kQuarter / 4];
#pragma unroll
        for (int p = 0; p < kQuarter / kPart; ++p) {
          uint64_t of_part = 0;
#pragma unroll
          for (int i = p * kPart; i < (p + 1) * kPart; i += 4) {
            float w[4];
            w[0] = exp2_approx(__uint_as_float(y[i]));
            w[1] = exp2_approx(__uint_as_float(y[i + 1]));
            if (i % 8 == 0) {
              unpack2(exp2_polynomial2<3>(pack2(__uint_as_float(y[i + 2]), __uint_as_float(y[i + 3]))), w[2], w[3]);
            } else {
              w[2] = exp2_approx(__uint_as_float(y[i + 2]));
              w[3] = exp2_approx(__uint_as_float(y[i + 3]));
            }
            of_part = add2(of_part, add2(pack2(w[0], w[1]), pack2(w[2], w[3])));
            weight_codes(w, a[i / 4], b[i / 4]);
          }
          float s0, s1;
          unpack2(of_part, s0, s1);
          sum = fmaf(s0 + s1, v_inverse[p], sum);
        }
        tmem_st_x8(s_at + quarter * (kQuarter / 4), a);
        tmem_st_x8(s_at + kKeyTile / 4 + quarter * (kQuarter / 4), b);
        tmem_st_wait();
      }
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&c->p_full);
    }
    // the next segment's queries are on their way during the end of this one
    const uint32_t following = segments + 1;
    const bool known = mbar_wait_warp(smem_u32(&c->segment_full[following % kSegments]), (following / kSegments) & 1);
    some = known && c->has_segment[following % kSegments];
    if (some) load_queries<S>(args, c->segment[following % kSegments], 0, queries);
    c->sum[quarter][row] = sum;
    ok = mbar_wait_warp(smem_u32(&c->o_full), (no & 1) ^ 1) && known;
    tcgen05_fence_after();
    if (!ok) *failed = 1;
    softmax_sync<S>();
    const bool alone = s.part < 0;
    if (has_rows) {
      const int to = c->out_row[0][row];
      const float all = ((c->sum[0][row] + c->sum[1][row]) + (c->sum[2][row] + c->sum[3][row])) * kCodeScale, inverse = 1.0f / all;
      const bool bad = c->found_bad != 0;
      float* slot = split.slots + slot_floats(S::kRows) * max(s.part, 0);
      // each quarter has 32 of the dimensions
#pragma unroll 1
      for (int d = quarter * 32; d < quarter * 32 + 32; d += 16) {
        uint32_t a[16], b[16];
        tmem_ld_x16_async(lanes + kSums + d, a);
        tmem_ld_x16_async(lanes + kSums + kHeadDim + d, b);
        tmem_ld_wait();
        registers_loaded<16>(a);
        registers_loaded<16>(b);
        float o[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          o[i] = fmaf(__uint_as_float(b[i]), 0.0625f, __uint_as_float(a[i]));
          if (bad && limit >= c->first_bad[d + i]) o[i] = NAN;
        }
        if (to < 0) continue;
        if (alone && P == Part::kAll) {
          uint32_t two[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) two[i] = pack_bf16(o[2 * i] * inverse, o[2 * i + 1] * inverse);
          uint4* out = reinterpret_cast<uint4*>(args.out + static_cast<size_t>(to) * kHeadDim + d);
          out[0] = make_uint4(two[0], two[1], two[2], two[3]);
          out[1] = make_uint4(two[4], two[5], two[6], two[7]);
        } else {
          float4* out = reinterpret_cast<float4*>((alone ? args.sums + static_cast<size_t>(to) * kHeadDim : slot + row * kHeadDim) + d);
#pragma unroll
          for (int i = 0; i < 4; ++i) __stcg(out + i, make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]));
        }
      }
      if (P != Part::kAll && quarter == 0) leave_row_part(args, s, to, row, all == 0.0f ? -INFINITY : -shift, all);
      if (!alone && quarter == 0) {  // (a row that has seen no token, all being behind its mask, leaves nothing)
        __stcg(slot + S::kRows * kHeadDim + row, all == 0.0f ? -INFINITY : -shift);
        __stcg(slot + S::kRows * (kHeadDim + 1) + row, all);
      }
    }
    tcgen05_fence_before();
    if (!alone && P == Part::kAll) {
      if (threadIdx.x == 0) c->to_join[joins] = s;
      ++joins;
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&c->segment_empty[segments % kSegments]);
  }
  if (P == Part::kAll) announce_and_join<S>(args, split, joins, c);
  return true;
}

template <Part P>
__global__ void __launch_bounds__(S::kThreads, 1)
    cached_rows_kernel(const __grid_constant__ CUtensorMap map, const CachedArgs args, const Split split) {
  extern __shared__ uint8_t raw[];
  uint8_t* keys = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  uint8_t* values = keys + S::kKeySlots * kKeyTileBytes;
  uint8_t* q = values + S::kValueSlots * kKeyTileBytes;
  Control* c = reinterpret_cast<Control*>(q + S::kQueryBytes);
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    init_work<S>(c);
    mbar_init(&c->s_full[0], 1);
    mbar_init(&c->s_full[1], 1);
    mbar_init(&c->p_full, S::kSoftmaxWarps);
    mbar_init(&c->o_full, 1);
    c->failed = 0;
    fence_barrier_init();
  }
  if (warp == S::kSoftmaxWarps) {
    tmem_alloc(&c->tmem, kColumns);
    tmem_relinquish();
  }
  tcgen05_fence_before();
  if (P != Part::kOwn) wait_for_predecessor();  // (kOwn: see launch_attention_shared())
  find_begin<S, P>(args, c);
  __syncthreads();
  release_successor();  // (the columns of TMEM are there)
  tcgen05_fence_after();
  const uint32_t tmem = c->tmem;
  if (warp < S::kSoftmaxWarps) {
    if (!softmax_role<P>(args, split, values, q, tmem, c) && (threadIdx.x & 31) == 0) {
      report_cache_error(args.cache.error, kDevWaitTimeout);
    }
  } else if (warp == S::kSoftmaxWarps) {
    const bool ok = mma_role(smem_u32(keys), smem_u32(values), smem_u32(q), tmem, c);
    if (elect_one()) {
      if (!ok) report_cache_error(args.cache.error, kDevWaitTimeout);
      tcgen05_commit(&c->drained);
    }
    __syncwarp();
    mbar_wait_warp(smem_u32(&c->drained), 0);
  } else {
    load_role<S, P>(args, &map, smem_u32(keys), smem_u32(values), c);
  }
  tcgen05_fence_before();
  __syncthreads();
  if (warp == S::kSoftmaxWarps) {
    tcgen05_fence_after();
    tmem_dealloc(tmem, kColumns);
  }
  if (P == Part::kOwn) wait_for_predecessor();
}

template <Part P>
cudaError_t launch(const CUtensorMap& map, const CachedArgs& args, const Split& split, int sms, cudaStream_t stream) {
  static std::atomic<uint64_t> allowed{0};
  cudaError_t err = allow_shared_memory_once(cached_rows_kernel<P>, allowed);
  if (err != cudaSuccess) return err;
  return launch_kernel(cached_rows_kernel<P>, dim3(sms), S::kThreads, kSharedBytes, LaunchStream(stream, true),
                       map, args, split);
}

}  // namespace

cudaError_t launch_cached_rows(const CUtensorMap& map, const CachedArgs& args, Part part, const Split& split, int sms, cudaStream_t stream) {
  return part == Part::kAll      ? launch<Part::kAll>(map, args, split, sms, stream)
         : part == Part::kShared ? launch<Part::kShared>(map, args, split, sms, stream)
                                 : launch<Part::kOwn>(map, args, split, sms, stream);
}

}  // namespace nmoe
