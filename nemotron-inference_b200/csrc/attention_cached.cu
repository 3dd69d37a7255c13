// Attention over the 8-bit cache for up to 16 rows of queries to a key head; what there is to both kernels is in
// attention_cached.cuh.
//
// A thread per token: with R rows and tiles of 128 tokens
//   S^T = K [a | b]^T   M = 128 tokens, N = 2R, K = 128: both terms of the queries, both operands in shared memory
//   softmax             a thread has its token's scores of all rows; the terms are added up with b's sixteen fold
//   O^T += V^T [a | b]  M = 128 dimensions, N = 2R, K = 128 tokens: the values' tile is read along its rows
// Rows being few, all 128 threads have work and the tensor cores run far below what they can do, while the memory
// is read at its rate.  Two blocks to an SM, a tile's chain of some 1500 cycles in one beside the other's.
//
// Measured, 32 heads on 8 key heads, pages of 64: 64 sequences of 2048 tokens on average 56 us (268 MB: 4.8 TB/s, 0.73
// of the copy rate; some 11 us of it before the first tiles arrive and after the last), one of 65536 tokens 34 us
// (134 MB).  One of 1500 tokens on 2 key heads 10.9 us: launch, the chain sequence - length - page - tile, and the
// join of 12 pieces.
#include <algorithm>

#include "attention_cached.cuh"

namespace nmoe {
namespace {

template <int R>
struct Shape {
  static constexpr int kRows = R;
  static constexpr int kWidth = 2 * R;  // columns of S and O, bytes of a token's weights
  static constexpr int kBlocks = 2;     // on an SM
  // What a (sequence, key head, rows) costs a block beside its tiles, in tiles: its queries, and its results on their way
  // out.  Counted where tiles are shared, or blocks that meet many come last by 20 %.
  static constexpr int kUnitCost = 1;
  static constexpr int kKeySlots = 3, kValueSlots = 3;  // tiles in flight
  static constexpr int kSoftmaxWarps = 4;
  static constexpr int kBatch = R / kSoftmaxWarps;  // rows of queries to a warp
  static constexpr int kThreads = 32 * (kSoftmaxWarps + 2);
  static constexpr int kValueReaders = 1, kSegmentReaders = kSoftmaxWarps + 1, kQueryWriters = kSoftmaxWarps;
  static constexpr int kColumns = 3 * kWidth <= 64 ? 64 : 128;  // two buffers of S, and O
  static constexpr uint32_t kQueryBytes = 2 * R * kHeadDim, kWeightBytes = 2 * R * kKeyTile;
};

template <typename S>
struct Control : WorkControl<S> {
  uint64_t s_full[2], s_empty[2], p_full, p_empty;
  alignas(16) float shift[S::kRows];                 // kWeightBits - the reference
  alignas(16) float rise[S::kRows], fade[S::kRows];  // of a reference, and what that leaves of its sums
  int highest[S::kRows];                             // largest exponents of a tile, as ordered()
  uint32_t risen;                                    // the rows whose references have changed
  uint32_t anew;                                     // those that begin anew
  float warp_sum[S::kSoftmaxWarps][S::kRows];
  float sum[S::kRows], inverse[S::kRows];
  int failed;
};

template <typename S>
constexpr size_t shared_bytes() {
  return 1024 + (S::kKeySlots + S::kValueSlots) * kKeyTileBytes + S::kQueryBytes + S::kWeightBytes + sizeof(Control<S>);
}

// The blocks fit beside each other.
template <typename S>
constexpr bool fits_on_sm() {
  return S::kBlocks * (shared_bytes<S>() + 1024) <= 228 * 1024 && S::kBlocks * S::kColumns <= 512;
}

// Sums N values over the warp: lane L holds in v[0..] the totals of the rows sum_row<N>(L, 0..).  Half of
// the values change hands in each step.
template <int N>
__device__ __forceinline__ void warp_sums(float (&v)[N], int lane) {
  int count = N;
#pragma unroll
  for (int stride = 16; stride > 0; stride /= 2) {
    if (count > 1) {
      count /= 2;
      const bool upper = (lane & stride) != 0;
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        if (i < count) {
          const float send = upper ? v[i] : v[i + count], keep = upper ? v[i + count] : v[i];
          v[i] = keep + __shfl_xor_sync(0xffffffffu, send, stride);
        }
      }
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], stride);
    }
  }
}
template <int N>
__device__ __forceinline__ int sum_row(int lane, int i) {
  int row = 0, count = N;
#pragma unroll
  for (int stride = 16; stride > 0; stride /= 2) {
    if (count > 1) {
      count /= 2;
      if (lane & stride) row += count;
    }
  }
  return row + i;
}

template <typename S>
__device__ bool mma_role(uint32_t keys_at, uint32_t values_at, uint32_t q_at, uint32_t weights_at, uint32_t tmem, Control<S>* c) {
  constexpr uint32_t kScoresDesc = make_idesc_e4m3(S::kWidth, false, false), kValuesDesc = make_idesc_e4m3(S::kWidth, true, true);
  // a token's weights are 16 or 32 bytes, swizzled in as many
  const uint64_t q_desc = make_smem_desc(q_at, 16, 1024, 2);
  const uint64_t p_desc = S::kWidth == 16 ? make_smem_desc(weights_at, 128, 128, 0) : make_smem_desc(weights_at, 16, 8 * S::kWidth, 6);
  const uint32_t o = tmem + 2 * S::kWidth;
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
    // scores are a tile ahead of the values
#pragma unroll 1
    for (int j = 0; j <= tiles; ++j) {
      if (j < tiles) {
        const uint32_t no = first_no + j, slot = no % S::kKeySlots, buffer = no & 1;
        if (!mbar_wait_warp(smem_u32(&c->k_full[slot]), (no / S::kKeySlots) & 1)) return false;
        if (!mbar_wait_warp(smem_u32(&c->s_empty[buffer]), ((no >> 1) & 1) ^ 1)) return false;
        tcgen05_fence_after();
        if (elect_one()) {
          const uint64_t k_desc = make_smem_desc(keys_at + slot * kKeyTileBytes, 16, 1024, 2);
#pragma unroll
          for (int k = 0; k < kHeadDim / 32; ++k) {
            mma_e4m3(tmem + buffer * S::kWidth, advance_smem_desc(k_desc, k * 32), advance_smem_desc(q_desc, k * 32), kScoresDesc, k > 0);
          }
          tcgen05_commit(&c->s_full[buffer]);
          tcgen05_commit(&c->k_empty[slot]);
        }
        __syncwarp();
      }
      if (j > 0) {
        const uint32_t no = first_no + j - 1, slot = no % S::kValueSlots;
        if (!mbar_wait_warp(smem_u32(&c->v_full[slot]), (no / S::kValueSlots) & 1)) return false;
        if (!mbar_wait_warp(smem_u32(&c->p_full), no & 1)) return false;
        tcgen05_fence_after();
        if (elect_one()) {
          // (eight tokens are 1024 bytes of values)
          const uint64_t v_desc = make_smem_desc(values_at + slot * kKeyTileBytes, 16, 1024, 2);
#pragma unroll
          for (int k = 0; k < kKeyTile / 32; ++k) {
            mma_e4m3(o, advance_smem_desc(v_desc, k * 4096), advance_smem_desc(p_desc, k * 32 * S::kWidth), kValuesDesc, j > 1 || k > 0);
          }
          tcgen05_commit(&c->p_empty);
          tcgen05_commit(&c->v_empty[slot]);
        }
        __syncwarp();
      }
    }
    first_no += tiles;
  }
}

// Where byte `column` (a multiple of 8) of a token's weights lies.
template <typename S>
__device__ __forceinline__ uint32_t weight_offset(int token, int column) {
  const uint32_t at = token * S::kWidth + column;
  constexpr uint32_t mask = (S::kWidth / 16 - 1) << 4;
  return at ^ ((at >> 3) & mask);
}

template <typename S, Part P>
__device__ bool softmax_role(const CachedArgs& args, const Split& split, uint8_t* values, uint8_t* q, uint8_t* weights,
                             uint32_t tmem, Control<S>* c) {
  constexpr int R = S::kRows;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int token = threadIdx.x;
  const uint32_t lanes = tmem + (static_cast<uint32_t>(warp & 3) << 21);
  const uint32_t s_at = lanes, o_at = lanes + 2 * S::kWidth;
  const int page_shift = args.cache.page_shift;
  const uint64_t* shifts = reinterpret_cast<const uint64_t*>(c->shift);
  const uint64_t* rises = reinterpret_cast<const uint64_t*>(c->rise);
  const uint64_t* fades = reinterpret_cast<const uint64_t*>(c->fade);
  volatile int* failed = &c->failed;
  int joins = 0;
  uint32_t no = 0;  // tiles so far
  bool ok = mbar_wait_warp(smem_u32(&c->segment_full[0]), 0);
  int some = ok && c->has_segment[0];
  uint2 queries[S::kBatch];
  c->first_bad[token] = INT32_MAX;
  if (some) {
    load_queries<S>(args, c->segment[0], 0, queries);
    prepare_queries<S, 16>(args, c->segment[0], 0, queries, q, c);
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&c->q_full);
  }
#pragma unroll 1
  for (uint32_t segments = 0;; ++segments) {
    const Segment& s = c->segment[segments % kSegments];
    const uint32_t following = segments + 1;
    const uint64_t* factors = reinterpret_cast<const uint64_t*>(c->factor[segments & 1]);
    const int* limits = c->limit[segments & 1];
    if (!ok) *failed = 1;
    if (token < R) {
      c->shift[token] = 0.0f;
      c->highest[token] = kLowest;
    }
    softmax_sync<S>();
    if (*failed) return false;
    if (!some) break;
    uint64_t sum[R / 2];
#pragma unroll
    for (int r = 0; r < R / 2; ++r) sum[r] = 0;
    const int clear = P == Part::kShared ? s.length : s.length - s.rows;  // the last token that every row sees
#pragma unroll 1
    for (int j = 0; j < s.tiles; ++j, ++no) {
      const uint32_t slot = no % S::kValueSlots, buffer = no & 1;
      const int first = (s.tile + j) * kKeyTile, position = first + token;
      const bool at_end = first + kKeyTile - 1 > clear, is_first = j == 0;
      ok = mbar_wait_warp(smem_u32(&c->v_full[slot]), (no / S::kValueSlots) & 1);
      ok = mbar_wait_warp(smem_u32(&c->s_full[buffer]), (no >> 1) & 1) && ok;
      tcgen05_fence_after();
      // (places behind the sequence may lie in pages that it does not have)
      const int page = token >> page_shift;
      const float k_scale = exp2_approx(static_cast<float>(position < s.length ? c->powers[slot][0][page] : 0));
      const float v_power = static_cast<float>(position < s.length ? c->powers[slot][1][page] : 0);
      const uint64_t k2 = pack2(k_scale, k_scale), k2_16 = pack2(k_scale * 0.0625f, k_scale * 0.0625f);
      const uint64_t v2 = pack2(v_power, v_power);
      const float v_inverse = exp2_approx(-v_power);
      const uint64_t v2_inverse = pack2(v_inverse, v_inverse);
      if (j + 1 == s.tiles) {  // the next segment's queries are on their way meanwhile
        const bool known = mbar_wait_warp(smem_u32(&c->segment_full[following % kSegments]), (following / kSegments) & 1);
        some = known && c->has_segment[following % kSegments];
        if (some) load_queries<S>(args, c->segment[following % kSegments], 0, queries);
        ok = ok && known;
      }
      if (at_end) clean_values<S>(values + slot * kKeyTileBytes, token, position, s, c);
      // exponents of the weights, rows in pairs: score + power of the values - reference + kWeightBits
      uint64_t y[R / 2];
      float high = -INFINITY;
      auto exponents = [&] {  // (the second terms are sixteen fold)
        uint32_t a[R], b[R];
#pragma unroll
        for (int i = 0; i < R; i += 8) {
          tmem_ld_x8_async(s_at + buffer * S::kWidth + i, a + i);
          tmem_ld_x8_async(s_at + buffer * S::kWidth + R + i, b + i);
        }
        tmem_ld_wait();
        registers_loaded<R>(a);
        registers_loaded<R>(b);
#pragma unroll
        for (int i = 0; i < R / 2; ++i) {
          const uint64_t product =
              fma2(pack2(__uint_as_float(b[2 * i]), __uint_as_float(b[2 * i + 1])), k2_16,
                   mul2(pack2(__uint_as_float(a[2 * i]), __uint_as_float(a[2 * i + 1])), k2));
          y[i] = fma2(product, factors[i], add2(shifts[i], v2));
        }
        if (at_end) {
#pragma unroll
          for (int r = 0; r < R; r += 2) {
            float y0, y1;
            unpack2(y[r / 2], y0, y1);
            if (position > limits[r]) y0 = -INFINITY;
            if (position > limits[r + 1]) y1 = -INFINITY;
            y[r / 2] = pack2(y0, y1);
          }
        }
      };
      exponents();
#pragma unroll
      for (int r = 0; r < R / 2; ++r) {
        float y0, y1;
        unpack2(y[r], y0, y1);
        high = fmaxf(high, fmaxf(y0, y1));
      }
      // the weights of the tile before have been read, and O holds it
      ok = mbar_wait_warp(smem_u32(&c->p_empty), (no & 1) ^ 1) && ok;
      tcgen05_fence_after();
      if (!ok) *failed = 1;
      const bool rise = softmax_any<S>(is_first || high > kLargestBits);
      if (*failed) return false;
      if (rise) {
        // the largest of each row that it may be, eight rows at a time
        auto find_highest = [&](bool all) {
#pragma unroll
          for (int i = 0; i < R; i += 8) {
            float z[8];
#pragma unroll
            for (int k = 0; k < 8; k += 2) unpack2(y[(i + k) / 2], z[k], z[k + 1]);
            const float of_eight = fmaxf(fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3])),
                                         fmaxf(fmaxf(z[4], z[5]), fmaxf(z[6], z[7])));
            if (!__any_sync(0xffffffffu, all || of_eight > kLargestBits)) continue;
            int mine = kLowest;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const int largest = __reduce_max_sync(0xffffffffu, ordered(z[k]));
              if (lane == k) mine = largest;
            }
            if (lane < 8 && (all || mine > ordered(kLargestBits))) atomicMax(&c->highest[i + lane], mine);
          }
          softmax_sync<S>();
        };
        find_highest(is_first);
        if (token < 32) {
          bool risen = false, far = false;
          if (token < R) {
            const int r = token;
            const float top = from_ordered(c->highest[r]);
            c->highest[r] = kLowest;
            risen = top > -INFINITY;
            far = !is_first && top > kFarBits;
            const float by = risen && !far ? top - kWeightBits : 0.0f;  // (in a first tile a reference may fall, too)
            c->rise[r] = -by;
            c->fade[r] = is_first ? 1.0f : far ? 0.0f : exp2_approx(-by);
            c->shift[r] = far ? 0.0f : is_first && top == -INFINITY ? -kNoReference : c->shift[r] - by;
          }
          const uint32_t rows = __ballot_sync(0xffffffffu, risen), rows_anew = __ballot_sync(0xffffffffu, far);
          if (lane == 0) {
            c->risen = rows;
            c->anew = rows_anew;
          }
        }
        softmax_sync<S>();
#pragma unroll
        for (int r = 0; r < R / 2; ++r) {
          y[r] = add2(y[r], rises[r]);
          sum[r] = mul2(sum[r], fades[r]);
        }
        if (!is_first) {
#pragma unroll 1
          for (int i = 0; i < R; i += 8) {
            if ((c->risen >> i & 0xffu) == 0) continue;
            uint32_t o[16];
            tmem_ld_x8_async(o_at + i, o);
            tmem_ld_x8_async(o_at + R + i, o + 8);
            tmem_ld_wait();
            registers_loaded<16>(o);
#pragma unroll
            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * c->fade[i + (k & 7)]);
            tmem_st_x8(o_at + i, o);
            tmem_st_x8(o_at + R + i, o + 8);
          }
          tmem_st_wait();
          if (c->anew != 0) {  // (hardly ever) as in a first tile, for these rows
            exponents();
            find_highest(true);
            if (token < R) {
              const float top = from_ordered(c->highest[token]);
              c->highest[token] = kLowest;
              const float by = (c->anew >> token & 1) && top > -INFINITY ? top - kWeightBits : 0.0f;
              c->rise[token] = -by;
              c->shift[token] -= by;
            }
            softmax_sync<S>();
#pragma unroll
            for (int r = 0; r < R / 2; ++r) y[r] = add2(y[r], rises[r]);
          }
        }
      }
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&c->s_empty[buffer]);
#pragma unroll
      for (int i = 0; i < R; i += 8) {
        uint32_t a[2], b[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float w[4];
#pragma unroll
          for (int r = 0; r < 4; r += 2) {
            const int pair = i / 2 + 2 * k + r / 2;
            unpack2(y[pair], w[r], w[r + 1]);
            w[r] = exp2_approx(w[r]);
            w[r + 1] = exp2_approx(w[r + 1]);
            sum[pair] = fma2(pack2(w[r], w[r + 1]), v2_inverse, sum[pair]);
          }
          weight_codes(w, a[k], b[k]);
        }
        *reinterpret_cast<uint2*>(weights + weight_offset<S>(token, i)) = make_uint2(a[0], a[1]);
        *reinterpret_cast<uint2*>(weights + weight_offset<S>(token, R + i)) = make_uint2(b[0], b[1]);
      }
      fence_proxy_async_smem();
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&c->p_full);
    }
    if (some) {  // (all scores of this segment are done)
      prepare_queries<S, 16>(args, c->segment[following % kSegments], following & 1, queries, q, c);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&c->q_full);
    }
    // the rows' sums of weights over the 128 threads, in a fixed order
    float each[R];
#pragma unroll
    for (int r = 0; r < R; r += 2) unpack2(sum[r / 2], each[r], each[r + 1]);
    warp_sums<R>(each, lane);
    c->warp_sum[warp][sum_row<R>(lane, 0)] = each[0];
    ok = mbar_wait_warp(smem_u32(&c->p_empty), (no & 1) ^ 1);
    tcgen05_fence_after();
    if (!ok) *failed = 1;
    softmax_sync<S>();
    if (token < R) {
      float x = 0.0f;
#pragma unroll
      for (int w = 0; w < 4; ++w) x += c->warp_sum[w][token];
      c->sum[token] = x * kCodeScale;
      c->inverse[token] = 1.0f / (x * kCodeScale);
    }
    softmax_sync<S>();
    // a thread per dimension now
    const bool alone = s.part < 0;
    float* slot = split.slots + slot_floats(R) * max(s.part, 0);
    const int* out_rows = c->out_row[segments & 1];
    const int bad = c->first_bad[token];
    c->first_bad[token] = INT32_MAX;
#pragma unroll 1
    for (int i = 0; i < R && out_rows[i] >= 0; i += 8) {
      uint32_t a[16];
      tmem_ld_x8_async(o_at + i, a);
      tmem_ld_x8_async(o_at + R + i, a + 8);
      tmem_ld_wait();
      registers_loaded<16>(a);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int r = i + k, to = out_rows[r];
        float o = fmaf(__uint_as_float(a[k + 8]), 0.0625f, __uint_as_float(a[k]));
        if (limits[r] >= bad) o = NAN;
        if (to < 0) continue;
        if (P != Part::kAll && alone) {
          __stcg(args.sums + static_cast<size_t>(to) * kHeadDim + token, o);
        } else if (alone) {
          args.out[static_cast<size_t>(to) * kHeadDim + token] = __float2bfloat16(o * c->inverse[r]);
        } else {
          __stcg(slot + r * kHeadDim + token, o);
        }
      }
    }
    tcgen05_fence_before();
    if (P != Part::kAll && token < R) {
      leave_row_part(args, s, out_rows[token], token, c->sum[token] == 0.0f ? -INFINITY : -c->shift[token], c->sum[token]);
    }
    if (!alone) {
      if (token < R) {  // (a row that has seen no token, all being behind its mask, leaves nothing)
        __stcg(slot + R * kHeadDim + token, c->sum[token] == 0.0f ? -INFINITY : -c->shift[token]);
        __stcg(slot + R * (kHeadDim + 1) + token, c->sum[token]);
      }
      if (P == Part::kAll) {
        if (threadIdx.x == 0) c->to_join[joins] = s;
        ++joins;
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&c->segment_empty[segments % kSegments]);
  }
  if (P == Part::kAll) announce_and_join<S>(args, split, joins, c);
  return true;
}

template <typename S, Part P>
__global__ void __launch_bounds__(S::kThreads, S::kBlocks)
    cached_kernel(const __grid_constant__ CUtensorMap map, const CachedArgs args, const Split split) {
  static_assert(fits_on_sm<S>());
  extern __shared__ uint8_t raw[];
  uint8_t* keys = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  uint8_t* values = keys + S::kKeySlots * kKeyTileBytes;
  uint8_t* q = values + S::kValueSlots * kKeyTileBytes;
  uint8_t* weights = q + S::kQueryBytes;
  Control<S>* c = reinterpret_cast<Control<S>*>(weights + S::kWeightBytes);
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    init_work<S>(c);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&c->s_full[i], 1);
      mbar_init(&c->s_empty[i], 4);
    }
    mbar_init(&c->p_full, 4);
    mbar_init(&c->p_empty, 1);
    c->failed = 0;
    fence_barrier_init();
  }
  if (warp == S::kSoftmaxWarps) {
    tmem_alloc(&c->tmem, S::kColumns);
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
    if (!softmax_role<S, P>(args, split, values, q, weights, tmem, c) && (threadIdx.x & 31) == 0) {
      report_cache_error(args.cache.error, kDevWaitTimeout);
    }
  } else if (warp == S::kSoftmaxWarps) {
    const bool ok = mma_role<S>(smem_u32(keys), smem_u32(values), smem_u32(q), smem_u32(weights), tmem, c);
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
    tmem_dealloc(tmem, S::kColumns);
  }
  if (P == Part::kOwn) wait_for_predecessor();
}

template <typename S, Part P>
cudaError_t launch(const CUtensorMap& map, const CachedArgs& args, const Split& split, int sms, cudaStream_t stream) {
  static std::atomic<uint64_t> allowed{0};
  cudaError_t err = allow_shared_memory_once(cached_kernel<S, P>, allowed);
  if (err != cudaSuccess) return err;
  return launch_kernel(cached_kernel<S, P>, dim3(sms * S::kBlocks), S::kThreads, shared_bytes<S>(),
                       LaunchStream(stream, true), map, args, split);
}

template <typename S>
cudaError_t launch(const CUtensorMap& map, const CachedArgs& args, Part part, const Split& split, int sms, cudaStream_t stream) {
  return part == Part::kAll      ? launch<S, Part::kAll>(map, args, split, sms, stream)
         : part == Part::kShared ? launch<S, Part::kShared>(map, args, split, sms, stream)
                                 : launch<S, Part::kOwn>(map, args, split, sms, stream);
}

}  // namespace

size_t attention_cached_slot_bytes() {
  // (two blocks of 16 rows need less than one of 128)
  return sizeof(float) * slot_floats(kMaxRows) * kSlotsPerBlock * device_sms();
}

size_t attention_cached_workspace_bytes() { return kAttendCounterBytes + attention_cached_slot_bytes(); }

int attention_cached_slot_rows(int64_t rows) { return rows <= 8 ? 8 : rows <= 16 ? 16 : kMaxRows; }

cudaError_t launch_attention_cached(const CachedArgs& args, cudaStream_t stream) {
  // By the query rows that the entries have on average.  Entries with more are taken 8, 16 or 128 at a time
  // and read their keys and values again each time.  64 sequences of 2048 tokens, 8 key heads, cold, in us, by 8 / 16 /
  // 128 at a time: 8 rows 72 / 74 / 113, 12 rows 110 / 76 / 113, 16 rows 109 / 76 / 115, 24 rows 149 / 113 / 117, 32 rows
  // 191 / 113 / 117, 48 rows 270 / 152 / 125.  One of 65536: 16 rows 57 / 45 / 61, 24 rows 66 / 57 / 64, 48 rows
  // 119 / 72 / 68.  So 17 to 32 rows give away some 4 %, and so does a batch most of whose entries have no rows: 4 of 8
  // rows x 16 heads among 64 places, 8192 tokens each, are taken 8 at a time, 43 us where 128 at a time take 33.
  const int64_t rows = (args.batch.rows + args.batch.count - 1) / args.batch.count *
                       static_cast<int64_t>(args.heads / args.cache.kv_heads);
  return launch_cached_part(args, Part::kAll, rows, reinterpret_cast<float*>(args.cache.attend_workspace + kAttendCounterBytes),
                            stream);
}

cudaError_t launch_cached_part(const CachedArgs& args, Part part, int64_t rows, float* slots, cudaStream_t stream) {
  const int sms = device_sms();
  if (sms * 2 > kMaxBlocks) return cudaErrorInvalidValue;
  CUtensorMap map;
  if (!pages_tensor_map(args.cache, &map)) return cudaErrorInvalidValue;
  const Split split{reinterpret_cast<JoinCounters*>(args.cache.attend_workspace), slots};
  switch (attention_cached_slot_rows(rows)) {
    case 8: return launch<Shape<8>>(map, args, part, split, sms, stream);
    case 16: return launch<Shape<16>>(map, args, part, split, sms, stream);
    default: return launch_cached_rows(map, args, part, split, sms, stream);
  }
}

}  // namespace nmoe
