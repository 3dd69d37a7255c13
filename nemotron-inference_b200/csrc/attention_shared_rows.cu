// Attention of more than 128 rows of queries at once over tokens that all of them see (a prompt that many sequences
// continue): the first of the launches of attention_shared.cu, for large groups.
//
// A block works on two tiles of 128 rows of a key head, so that each tile of keys and values that it brings in serves
// both, and one tile's exponentials run while the tensor cores work on the other.  Per tile of 128 tokens and of rows:
//   S = a K^T + b K^T   M = 128 rows, N = 128 tokens, K = 128, twice: queries as two E4M3 terms, as in the kernel for
//                       up to 128 rows
//   softmax             two threads per row, a half of the tokens each: weights 2^(s - reference), as binary16 over the
//                       scores
//   O += P V            M = 128 rows, N = 128 dimensions, K = 128 tokens
// Values become binary16 on their way, exactly but for a factor of 2^-8: the seven bits behind a code's sign lie in both
// formats in the same order.  So a weight needs one term, is within 2^-11 of itself down to 2^-14 of the largest, and
// is made with half the instructions of two E4M3 terms; both ways take the tensor cores 512 cycles.  The softmax
// warps do it, each its share, while they wait for scores.  (Two warps of their own took 4700 cycles for a tile.)
//
// The queries' terms are made once, by a kernel ahead of this one, and copied in by TMA: 256 rows made by each block
// that needs them took 24000 cycles.
//
// What bounds it: the tensor cores, 2048 cycles for both tiles of rows.  Measured (B200): 3750 cycles, since the softmax
// warps' instructions (they issue in 46 % of the cycles) go with one tile's MMAs but for what two tiles' turns leave;
// 14000 cycles before a block's first products and 9000 for a unit's sums besides.  Eight groups of 16 sequences that
// share 16384 tokens, 4 rows each, 32 query and 2 key heads: 115 us; 64 that share
// 8192, 8 key heads, a row each: 26 us.
#include "attention_cached.cuh"

namespace nmoe {
namespace {

struct Pair {
  static constexpr int kTiles = 2;                      // of 128 rows
  static constexpr int kRows = kTiles * 128;
  static constexpr int kKeySlots = 3, kValueSlots = 2;  // tiles in flight
  static constexpr int kSoftmaxWarps = 16;
  static constexpr int kUnitCost = 2;  // what a (group, key head, rows) costs a block beside its tiles, in tiles
  static constexpr int kThreads = 32 * (kSoftmaxWarps + 2);
  static constexpr int kValueReaders = kSoftmaxWarps, kSegmentReaders = kSoftmaxWarps + 1, kQueryWriters = 1;
  static constexpr uint32_t kQueryBytes = 2 * kRows * kHeadDim;
};
using S = Pair;

constexpr int kMmaWarp = S::kSoftmaxWarps;  // the one behind it loads
constexpr int kWideSlots = 2;                       // tiles of binary16 values
constexpr uint32_t kWideBytes = 2 * kKeyTileBytes;  // two panels of 64 dimensions
constexpr uint32_t kTermBytes = S::kRows * kHeadDim, kTileRowsBytes = 128 * kHeadDim;
constexpr int kColumns = 512, kSums = 2 * kKeyTile;  // S of both tiles, O of both tiles
constexpr int kPart = 16;                            // tokens that never lie in two pages
constexpr int kHalf = kKeyTile / 2;                  // tokens of a thread
constexpr float kRiseBits = 8.0f;                    // binary orders by which a maximum may outgrow its reference
constexpr float kSumScale = kCodeScale;              // of what is left, as the other kernels leave it
constexpr float kValueScale = 256.0f * kSumScale;    // and of the products with values

struct Control : WorkControl<S> {
  // q_empty: by the MMA warp, whose products have read the queries, and by the softmax warps, which have seen q_full (they
  // may still leave a segment's sums when the next one, of a single tile, has its products with its queries)
  uint64_t s_full[2], p_full[2], o_full[2], o_empty[2], q_empty, wide_full[kWideSlots], wide_empty[kWideSlots];
  float top[2][S::kRows], other_sum[S::kRows];  // by halves of the tokens
  int failed[2];                                // a wait of a tile's warps has run out
};

constexpr size_t kSharedBytes =
    1024 + (S::kKeySlots + S::kValueSlots) * kKeyTileBytes + kWideSlots * kWideBytes + S::kQueryBytes + sizeof(Control);
static_assert(kSharedBytes <= kMaxSharedBytes);

// The queries' terms, [2][kv_heads][rows x heads that share a key head][128], and what the rows' products of codes are
// multiplied by.
struct Queries {
  uint8_t* codes;
  float* factors;
};

constexpr int kPrepareThreads = 256;

// A warp to a row.
__global__ void __launch_bounds__(kPrepareThreads) prepare_kernel(const CachedArgs args, const Queries queries) {
  wait_for_predecessor();
  release_successor();
  const int lane = threadIdx.x & 31, group = args.heads / args.cache.kv_heads;
  const int64_t pair = (static_cast<int64_t>(blockIdx.x) * kPrepareThreads + threadIdx.x) >> 5;
  const int64_t pairs = static_cast<int64_t>(args.batch.rows) * args.heads;
  if (pair >= pairs) return;
  const int row = static_cast<int>(pair / args.heads), head = static_cast<int>(pair % args.heads);
  const uint2 raw = *reinterpret_cast<const uint2*>(args.q + row * args.q_stride + head * kHeadDim + lane * 4);
  uint32_t a, b;
  float factor;
  query_terms<1>(raw, args.scale, a, b, factor);
  const int64_t of_head = static_cast<int64_t>(args.batch.rows) * group;
  const int64_t at = head / group * of_head + static_cast<int64_t>(row) * group + head % group;
  const int64_t terms = args.cache.kv_heads * of_head;
  *reinterpret_cast<uint32_t*>(queries.codes + at * kHeadDim + lane * 4) = a;
  *reinterpret_cast<uint32_t*>(queries.codes + (terms + at) * kHeadDim + lane * 4) = b;
  if (lane == 0) queries.factors[at] = factor;
}

// (what is no number does not count)
__device__ __forceinline__ float largest_of(float a, float b, float c) {
  float x;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(x) : "f"(a), "f"(b), "f"(c));
  return x;
}

// Eight warps of a tile of rows.
__device__ __forceinline__ bool tile_any(int t, bool mine) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.or.pred q, %2, 256, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(any)
      : "r"(static_cast<uint32_t>(mine)), "r"(1 + t)
      : "memory");
  return any != 0;
}
__device__ __forceinline__ void tile_sync(int t) { asm volatile("bar.sync %0, 256;" ::"r"(1 + t) : "memory"); }

// kind::f16 on binary16 operands, FP32 sums, M = 128, B in rows of consecutive n.
constexpr uint32_t kValuesDesc = (1u << 4) | (1u << 16) | ((kHeadDim >> 3) << 17) | ((128u >> 4) << 24);

// Rows that a segment has of tile t.
__device__ __forceinline__ int rows_of(const CachedArgs& args, const Segment& s, int t) {
  return s.rows * (args.heads / args.cache.kv_heads) - s.row0 - t * 128;
}

__device__ bool mma_role(const CachedArgs& args, uint32_t keys_at, uint32_t wide_at, uint32_t q_at, uint32_t tmem, Control* c) {
  constexpr uint32_t kScoresDesc = make_idesc_e4m3(kKeyTile, false, false);
  const uint64_t q_desc = make_smem_desc(q_at, 16, 1024, 2);
  uint32_t no = 0;               // tiles so far
  uint32_t p_uses[2] = {0, 0}, o_uses[2] = {0, 0};
  auto scores = [&](int t, uint32_t slot) {
    if (elect_one()) {
      const uint64_t k_desc = make_smem_desc(keys_at + slot * kKeyTileBytes, 16, 1024, 2);
#pragma unroll
      for (int k = 0; k < 2 * kHeadDim / 32; ++k) {
        mma_e4m3(tmem + t * kKeyTile, advance_smem_desc(q_desc, k / 4 * kTermBytes + t * kTileRowsBytes + k % 4 * 32),
                 advance_smem_desc(k_desc, k % 4 * 32), kScoresDesc, k > 0);
      }
      tcgen05_commit(&c->s_full[t]);
    }
    __syncwarp();
  };
  auto release = [&](uint64_t* bar) {
    if (elect_one()) tcgen05_commit(bar);
    __syncwarp();
  };
#pragma unroll 1
  for (uint32_t segments = 0;; ++segments) {
    const uint32_t place = segments % kSegments;
    if (!mbar_wait_warp(smem_u32(&c->segment_full[place]), (segments / kSegments) & 1)) return false;
    const int some = c->has_segment[place], tiles = warp_uniform(c->segment[place].tiles);
    const int both = warp_uniform(some ? static_cast<int>(rows_of(args, c->segment[place], 1) > 0) : 0);
    __syncwarp();
    if (!some) return true;
    if (elect_one()) mbar_arrive(&c->segment_empty[place]);
    __syncwarp();
    if (!mbar_wait_warp(smem_u32(&c->q_full), segments & 1)) return false;
    if (!mbar_wait_warp(smem_u32(&c->k_full[no % S::kKeySlots]), (no / S::kKeySlots) & 1)) return false;
    tcgen05_fence_after();
    for (int t = 0; t <= both; ++t) scores(t, no % S::kKeySlots);
    release(&c->k_empty[no % S::kKeySlots]);
    if (tiles == 1) release(&c->q_empty);
#pragma unroll 1
    for (int j = 0; j < tiles; ++j) {
      const uint32_t wide = (no + j) % kWideSlots, next = no + j + 1;
      const bool more = j + 1 < tiles;
      if (!mbar_wait_warp(smem_u32(&c->wide_full[wide]), ((no + j) / kWideSlots) & 1)) return false;
      if (more && !mbar_wait_warp(smem_u32(&c->k_full[next % S::kKeySlots]), (next / S::kKeySlots) & 1)) return false;
#pragma unroll 1
      for (int t = 0; t <= both; ++t) {
        if (!mbar_wait_warp(smem_u32(&c->p_full[t]), p_uses[t] & 1)) return false;
        ++p_uses[t];
        if (j == 0) {
          if (!mbar_wait_warp(smem_u32(&c->o_empty[t]), (o_uses[t] & 1) ^ 1)) return false;
          ++o_uses[t];
        }
        tcgen05_fence_after();
        if (elect_one()) {
          // (eight tokens are 1024 bytes of a panel)
          const uint64_t v_desc = make_smem_desc(wide_at + wide * kWideBytes, kKeyTileBytes, 1024, 2);
#pragma unroll
          for (int k = 0; k < kKeyTile / 16; ++k) {
            mma_f16_ts(tmem + kSums + t * kHeadDim, tmem + t * kKeyTile + k * 8, advance_smem_desc(v_desc, k * 2048), kValuesDesc,
                       j > 0 || k > 0);
          }
          if (!more) tcgen05_commit(&c->o_full[t]);
        }
        __syncwarp();
        if (more) scores(t, next % S::kKeySlots);
      }
      release(&c->wide_empty[wide]);
      if (more) release(&c->k_empty[next % S::kKeySlots]);
      if (j + 2 == tiles) release(&c->q_empty);
    }
    no += tiles;
  }
}

// Two codes of the low half of `x`, of 2^-8 their value as binary16.
__device__ __forceinline__ uint32_t widen(uint32_t x, uint32_t selector) {
  const uint32_t high = __byte_perm(x, 0, selector);  // a code in each half's upper byte
  return (high & 0x80008000u) | ((high & 0x7f007f00u) >> 1);
}

// 0x3f80 is what becomes of a code that is no number.
__device__ __forceinline__ uint32_t no_numbers(uint32_t two) {
  if ((two & 0x7fffu) == 0x3f80u) two |= 0x7fffu;
  if ((two & 0x7fff0000u) == 0x3f800000u) two |= 0x7fff0000u;
  return two;
}

// A thread's share of a tile of values, as binary16: sixteen codes at a time, eight threads to a token.
__device__ __forceinline__ void widen_values(const uint8_t* values, uint8_t* wide) {
  const int chunk = threadIdx.x & 7;
  uint8_t* panel = wide + (chunk >> 2) * kKeyTileBytes;
  constexpr int kTokens = 32 * S::kSoftmaxWarps / 8;
#pragma unroll
  for (int i = 0; i < kKeyTile / kTokens; ++i) {
    const int token = (threadIdx.x >> 3) + i * kTokens;
    const uint4 x = *reinterpret_cast<const uint4*>(values + token * kHeadDim + ((chunk ^ (token & 7)) << 4));
    uint4 lo = make_uint4(widen(x.x, 0x1404), widen(x.x, 0x3424), widen(x.y, 0x1404), widen(x.y, 0x3424));
    uint4 hi = make_uint4(widen(x.z, 0x1404), widen(x.z, 0x3424), widen(x.w, 0x1404), widen(x.w, 0x3424));
    const uint32_t any = ((x.x & 0x7f7f7f7fu) + 0x01010101u) | ((x.y & 0x7f7f7f7fu) + 0x01010101u) |
                         ((x.z & 0x7f7f7f7fu) + 0x01010101u) | ((x.w & 0x7f7f7f7fu) + 0x01010101u);
    if (any & 0x80808080u) {  // (hardly ever) codes that are no numbers
      lo = make_uint4(no_numbers(lo.x), no_numbers(lo.y), no_numbers(lo.z), no_numbers(lo.w));
      hi = make_uint4(no_numbers(hi.x), no_numbers(hi.y), no_numbers(hi.z), no_numbers(hi.w));
    }
    // (the threads of the two panels in turn: together they meet every bank once)
    const int first = 2 * (chunk & 3), odd = chunk >> 2;
    *reinterpret_cast<uint4*>(panel + token * 128 + (((first + odd) ^ (token & 7)) << 4)) = odd ? hi : lo;
    *reinterpret_cast<uint4*>(panel + token * 128 + (((first + 1 - odd) ^ (token & 7)) << 4)) = odd ? lo : hi;
  }
  fence_proxy_async_smem();
  __syncwarp();
}

__device__ bool softmax_role(const CachedArgs& args, const Split& split, const Queries& queries, const uint8_t* values, uint8_t* wide,
                             uint32_t tmem, Control* c) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, t = warp >> 3, half = (warp >> 2) & 1;
  const int row = t * 128 + (warp & 3) * 32 + lane;  // of the segment's
  const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;
  const uint32_t s_at = tmem + lanes + t * kKeyTile + half * kHalf, p_at = tmem + lanes + t * kKeyTile + half * (kHalf / 2);
  const uint32_t o_at = tmem + lanes + kSums + t * kHeadDim + half * kHalf;
  const int page_shift = args.cache.page_shift, group = args.heads / args.cache.kv_heads;
  uint32_t no = 0, s_uses = 0, o_uses = 0;
  // A wait that runs out: the eight warps of a tile meet at barriers that know no limit, so they agree at the next of these
  // and leave there together.  (The other tile's find out by waits of their own.)
  bool ok = true;
#pragma unroll 1
  for (uint32_t segments = 0;; ++segments) {
    const uint32_t place = segments % kSegments;
    ok = mbar_wait_warp(smem_u32(&c->segment_full[place]), (segments / kSegments) & 1);
    const bool some = ok && c->has_segment[place];
    ok = ok && (!some || mbar_wait_warp(smem_u32(&c->q_full), segments & 1));  // (the factors were there before)
    if (tile_any(t, !ok)) return false;
    if (!some) return true;
    if (lane == 0) mbar_arrive(&c->q_empty);
    const Segment& s = c->segment[place];
    const int rows = s.rows * group - s.row0;
    const bool present = rows > t * 128;                                      // the tile has rows, ...
    const bool has_rows = rows > t * 128 + (warp & 3) * 32, valid = row < rows;  // ... the warp, the thread
    float factor = 0.0f, shift = 0.0f, sum = 0.0f;
    if (valid) {
      factor = __ldcg(queries.factors + (static_cast<int64_t>(s.kv_head) * args.batch.rows + s.first) * group + s.row0 + row);
    }
#pragma unroll 1
    for (int j = 0; j < s.tiles; ++j, ++no) {
      const uint32_t slot = no % S::kValueSlots;
      const uint32_t wide_slot = no % kWideSlots;
      ok = mbar_wait_warp(smem_u32(&c->v_full[slot]), (no / S::kValueSlots) & 1) &&
           mbar_wait_warp(smem_u32(&c->wide_empty[wide_slot]), ((no / kWideSlots) & 1) ^ 1);
      if (ok) {
        widen_values(values + slot * kKeyTileBytes, wide + wide_slot * kWideBytes);
        if (lane == 0) mbar_arrive(&c->wide_full[wide_slot]);
      }
      if (!present) {
        if (tile_any(t, !ok)) return false;
      } else {
        ok = ok && mbar_wait_warp(smem_u32(&c->s_full[t]), s_uses & 1);
        if (!ok) *const_cast<volatile int*>(&c->failed[t]) = 1;
        ++s_uses;
        tcgen05_fence_after();
        const bool is_first = j == 0;
        uint32_t p[kHalf / 2];
        float high = -INFINITY, added = 0.0f;
        // Weights by exponents, score + power of the values - reference.  A first tile sets the references, others raise
        // them where that is due, for both halves of a row alike, and the weights are made again.  (One loop: code that
        // runs once in a while is not in the cache, and a way of its own for it took 8000 cycles.)  A row whose scores
        // are very far above its reference takes them as they are first, so that no rounding matters.
        const float before = shift;
        bool anew = is_first;
#pragma unroll 1
        for (int attempt = 0; attempt < 4; ++attempt) {
          if (has_rows) {
            high = -INFINITY;
            added = 0.0f;
            uint32_t y[2][kPart];  // (sixteen tokens of scores are on their way during the sixteen before)
            tmem_ld_x16_async(s_at, y[0]);
#pragma unroll
            for (int part = 0; part < kHalf; part += kPart) {
              uint32_t(&now)[kPart] = y[part / kPart & 1];
              tmem_ld_wait();
              registers_loaded<kPart>(now);
              if (part + kPart < kHalf) tmem_ld_x16_async(s_at + part + kPart, y[(part / kPart + 1) & 1]);
              const int page = (half * kHalf + part) >> page_shift;
              const int k_power = c->powers[slot][0][page], v_power = c->powers[slot][1][page];
              const float scale = factor * power_of_two(k_power), bias = static_cast<float>(v_power) + shift;
              const uint64_t scale2 = pack2(scale, scale), bias2 = pack2(bias, bias);
              uint64_t of_part = 0;
#pragma unroll
              for (int k = 0; k < kPart / 2; ++k) {
                const uint64_t x = fma2(pack2(__uint_as_float(now[2 * k]), __uint_as_float(now[2 * k + 1])), scale2, bias2);
                float a, b;
                unpack2(x, a, b);
                high = largest_of(high, a, b);
                if (k % 4 == 3) {
                  unpack2(exp2_polynomial2<3>(x), a, b);
                } else {
                  a = exp2_approx(a);
                  b = exp2_approx(b);
                }
                of_part = add2(of_part, pack2(a, b));
                const __half2 two = __floats2half2_rn(a, b);
                p[part / 2 + k] = *reinterpret_cast<const uint32_t*>(&two);
              }
              float s0, s1;
              unpack2(of_part, s0, s1);
              added = fmaf(s0 + s1, power_of_two(-v_power), added);
            }
          }
          // (behind this both halves have read the scores: weights may be written over them)
          if (!tile_any(t, anew || high > kRiseBits || !ok)) break;
          if (*const_cast<volatile int*>(&c->failed[t])) return false;
          c->top[half][row] = high;
          tile_sync(t);
          const float top = fmaxf(c->top[0][row], c->top[1][row]);
          if (!anew && top > kFarBits) {
            anew = true;
            shift = 0.0f;
          } else if (anew || top > kRiseBits) {
            shift = top == -INFINITY ? -kNoReference : shift - top;
            anew = false;
          }
        }
        const float keep = shift == before || is_first ? 1.0f : exp2_approx(shift - before);
        if (has_rows && __any_sync(0xffffffffu, keep != 1.0f)) {
          // (O holds the tiles before: their products were asked for ahead of these scores)
          sum *= keep;
#pragma unroll 1
          for (int i = 0; i < kHalf; i += 32) {
            uint32_t o[32];
            tmem_ld_x32_async(o_at + i, o);
            tmem_ld_wait();
            registers_loaded<32>(o);
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * keep);
            tmem_st_x32(o_at + i, o);
          }
        }
        if (has_rows) {
          sum += added;
          tmem_st_x32(p_at, p);
          tmem_st_wait();
        }
        tcgen05_fence_before();
      }
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&c->v_empty[slot]);  // (its powers have been read)
        if (present) mbar_arrive(&c->p_full[t]);
      }
    }
    if (present) {
      ok = mbar_wait_warp(smem_u32(&c->o_full[t]), o_uses & 1);
      ++o_uses;
      tcgen05_fence_after();
      if (half) c->other_sum[row] = sum;
      if (tile_any(t, !ok)) return false;
      const int to = valid ? (s.first + (s.row0 + row) / group) * args.heads + s.kv_head * group + (s.row0 + row) % group : -1;
      float* slot = split.slots + slot_floats(S::kRows) * max(s.part, 0);
      float* at = (s.part < 0 ? args.sums + static_cast<size_t>(max(to, 0)) * kHeadDim : slot + row * kHeadDim) + half * kHalf;
      if (has_rows) {
#pragma unroll 1
        for (int i = 0; i < kHalf; i += 32) {
          uint32_t o[32];
          tmem_ld_x32_async(o_at + i, o);
          tmem_ld_wait();
          registers_loaded<32>(o);
          if (!valid) continue;
#pragma unroll
          for (int k = 0; k < 32; k += 8) {
            uint32_t w[8];
#pragma unroll
            for (int m = 0; m < 8; ++m) w[m] = __float_as_uint(__uint_as_float(o[k + m]) * kValueScale);
            store_32_bytes(at + i + k, w, true);
          }
        }
        if (valid && half == 0) {
          sum = (sum + c->other_sum[row]) * kSumScale;
          const float reference = sum == 0.0f ? -INFINITY : -shift;  // (a row that has seen only masked tokens leaves nothing)
          leave_row_part(args, s, to, row, reference, sum);
          if (s.part >= 0) {
            slot[S::kRows * kHeadDim + row] = reference;
            slot[S::kRows * (kHeadDim + 1) + row] = sum;
          }
        }
      }
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&c->o_empty[t]);
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&c->segment_empty[place]);
  }
}

__global__ void __launch_bounds__(S::kThreads, 1)
    shared_pairs_kernel(const __grid_constant__ CUtensorMap map, const __grid_constant__ CUtensorMap q_map, const CachedArgs args,
                        const Split split, const Queries queries) {
  extern __shared__ uint8_t raw[];
  uint8_t* keys = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  uint8_t* values = keys + S::kKeySlots * kKeyTileBytes;
  uint8_t* wide = values + S::kValueSlots * kKeyTileBytes;
  uint8_t* q = wide + kWideSlots * kWideBytes;
  Control* c = reinterpret_cast<Control*>(q + S::kQueryBytes);
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    init_work<S>(c);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&c->s_full[i], 1);
      mbar_init(&c->p_full[i], S::kSoftmaxWarps / 2);
      mbar_init(&c->o_full[i], 1);
      mbar_init(&c->o_empty[i], S::kSoftmaxWarps / 2);
    }
    mbar_init(&c->q_empty, S::kSoftmaxWarps + 1);
    c->failed[0] = c->failed[1] = 0;
    for (int i = 0; i < kWideSlots; ++i) {
      mbar_init(&c->wide_full[i], S::kSoftmaxWarps);
      mbar_init(&c->wide_empty[i], 1);
    }
    fence_barrier_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(&c->tmem, kColumns);
    tmem_relinquish();
  }
  tcgen05_fence_before();
  // (all but the queries' terms was there before the launch that makes these, whose blocks have all waited for that)
  find_begin<S, Part::kShared>(args, c);
  __syncthreads();
  release_successor();  // (the columns of TMEM are there)
  tcgen05_fence_after();
  const uint32_t tmem = c->tmem;
  bool ok = true;
  if (warp < S::kSoftmaxWarps) {
    ok = softmax_role(args, split, queries, values, wide, tmem, c);
  } else if (warp == kMmaWarp) {
    ok = mma_role(args, smem_u32(keys), smem_u32(wide), smem_u32(q), tmem, c);
    if (elect_one()) tcgen05_commit(&c->drained);
    __syncwarp();
    mbar_wait_warp(smem_u32(&c->drained), 0);
  } else {
    const int group = args.heads / args.cache.kv_heads;
    load_role<S, Part::kShared>(args, &map, smem_u32(keys), smem_u32(values), c, [&](const Segment& s, uint32_t number) {
      if (number == 0) wait_for_predecessor();
      if (!mbar_wait_warp(smem_u32(&c->q_empty), (number & 1) ^ 1)) return false;
      const int tiles = s.rows * group - s.row0 > 128 ? 2 : 1, of_head = args.batch.rows * group;
      if (elect_one()) {
        const uint32_t bar = smem_u32(&c->q_full);
        mbar_arrive_expect_tx_at(bar, 2 * tiles * kTileRowsBytes);
        for (int term = 0; term < 2; ++term) {
          for (int t = 0; t < tiles; ++t) {
            tma_load_2d_at(smem_u32(q) + term * kTermBytes + t * kTileRowsBytes, &q_map, 0,
                           (term * args.cache.kv_heads + s.kv_head) * of_head + s.first * group + s.row0 + t * 128, bar);
          }
        }
      }
      __syncwarp();
      return true;
    });
  }
  if (!ok && (threadIdx.x & 31) == 0) report_cache_error(args.cache.error, kDevWaitTimeout);
  wait_for_predecessor();  // (this launch ends behind that of the queries)
  tcgen05_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tcgen05_fence_after();
    tmem_dealloc(tmem, kColumns);
  }
}

}  // namespace

size_t shared_pairs_slot_bytes() { return sizeof(float) * slot_floats(S::kRows) * kSlotsPerBlock * device_sms(); }
int shared_pairs_slot_rows() { return S::kRows; }

size_t shared_pairs_query_bytes(int64_t rows, int heads) {
  return static_cast<size_t>(rows) * heads * (2 * kHeadDim + sizeof(float));
}

bool shared_pairs_supported(int64_t rows, int heads) { return 2 * rows * heads <= INT32_MAX - 256; }

cudaError_t launch_shared_pairs(const CachedArgs& args, float* slots, char* query_space, cudaStream_t stream) {
  const int sms = device_sms();
  if (sms > kMaxBlocks) return cudaErrorInvalidValue;
  const int64_t pairs = static_cast<int64_t>(args.batch.rows) * args.heads;
  const Queries queries{reinterpret_cast<uint8_t*>(query_space), reinterpret_cast<float*>(query_space + pairs * 2 * kHeadDim)};
  CUtensorMap map, q_map;
  if (!pages_tensor_map(args.cache, &map) || !codes_tensor_map(queries.codes, 2 * pairs, 128, &q_map)) return cudaErrorInvalidValue;
  static std::atomic<uint64_t> allowed{0};
  cudaError_t err = allow_shared_memory_once(shared_pairs_kernel, allowed);
  if (err != cudaSuccess) return err;
  err = launch_kernel(prepare_kernel, dim3(static_cast<unsigned>((pairs * 32 + kPrepareThreads - 1) / kPrepareThreads)), kPrepareThreads, 0,
                      LaunchStream(stream, true), args, queries);
  if (err != cudaSuccess) return err;
  const Split split{reinterpret_cast<JoinCounters*>(args.cache.attend_workspace), slots};
  return launch_kernel(shared_pairs_kernel, dim3(sms), S::kThreads, kSharedBytes, LaunchStream(stream, true), map, q_map, args, split,
                       queries);
}

}  // namespace nmoe
