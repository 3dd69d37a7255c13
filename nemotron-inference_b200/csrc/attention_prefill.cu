// Causal attention over whole prompts packed one behind the other.
//
//   s_tj = scale q_t . k_j for j <= t,  m_t = max_j s_tj,  o_t = sum_j e^(s_tj - m_t) v_j / sum_j e^(s_tj - m_t)
//
// in one pass over the keys: 128 rows against 128 keys at a time, the running maximum and sum of a row
// in the registers of one thread, scores and results in TMEM.
//
// A block works on two tiles of 128 query rows of one key head, so that each key and value tile that it
// brings in serves both, and one tile's exponentials run while the tensor cores work on the other.  The
// tiles are the same rows of two heads where a key head has an even number of them (the two then
// have as many key tiles each), else consecutive rows of one head.  Per key tile and query tile:
//   S = Q K^T      8 MMAs of 128 x 128 x 16, shared memory x shared memory -> TMEM
//   softmax warps  S -> registers, P = 2^(c S - c m) as bf16 back into TMEM, over S
//   O += P V       8 MMAs, TMEM x shared memory -> TMEM
// The reference m of a row is the maximum that it began with; only when a maximum has risen by more
// than 2^8 are O and the sum scaled anew, which keeps P within bf16's precision and the exponentials
// far from overflow, and which hardly ever happens after a row's first tile.
//
// Blocks ask for further blocks of the grid as they finish (no counter in memory, nothing to clear), so
// loads of the next tiles go on during the last exponentials of the current ones.
//
// What bounds it: a long prompt, the exponentials beside the MMAs.  Of a tile's 16384 a quarter are polynomials
// in FP32, the rest take the special function unit's 16 a cycle; alone the unit would take as long as the
// tile's 1024 MMA cycles.  8192 tokens, 32 heads on 2 key heads: 433 us alone = 1.27 PFLOP/s = 0.76 of the measured
// bf16 rate, the tensor pipe active in 68 % of the cycles.  Short prompts: some 5000 cycles of a block's item beside
// its tiles (queries in, the first tile's scores, the last one's results out), 8190 tokens in 23 prompts 81 us, the
// tensor pipe active in 33 %.  17 tokens: 10 us, a launch and one item.
#include <algorithm>

#include "attention.h"
#include "attention_mma.cuh"
#include "kernels.h"

namespace nmoe {
namespace {

constexpr int kTile = 128;                    // query rows, and keys, of a tile
constexpr int kTileBytes = kTile * kHeadDim * 2;
constexpr int kPanelBytes = kTileBytes / 2;   // 64 of the 128 dimensions: rows of 128 bytes
constexpr int kSlots = 5;                     // key and value tiles in flight, in turn
constexpr int kSoftmaxWarps = 8;              // four per query tile, a thread per row
constexpr int kMmaWarp = 8, kLoadWarp = 9, kCheckWarps = 10;  // and 11
constexpr int kThreads = 384;
constexpr int kSoftmaxRegisters = 216, kOtherRegisters = 72;  // 2 * 216 + 72 = 3 * 168, as launched
constexpr int kTmemColumns = 512;             // S of both tiles, O of both tiles, 128 columns each
constexpr float kRescale = 8.0f;              // binary orders by which a maximum may outgrow its reference

struct Work {
  int first, length;   // the prompt's first row, its rows
  int head[2], row[2]; // of each tile; row: first query row in the prompt
  int tiles[2];        // key tiles of each, 0: no such tile
  int kv_head;
};

struct Control {
  uint64_t q_full[2], q_empty[2], kv_full[kSlots], kv_empty[kSlots];
  uint64_t s_full[2], p_half[2], p_full[2], o_full[2], o_empty[2];
  uint64_t work_full[2], work_empty[2], next_full, drained;
  uint64_t unchecked_full[kSlots];  // values of a masked tile that the check warps have yet to see
  alignas(16) uint32_t next[4];
  Work work[2];
  int has_work[2];
  uint32_t tmem;
  int bad_values;  // a value in a masked tile is no number
  int stopped;
};

constexpr size_t kSharedBytes = 1024 + (2 + kSlots) * kTileBytes + sizeof(Control);
static_assert(kSharedBytes <= kMaxSharedBytes);

// Bits 15 and 31 are set for an infinity or NaN in the low or high half.
__device__ __forceinline__ uint32_t no_numbers(uint32_t two_bf16) { return (two_bf16 & 0x7f807f80u) + 0x00800080u; }

// What block `index` of the grid works on; a warp together.  Prompts in order, their last rows (which
// have the most keys) first, the heads that share keys next to one another.
__device__ __forceinline__ bool find_work(const PrefillArgs& args, bool two_heads, int index, Work& w) {
  const int rows = two_heads ? kTile : 2 * kTile;
  const int columns = two_heads ? args.heads / 2 : args.heads;
  const int column = index % columns;
  auto bounds = [&](int i, int& from, int& length) {
    from = min(max(args.offsets[i], 0), args.tokens);
    length = min(max(args.offsets[i + 1], from), args.tokens) - from;
  };
  const int2 unit = locate_unit(args.sequences, index / columns, [&](int i) {
    int from, length;
    bounds(i, from, length);
    return (length + rows - 1) / rows;
  });
  if (unit.x < 0) return false;
  bounds(unit.x, w.first, w.length);
  const int row = ((w.length + rows - 1) / rows - 1 - unit.y) * rows;
  const int head = two_heads ? 2 * column : column;
  w.kv_head = head / (args.heads / args.kv_heads);
  w.head[0] = head;
  w.head[1] = two_heads ? head + 1 : head;
  w.row[0] = row;
  w.row[1] = two_heads ? row : row + kTile;
  w.tiles[0] = row / kTile + 1;
  w.tiles[1] = w.row[1] < w.length ? w.row[1] / kTile + 1 : 0;
  return true;
}

// Brings queries, keys and values in.  The whole warp runs it, one lane issues.
__device__ void load_role(const PrefillArgs& args, bool two_heads, const CUtensorMap* q_map,
                          const CUtensorMap* k_map, const CUtensorMap* v_map, uint32_t q_at,
                          uint32_t slots_at, Control* c) {
  uint32_t loads = 0, q_loads[2] = {0, 0}, items = 0;
  int index = blockIdx.x;
  bool ok = true;
  for (;; ++items) {
    Work w;
    const bool some = index >= 0 && find_work(args, two_heads, index, w);
    const uint32_t place = items & 1;
    if (!(ok = wait_warp(smem_u32(&c->work_empty[place]), ((items >> 1) & 1) ^ 1))) break;
    if (elect_one()) {
      c->work[place] = w;
      c->has_work[place] = some;
      mbar_arrive(&c->work_full[place]);
      if (some) {
        fence_proxy_async_smem();  // (the answer before this one has been read)
        mbar_arrive_expect_tx(&c->next_full, 16);
        request_next_block(smem_u32(c->next), smem_u32(&c->next_full));
      }
    }
    __syncwarp();
    if (!some) break;
    const int most = max(w.tiles[0], w.tiles[1]);
    for (int load = 0; load < 2 * most && ok; ++load) {
      if (load == 0) {  // (the queries go with the first keys)
        for (int t = 0; t < 2 && ok; ++t) {
          if (w.tiles[t] == 0) continue;
          if (!(ok = wait_warp(smem_u32(&c->q_empty[t]), (q_loads[t] & 1) ^ 1))) break;
          ++q_loads[t];
          if (elect_one()) {
            const uint32_t bar = smem_u32(&c->q_full[t]);
            mbar_arrive_expect_tx_at(bar, kTileBytes);
            for (int panel = 0; panel < 2; ++panel) {
              tma_load_2d_at(q_at + t * kTileBytes + panel * kPanelBytes, q_map,
                             w.head[t] * kHeadDim + panel * 64, w.first + w.row[t], bar);
            }
          }
          __syncwarp();
        }
        if (!ok) break;
      }
      const uint32_t slot = loads % kSlots;
      if (!(ok = wait_warp(smem_u32(&c->kv_empty[slot]), ((loads / kSlots) & 1) ^ 1))) break;
      if (elect_one()) {
        const int tile = (load >> 1) + 1;
        const bool masked = (load & 1) && (tile == w.tiles[0] || tile == w.tiles[1]);
        const uint32_t bar = smem_u32(masked ? &c->unchecked_full[slot] : &c->kv_full[slot]);
        mbar_arrive_expect_tx_at(bar, kTileBytes);
        if (!masked) mbar_arrive_at(bar);  // (as many arrivals as the two check warps')
        for (int panel = 0; panel < 2; ++panel) {
          tma_load_2d_at(slots_at + slot * kTileBytes + panel * kPanelBytes, load & 1 ? v_map : k_map,
                         w.kv_head * kHeadDim + panel * 64, w.first + (load >> 1) * kTile, bar);
        }
      }
      __syncwarp();
      ++loads;
    }
    if (!ok) break;
    if (!(ok = wait_warp(smem_u32(&c->next_full), items & 1))) break;
    index = next_block(smem_u32(c->next));
  }
  if (ok) return;
  if (elect_one()) report_cache_error(args.error, kDevWaitTimeout);
  // what is in flight arrives before the block's shared memory is given up
  for (uint32_t back = 1; back <= min(loads, static_cast<uint32_t>(kSlots)); ++back) {
    const uint32_t load = loads - back;
    wait_warp(smem_u32(&c->kv_full[load % kSlots]), (load / kSlots) & 1);  // (the check warps' arrivals, too)
  }
  for (int t = 0; t < 2; ++t) {
    if (q_loads[t]) wait_warp(smem_u32(&c->q_full[t]), (q_loads[t] - 1) & 1);
  }
}

struct MmaRole {
  Control* c;
  uint32_t q_at, slots_at, tmem;
  uint32_t loads = 0, q_uses[2] = {0, 0}, p_uses[2] = {0, 0}, o_uses[2] = {0, 0};

  // S of tile t against the keys in `slot`.
  __device__ void scores(int t, uint32_t slot) {
    constexpr uint32_t idesc = make_idesc_bf16(kTile, false);
    const uint64_t a = make_smem_desc(q_at + t * kTileBytes, 16, 1024, 2);
    const uint64_t b = make_smem_desc(slots_at + slot * kTileBytes, 16, 1024, 2);
    if (elect_one()) {
#pragma unroll
      for (int k = 0; k < kHeadDim / 16; ++k) {
        const uint32_t at = (k / 4) * kPanelBytes + (k % 4) * 32;
        mma_f16_ss(tmem + t * kTile, advance_smem_desc(a, at), advance_smem_desc(b, at), idesc, k > 0);
      }
      tcgen05_commit(&c->s_full[t]);
    }
    __syncwarp();
  }

  // O of tile t, with the values in `slot`: a token's row is 128 consecutive n, 64 to a panel; eight
  // tokens are 1024 bytes.  The weights come in two halves.
  __device__ bool values(int t, uint32_t slot, bool first, bool last) {
    constexpr uint32_t idesc = make_idesc_bf16(kHeadDim, true);
    const uint64_t b = make_smem_desc(slots_at + slot * kTileBytes, kPanelBytes, 1024, 2);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (!wait(half ? &c->p_full[t] : &c->p_half[t], p_uses[t] & 1)) return false;
      if (elect_one()) {
#pragma unroll
        for (int k = half * 4; k < half * 4 + 4; ++k) {
          mma_f16_ts(tmem + 2 * kTile + t * kHeadDim, tmem + t * kTile + k * 8,
                     advance_smem_desc(b, k * 2048), idesc, !first || k > 0);
        }
        if (half && last) tcgen05_commit(&c->o_full[t]);
      }
      __syncwarp();
    }
    ++p_uses[t];
    return true;
  }

  __device__ bool wait(uint64_t* bar, uint32_t parity) {
    const bool ok = wait_warp(smem_u32(bar), parity);
    tcgen05_fence_after();
    return ok;
  }
  __device__ bool wait_load(uint32_t load) {
    return wait(&c->kv_full[load % kSlots], (load / kSlots) & 1);
  }
  __device__ void release(uint64_t* bar) {
    if (elect_one()) tcgen05_commit(bar);
    __syncwarp();
  }

  __device__ bool item(const int (&tiles)[2]) {
    const int most = max(tiles[0], tiles[1]);
    if (!wait_load(loads)) return false;
    for (int t = 0; t < 2; ++t) {
      if (tiles[t] == 0) continue;
      if (!wait(&c->q_full[t], q_uses[t] & 1)) return false;
      ++q_uses[t];
      scores(t, loads % kSlots);
      if (tiles[t] == 1) release(&c->q_empty[t]);
    }
    release(&c->kv_empty[loads % kSlots]);
    for (int j = 0; j < most; ++j) {
      const uint32_t v_load = loads + 2 * j + 1, k_load = v_load + 1;
      if (!wait_load(v_load)) return false;
      if (j + 1 < most && !wait_load(k_load)) return false;
      for (int t = 0; t < 2; ++t) {
        if (j >= tiles[t]) continue;
        if (j == 0) {
          if (!wait(&c->o_empty[t], (o_uses[t] & 1) ^ 1)) return false;
          ++o_uses[t];
        }
        if (!values(t, v_load % kSlots, j == 0, j + 1 == tiles[t])) return false;
        if (j + 1 < tiles[t]) {
          scores(t, k_load % kSlots);
          if (j + 2 == tiles[t]) release(&c->q_empty[t]);
        }
      }
      release(&c->kv_empty[v_load % kSlots]);
      if (j + 1 < most) release(&c->kv_empty[k_load % kSlots]);
    }
    loads += 2 * most;
    return true;
  }
};

// Two warps that see the values of masked tiles before the tensor cores do: a weight of 0 times a value that is
// no number would be none either.  Such values become 0 here and are added by add_bad_values().  The masked tiles
// of a block's work are the last one of each query tile.
__device__ bool check_role(uint8_t* slots, Control* c) {
  const int thread = threadIdx.x - kCheckWarps * 32;
  uint32_t loads = 0, seen = 0;  // a bit per slot: the parity of what has been checked there
#pragma unroll 1
  for (uint32_t items = 0;; ++items) {
    const uint32_t place = items & 1;
    if (!wait_warp(smem_u32(&c->work_full[place]), (items >> 1) & 1)) return false;
    const int some = c->has_work[place], tiles[2] = {c->work[place].tiles[0], c->work[place].tiles[1]};
    __syncwarp();
    if (!some) return true;
    if ((thread & 31) == 0) mbar_arrive(&c->work_empty[place]);
#pragma unroll 1
    for (int t = 0; t < 2; ++t) {
      if (tiles[t] == 0 || (t == 1 && tiles[1] == tiles[0])) continue;
      const uint32_t slot = (loads + 2 * tiles[t] - 1) % kSlots;
      if (!wait_warp(smem_u32(&c->unchecked_full[slot]), (seen >> slot) & 1)) return false;
      seen ^= 1u << slot;
      uint4* tile = reinterpret_cast<uint4*>(slots + slot * kTileBytes) + thread;
#pragma unroll 1
      for (int i = 0; i < kTileBytes / 16; i += 8 * 64) {
        uint4 x[8];
        uint32_t bad = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = tile[i + k * 64];
#pragma unroll
        for (int k = 0; k < 8; ++k) bad |= no_numbers(x[k].x) | no_numbers(x[k].y) | no_numbers(x[k].z) | no_numbers(x[k].w);
        if ((bad & 0x80008000u) == 0) continue;
        c->bad_values = 1;
#pragma unroll 1
        for (int k = 0; k < 64; ++k) {
          uint16_t* value = reinterpret_cast<uint16_t*>(tile + i + k / 8 * 64) + k % 8;
          if ((*value & 0x7f80u) == 0x7f80u) *value = 0;
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if ((thread & 31) == 0) mbar_arrive(&c->kv_full[slot]);
    }
    loads += 2 * max(tiles[0], tiles[1]);
  }
}

// Adds what check_role() took out of the block's tiles to a row's result.
__device__ __forceinline__ void add_bad_values(const PrefillArgs& args, const Work& w, int t, int row,
                                               uint32_t (&o)[kHeadDim]) {
#pragma unroll 1
  for (int other = 0; other <= t; ++other) {
    if (w.tiles[other] == 0) continue;
    const int begin = (w.tiles[other] - 1) * kTile, end = min(begin + kTile, row + 1);
#pragma unroll 1
    for (int j = begin; j < end; ++j) {
      const __nv_bfloat16* v = args.v + (w.first + j) * args.v_stride + w.kv_head * kHeadDim;
#pragma unroll
      for (int i = 0; i < kHeadDim; ++i) {
        const float x = __bfloat162float(v[i]);
        if (!(fabsf(x) < INFINITY)) o[i] = __float_as_uint(__uint_as_float(o[i]) + x);
      }
    }
    if (w.row[0] == w.row[1]) break;  // (both tiles have the same last one)
  }
}

// Weights are 2^(s c - round(m c)), one fma each.  What the rounding adds to all of a row's exponents cancels, as
// long as references that follow one another are told apart by their rounded products, and it stays below 64.  Where
// |m c| is 2^30 or more (keys that are masked by the type's lowest value), scores that differ at all do so by 2^6
// orders; c is cut to a power of two there, so that m c is exact.
__device__ __forceinline__ float factor_for(float top, float factor) {
  const bool far = fabsf(top * factor) >= 1073741824.0f;
  return far ? __uint_as_float(__float_as_uint(factor) & 0x7f800000u) : factor;
}

// Four warps per query tile, a thread per row.
__device__ void softmax_role(const PrefillArgs& args, uint32_t tmem, Control* c) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t = warp >> 2, thread = threadIdx.x & (kTile - 1);
  const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // 32 lanes a warp, from bit 16
  const uint32_t s_at = tmem + lanes + t * kTile, o_at = tmem + lanes + 2 * kTile + t * kHeadDim;
  const float factor = args.scale * kLog2e;
  uint32_t s_uses = 0, o_uses = 0;
  for (uint32_t items = 0;; ++items) {
    const uint32_t place = items & 1;
    if (!wait_warp(smem_u32(&c->work_full[place]), (items >> 1) & 1)) break;
    if (!c->has_work[place]) return;
    const Work w = c->work[place];
    __syncwarp();
    if (lane == 0) mbar_arrive(&c->work_empty[place]);
    const int tiles = w.tiles[t];
    float top = 0.0f, own_factor = factor;
    uint64_t sum2 = 0, by_rounding2 = 0;
    bool ok = true;
    for (int j = 0; j < tiles; ++j) {
      if (!(ok = wait_warp(smem_u32(&c->s_full[t]), s_uses & 1))) break;
      ++s_uses;
      tcgen05_fence_after();
      uint32_t s[kTile];
#pragma unroll
      for (int part = 0; part < 4; ++part) tmem_ld_x32_async(s_at + part * 32, s + part * 32);
      tmem_ld_wait();
      registers_loaded<kTile>(s);
      if (j + 1 == tiles) {
#pragma unroll
        for (int i = 0; i < kTile; ++i) {
          if (i > thread) s[i] = 0xff800000u;
        }
      }
      float high[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) high[i] = __uint_as_float(s[i]);
#pragma unroll
      for (int i = 4; i < kTile; ++i) high[i & 3] = fmaxf(high[i & 3], __uint_as_float(s[i]));
      const float highest = fmaxf(fmaxf(high[0], high[1]), fmaxf(high[2], high[3]));
      if (j == 0) {
        top = highest;
        own_factor = factor_for(top, factor);
      } else if (__any_sync(0xffffffffu, (highest - top) * factor > kRescale)) {
        // (S of this tile is complete, so O of those before it is)
        const float higher = fmaxf(highest, top);
        const float next_factor = factor_for(higher, factor);
        const float by = own_factor == next_factor ? __fmul_rn(top, own_factor) - __fmul_rn(higher, own_factor)
                                                   : (top - higher) * factor;
        const float keep = top > -INFINITY ? exp2_approx(by) : 0.0f;  // (or both are -infinity)
        top = higher;
        own_factor = next_factor;
        const uint64_t keep2 = pack2(keep, keep);
        sum2 = mul2(sum2, keep2);
#pragma unroll 1
        for (int part = 0; part < 4; ++part) {
          uint32_t o[32];
          tmem_ld_x32_async(o_at + part * 32, o);
          tmem_ld_wait();
          registers_loaded<32>(o);
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * keep);
          tmem_st_x32(o_at + part * 32, o);
        }
      }
      const float shift = top == -INFINITY ? 0.0f : -__fmul_rn(top, own_factor);
      const uint64_t shift2 = pack2(shift, shift), factor2 = pack2(own_factor, own_factor);
      uint64_t part2[2] = {0, 0};
#pragma unroll
      for (int part = 0; part < 4; ++part) {
        uint32_t p[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int at = part * 32 + 2 * i;
          const uint64_t x = fma2(pack2(__uint_as_float(s[at]), __uint_as_float(s[at + 1])), factor2, shift2);
          float a, b;
          uint64_t e;
          if (i % 4 == 3) {
            e = exp2_polynomial2<4>(x);
            unpack2(e, a, b);
          } else {
            unpack2(x, a, b);
            a = exp2_approx(a);
            b = exp2_approx(b);
            e = pack2(a, b);
          }
          part2[i & 1] = add2(part2[i & 1], e);
          p[i] = pack_bf16(a, b);
        }
        tmem_st_x16(s_at + part * 16, p);
        if (part == 1) {
          tmem_st_wait();
          tcgen05_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&c->p_half[t]);
        }
      }
      part2[0] = add2(part2[0], part2[1]);
      sum2 = add2(sum2, part2[0]);
      tmem_st_wait();
      if (j + 1 == tiles) {
        uint64_t rounded2 = fma2(part2[0], pack2(-1.0f, -1.0f), 0);
#pragma unroll 1
        for (int part = 0; part < 2; ++part) {
          uint32_t p[32];
          tmem_ld_x32_async(s_at + part * 32, p);
          tmem_ld_wait();
          registers_loaded<32>(p);
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            rounded2 = add2(rounded2, pack2(__uint_as_float(p[i] << 16), __uint_as_float(p[i] & 0xffff0000u)));
          }
        }
        by_rounding2 = rounded2;
      }
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&c->p_full[t]);
    }
    if (!ok) break;
    if (tiles == 0) continue;
    if (!wait_warp(smem_u32(&c->o_full[t]), o_uses & 1)) break;
    ++o_uses;
    tcgen05_fence_after();
    float sum, other;
    unpack2(sum2, sum, other);
    sum += other;
    // What is divided by is the sum of the weights that were multiplied, those of the last tile as they were
    // rounded: in rows of a few keys, which all lie there, a rounding then only shifts the shares of the keys
    // (largest error of 20 prompts of 128, 40 heads: 2^-8 x 1.46 of the weighted |v| instead of 1.76).  Elsewhere
    // many roundings make up for one another.
    float by_rounding, by_rounding_too;
    unpack2(by_rounding2, by_rounding, by_rounding_too);
    by_rounding += by_rounding_too;
    const int row = w.row[t] + thread;
    const bool valid = row < w.length;
    const bool bad = *reinterpret_cast<volatile int*>(&c->bad_values) != 0;
    const float inverse = 1.0f / (sum + by_rounding);
    const size_t at = static_cast<size_t>(w.first + row) * args.heads + w.head[t];
    uint32_t o[kHeadDim];
#pragma unroll
    for (int part = 0; part < 4; ++part) tmem_ld_x32_async(o_at + part * 32, o + part * 32);
    tmem_ld_wait();
    registers_loaded<kHeadDim>(o);
    tcgen05_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(&c->o_empty[t]);
    if (valid) {
      if (bad) add_bad_values(args, w, t, row, o);
#pragma unroll
      for (int part = 0; part < 8; ++part) {  // 32 bytes, whole sectors
        uint32_t two[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int column = part * 16 + 2 * i;
          two[i] = pack_bf16(__uint_as_float(o[column]) * inverse, __uint_as_float(o[column + 1]) * inverse);
        }
        store_32_bytes(args.out + at * kHeadDim + part * 16, two, args.out_aligned);
      }
    }
    if (valid && args.lse != nullptr) args.lse[at] = kLn2 * (top * factor + log2f(sum));
  }
  if (lane == 0) report_cache_error(args.error, kDevWaitTimeout);
}

// Of a call that computes nothing: zeros, and no sums.  (Nobody asks for another's block then: all of the grid run.)
__device__ void clear_results(const PrefillArgs& args) {
  const int from = min(max(args.offsets[0], 0), args.tokens), to = min(args.offsets[args.sequences], args.tokens);
  for (int row = from + static_cast<int>(blockIdx.x); row < to; row += gridDim.x) {
    const size_t at = static_cast<size_t>(row) * args.heads;
    for (int i = threadIdx.x; i < args.heads * (kHeadDim / 8); i += kThreads) {
      reinterpret_cast<uint4*>(args.out + at * kHeadDim)[i] = make_uint4(0, 0, 0, 0);
    }
    if (args.lse == nullptr) continue;
    for (int i = threadIdx.x; i < args.heads; i += kThreads) args.lse[at + i] = -INFINITY;
  }
}

__global__ void __launch_bounds__(kThreads, 1)
    prefill_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                   const __grid_constant__ CUtensorMap v_map, const PrefillArgs args, bool two_heads) {
  extern __shared__ uint8_t raw[];
  uint8_t* shared = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  uint8_t* slots = shared + 2 * kTileBytes;
  Control* c = reinterpret_cast<Control*>(slots + kSlots * kTileBytes);
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&c->q_full[t], 1);
      mbar_init(&c->q_empty[t], 1);
      mbar_init(&c->s_full[t], 1);
      mbar_init(&c->p_half[t], 4);
      mbar_init(&c->p_full[t], 4);
      mbar_init(&c->o_full[t], 1);
      mbar_init(&c->o_empty[t], 4);
      mbar_init(&c->work_full[t], 1);
      mbar_init(&c->work_empty[t], kSoftmaxWarps + 3);
    }
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(&c->kv_full[i], 2);
      mbar_init(&c->unchecked_full[i], 1);
      mbar_init(&c->kv_empty[i], 1);
    }
    mbar_init(&c->next_full, 1);
    mbar_init(&c->drained, 1);
    c->bad_values = 0;
    fence_barrier_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(&c->tmem, kTmemColumns);
    tmem_relinquish();
  }
  tcgen05_fence_before();
  wait_for_predecessor();
  if (threadIdx.x == 0) c->stopped = *args.error != 0;  // a wait of an earlier call ran out
  __syncthreads();
  release_successor();  // (the columns of TMEM are there)
  tcgen05_fence_after();
  const uint32_t tmem = c->tmem;
  if (c->stopped) {
    clear_results(args);
  } else if (warp < kSoftmaxWarps) {
    more_registers<kSoftmaxRegisters>();
    softmax_role(args, tmem, c);
  } else if (warp == kMmaWarp) {
    fewer_registers<kOtherRegisters>();
    MmaRole role{c, smem_u32(shared), smem_u32(slots), tmem};
    bool ok = true;
    for (uint32_t items = 0;; ++items) {
      const uint32_t place = items & 1;
      if (!(ok = wait_warp(smem_u32(&c->work_full[place]), (items >> 1) & 1))) break;
      if (!c->has_work[place]) break;
      const int tiles[2] = {warp_uniform(c->work[place].tiles[0]), warp_uniform(c->work[place].tiles[1])};
      __syncwarp();
      if (elect_one()) mbar_arrive(&c->work_empty[place]);
      __syncwarp();
      if (!(ok = role.item(tiles))) break;
    }
    if (!ok && elect_one()) report_cache_error(args.error, kDevWaitTimeout);
    role.release(&c->drained);
    wait_warp(smem_u32(&c->drained), 0);
  } else {
    fewer_registers<kOtherRegisters>();
    if (warp == kLoadWarp) {
      load_role(args, two_heads, &q_map, &k_map, &v_map, smem_u32(shared), smem_u32(slots), c);
    } else if (!check_role(slots, c) && elect_one()) {
      report_cache_error(args.error, kDevWaitTimeout);
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tcgen05_fence_after();
    tmem_dealloc(tmem, kTmemColumns);
  }
}

}  // namespace

cudaError_t launch_attention_prefill(const PrefillArgs& args, cudaStream_t stream) {
  CUtensorMap q, k, v;
  if (!rows_tensor_map(args.q, args.tokens, args.heads, args.q_stride, kTile, &q) ||
      !rows_tensor_map(args.k, args.tokens, args.kv_heads, args.k_stride, kTile, &k) ||
      !rows_tensor_map(args.v, args.tokens, args.kv_heads, args.v_stride, kTile, &v)) {
    return cudaErrorInvalidValue;
  }
  const bool two_heads = args.heads / args.kv_heads % 2 == 0;
  const int64_t rows = two_heads ? kTile : 2 * kTile;
  const int64_t columns = two_heads ? args.heads / 2 : args.heads;
  const int64_t blocks = std::min<int64_t>(args.tokens, args.tokens / rows + args.sequences) * columns;
  if (blocks > INT32_MAX) return cudaErrorInvalidValue;
  static std::atomic<uint64_t> allowed{0};
  cudaError_t err = allow_shared_memory_once(prefill_kernel, allowed);
  if (err != cudaSuccess) return err;
  return launch_kernel(prefill_kernel, dim3(static_cast<unsigned>(blocks)), kThreads, kSharedBytes,
                       LaunchStream(stream, true), q, k, v, args, two_heads);
}

}  // namespace nmoe
