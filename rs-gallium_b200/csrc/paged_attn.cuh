// paged_attn.cuh -- what the two attention kernels share: arguments, the split of
// a batch into work items, and the output store.
//
//   o = sum_j e^(s_j - m) v_j / (e^(sink - m) + sum_j e^(s_j - m)),  s_j = scale (q . k_j)
//
// in one pass over K and V with a running maximum and sum.
//
// Work.  The query heads that share a KV head are rows of one tile, so each
// key is read once for all of them: a tile is (rows / group) tokens x group
// heads.  A sequence with at most kRows such rows (a decoding one) is one 16-row
// tile of attn_rows_kernel, any other goes to attn_tile_kernel's tiles of 128 or
// 256 rows (where the host's bounds tell that no sequence of the batch is a
// decoding one, attn_rows_kernel is not launched, and should the device's lengths
// say otherwise, the tile kernel takes that sequence too).  A tile's keys are cut
// over several CTAs when the batch has too few tiles to fill the GPU: each part
// writes its unnormalised sum with its maximum and its sum of weights, and a last
// kernel joins them in their order.  The lengths are on the device, so every CTA
// works out its own part from them (a scan over the sequences), and the grids are
// sized from the host's bounds.
#pragma once

#include <algorithm>

#include "paged.cuh"
#include "ptx.cuh"

namespace gb {
namespace paged {

// 2^x by the hardware's approximation (relative error 2^-22); 2^-inf = 0.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The factor of a part of a row (keys of one warp, of one split) whose sums refer to the
// maximum m, where all parts' refer to M; l: its sum of weights.  A maximum passes NaN
// over, so m stays -inf in a part that saw nothing, whose l is 0, and in one whose
// scores were NaN, whose l is NaN: l is the factor of both.
__device__ __forceinline__ float part_factor(float m, float l, float M) {
  return m == -INFINITY ? l : ex2(m - M);
}

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kRows = 16;      // rows of a decoding sequence's tile, and of a joining CTA
constexpr int kMaxGroup = 16;  // query heads per KV head

// Splitting.  n = the units (of `unit` keys) a sequence's rows see, t = ceil(5/4
// W / target) units per split (W: the units of all tiles; a quarter more than
// an even share, so that a batch of nearly `target` equal tiles stays whole),
// so a sequence has ceil(n / t) splits.  Tiles with more than one split have n >
// t, hence there are at most W / t <= target such tiles (Plan::target entries of
// `groups`) with at most 2 W / t <= 2 target splits (`slots`).
struct Plan {
  int tile_rows;  // rows per tile
  int unit;       // keys per unit
  int target;     // items to aim for
  int min_units;  // units per split, at least
  __host__ __device__ constexpr int slots() const { return 2 * target; }
};
// KV heads that a CTA of attn_rows_kernel takes side by side, where their number allows.
template <int HD>
__host__ __device__ constexpr int heads_side() { return HD == 128 ? 2 : 1; }
// Shares of attn_rows_kernel with HPC heads side by side: four, two or one CTA on each of
// 148 SMs, as shared memory holds; a unit is a step of the four warps, 64 keys in all.
template <int HD, int HPC>
__host__ __device__ constexpr Plan rows_plan() {
  return Plan{kRows, 64 / HPC, 148 * (HD == 64 ? 4 : HD == 128 ? 2 : 1), 2};
}
template <int HD>
constexpr Plan tile_plan() {
  return HD == 64    ? Plan{128, 64, 296, 8}  // two CTAs per SM
         : HD == 128 ? Plan{256, 128, 148, 4}
                     : Plan{128, 64, 148, 8};
}

struct Group {  // a split tile, for the joining kernel
  int row0, rows, g;
  int slot0, slot1, step;  // partial result s > 0 is in slot1 + s step, the first in slot0
  int splits;
};

struct Partials {
  int* n_groups;
  Group* groups;    // [target]
  float2* ml;       // [slots][tile_rows]: reference maximum (log2), sum of weights
  float* o;         // [slots][tile_rows][head_dim]
};

struct AttnArgs {
  Batch b;
  int nh, group, window, out_f32;
  int rows_grid;  // CTAs of attn_rows_kernel
  int side;       // KV heads that each takes side by side
  int all_tiles;  // attn_tile_kernel takes the decoding sequences too
  float scale;  // scale * log2 e
  const void* q;
  int64_t q_row, q_head;
  const void *k_pool, *v_pool;
  const float* sinks;
  void* out;
  int64_t o_row, o_head;
  Partials rows, tiles;
  uint64_t wait_ns;  // the tile kernel's test hooks (gb_paged_set_test_hooks)
  int withhold_q;
};

// What a CTA does: `tokens` tokens of sequence seq from row row0, the first at
// position pos0, KV head g, units [u0, u1).
struct Item {
  int seq, row0, tokens, pos0, g, u0, u1;
  int slot;  // of the partial result, -1: the tile is not split
};

__device__ __forceinline__ int first_unit(int pos, int window, int unit) {
  return window > 0 && pos >= window ? (pos - window + 1) / unit : 0;
}

// Sequences that a warp holds, a lane for every 32nd, and the items that they may have
// then: as many rows and heads do not fit in memory.
constexpr int kLaneSeqs = 128;
constexpr uint32_t kMaxItems = (1u << 25) - 1;

struct SeqWork {
  int tiles, units;
};
template <bool SMALL>
__device__ __forceinline__ SeqWork seq_work(const AttnArgs& a, const Plan& pl, const Seq& q,
                                            int tpt) {
  SeqWork w{0, 0};
  if ((!a.all_tiles && q.q_len * a.group <= kRows) != SMALL) return w;
  w.tiles = (q.q_len + tpt - 1) / tpt;
  const int last = q.kv_len - 1;
  if (w.tiles && last >= 0)
    w.units = last / pl.unit - first_unit(max(q.kv_len - q.q_len, 0), a.window, pl.unit) + 1;
  return w;
}

template <typename V>
__device__ __forceinline__ V warp_inclusive(V v) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V t = __shfl_up_sync(kFullMask, v, o);
    if ((threadIdx.x & 31) >= o) v += t;
  }
  return v;
}

// Units per split (see Plan): the same in every CTA.  So much work that the product would
// not fit (w at its limit) is never split.
constexpr unsigned long long kMaxWork = 1ull << 48;
__device__ __forceinline__ int split_units(const AttnArgs& a, const Plan& pl, unsigned long long w) {
  w = min(w, kMaxWork);
  const unsigned long long t = (w * a.b.nkv * 5 + 4 * pl.target - 1) / (4u * pl.target);
  return max(pl.min_units, (int)min(t, 1ull << 30));
}

// Item `j` (of its sequence) of sequence s with `splits` splits per tile; first_group,
// first_slot: the split tiles and their splits of the sequences before.
__device__ __forceinline__ Item make_item(const AttnArgs& a, const Plan& pl, const Partials& part,
                                          int tpt, int s, const Seq& q, const SeqWork& x, int splits,
                                          uint32_t j, uint32_t first_group, uint32_t first_slot,
                                          bool write_group) {
  Item it;
  it.seq = s;
  const uint32_t js = j / (uint32_t)a.b.nkv;
  it.g = (int)(j - js * (uint32_t)a.b.nkv);
  // the last tile, which sees most keys, first
  const uint32_t back = splits > 1 ? js / (uint32_t)splits : js;
  const int split = (int)(js - back * (uint32_t)splits), tile = x.tiles - 1 - (int)back;
  it.row0 = q.row0 + tile * tpt;
  it.tokens = min(tpt, q.q_len - tile * tpt);
  it.pos0 = q.kv_len - q.q_len + tile * tpt;
  const int last = it.pos0 + it.tokens - 1;
  const int lo = first_unit(it.pos0, a.window, pl.unit);
  const int n = last < 0 ? 0 : last / pl.unit - lo + 1;
  it.u0 = lo;
  it.u1 = lo + n;
  it.slot = -1;
  if (splits > 1) {
    const int per = (n + splits - 1) / splits;
    it.u0 = lo + min(split * per, n);
    it.u1 = lo + min((split + 1) * per, n);
    const int nth = tile * a.b.nkv + it.g;
    const int slot0 = (int)first_slot + nth * splits;
    it.slot = slot0 + split;
    if (split == 0 && write_group)
      part.groups[first_group + nth] = Group{it.row0, it.tokens * a.group, it.g, slot0, slot0, 1, splits};
  }
  return it;
}

// Finds the CTA's item among the sequences of one kind (SMALL: at most kRows
// rows); false: there is none.  Called by the whole CTA of THREADS threads; tpt:
// tokens per tile.  Up to 128 sequences every warp works it out for itself, a lane per
// sequence, without a barrier; more take the whole CTA.
// A q_start that goes back makes sequences share rows, and then more items than the
// host's bound has CTAs: the split tiles of a sequence whose items do not all have one
// are left out of n_groups (and those after it: the count runs with the items), since
// nobody may have written their groups.
template <bool SMALL, int THREADS>
__device__ bool find_item(const AttnArgs& a, const Plan& pl, const Partials& part, int tpt,
                          Item* out) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Batch& b = a.b;
  if (b.n_seqs <= kLaneSeqs) {
    Seq q[4];
    SeqWork x[4];
    unsigned long long w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      q[i] = Seq{0, 0, 0};
      x[i] = SeqWork{0, 0};
      if (32 * i >= b.n_seqs) continue;
      const int s = 32 * i + lane;
      if (s < b.n_seqs) q[i] = load_seq(b, s, blockIdx.x == 0 && warp == 0);
      x[i] = seq_work<SMALL>(a, pl, q[i], tpt);
      w += (unsigned long long)x[i].tiles * x[i].units;
    }
    // In parts of 24 bits, which add up in 32; with so much work in one lane there are
    // no splits, whatever the sum.
    w = min(w, kMaxWork - 1);
    w = (unsigned long long)__reduce_add_sync(kFullMask, (uint32_t)w & 0xffffffu) +
        ((unsigned long long)__reduce_add_sync(kFullMask, (uint32_t)(w >> 24) & 0xffffffu) << 24);
    const int t = split_units(a, pl, w);
    Item it{};
    bool found = false;
    uint32_t base = 0, base_groups = 0, base_slots = 0;  // of the sequences 32 i and on before
    uint32_t n_groups = 0;  // of the sequences whose items all have a CTA
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (32 * i >= b.n_seqs) continue;
      const int splits = x[i].units > t ? (x[i].units + t - 1) / t : 1;
      // no more than kMaxItems each: 128 of them still add up in 32 bits
      const uint32_t tiles = (uint32_t)min((unsigned long long)x[i].tiles * b.nkv, (unsigned long long)kMaxItems);
      const uint32_t items = (uint32_t)min((unsigned long long)tiles * splits, (unsigned long long)kMaxItems);
      const uint32_t upto = base + warp_inclusive(items);
      uint32_t groups = 0, slots = 0;
      const bool split = __any_sync(kFullMask, splits > 1);
      if (split) {
        groups = base_groups + warp_inclusive(splits > 1 ? tiles : 0);
        slots = base_slots + warp_inclusive(splits > 1 ? items : 0);
      }
      if (blockIdx.x < upto && blockIdx.x >= upto - items) {
        it = make_item(a, pl, part, tpt, 32 * i + lane, q[i], x[i], splits, blockIdx.x - (upto - items),
                       groups - tiles, slots - items, warp == 0);
        found = true;
      }
      base = __shfl_sync(kFullMask, upto, 31);
      if (split) {
        n_groups = max(n_groups, __reduce_max_sync(kFullMask, upto <= gridDim.x ? groups : 0));
        base_groups = __shfl_sync(kFullMask, groups, 31);
        base_slots = __shfl_sync(kFullMask, slots, 31);
      }
    }
    if (blockIdx.x == 0 && tid == 0) *part.n_groups = (int)n_groups;
    const unsigned m = __ballot_sync(kFullMask, found);
    if (!m) return false;
    const int src = __ffs(m) - 1;
    out->seq = __shfl_sync(kFullMask, it.seq, src);
    out->row0 = __shfl_sync(kFullMask, it.row0, src);
    out->tokens = __shfl_sync(kFullMask, it.tokens, src);
    out->pos0 = __shfl_sync(kFullMask, it.pos0, src);
    out->g = __shfl_sync(kFullMask, it.g, src);
    out->u0 = __shfl_sync(kFullMask, it.u0, src);
    out->u1 = __shfl_sync(kFullMask, it.u1, src);
    out->slot = __shfl_sync(kFullMask, it.slot, src);
    return true;
  }
  constexpr int kW = THREADS / 32;
  __shared__ unsigned long long red[kW];
  __shared__ unsigned long long run[kW][2];
  __shared__ Item found;
  __shared__ int have, n_groups;
  Seq mine{0, 0, 0};  // of the first THREADS sequences
  unsigned long long w = 0;
  for (int s = tid; s < b.n_seqs; s += THREADS) {
    const Seq q = load_seq(b, s, blockIdx.x == 0);
    if (s == tid) mine = q;
    const SeqWork x = seq_work<SMALL>(a, pl, q, tpt);
    w = min(w + (unsigned long long)x.tiles * x.units, kMaxWork);
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) w += __shfl_xor_sync(kFullMask, w, o);
  if (lane == 0) red[warp] = w;
  if (tid == 0) have = n_groups = 0;
  __syncthreads();
  w = 0;
#pragma unroll
  for (int i = 0; i < kW; ++i) w += red[i];
  const int t = split_units(a, pl, w);
  // prefixes over the sequences: items; splits (high half) and tiles of split sequences
  unsigned long long base_items = 0, base_groups = 0;
  for (int s0 = 0; s0 < b.n_seqs; s0 += THREADS) {
    const int s = s0 + tid;
    Seq q{0, 0, 0};
    if (s < b.n_seqs) q = s0 ? load_seq(b, s, false) : mine;
    const SeqWork x = seq_work<SMALL>(a, pl, q, tpt);
    const int splits = x.units > t ? (x.units + t - 1) / t : 1;
    const unsigned long long tiles = (unsigned long long)x.tiles * b.nkv;
    const unsigned long long items = tiles * splits;
    const unsigned long long groups = splits > 1 ? (items << 32) | tiles : 0;
    const unsigned long long ii = warp_inclusive(items), gg = warp_inclusive(groups);
    __syncthreads();
    if (lane == 31) {
      run[warp][0] = ii;
      run[warp][1] = gg;
    }
    __syncthreads();
    unsigned long long bi = base_items, bg = base_groups;
    for (int i = 0; i < kW; ++i) {
      if (i < warp) {
        bi += run[i][0];
        bg += run[i][1];
      }
      base_items += run[i][0];
      base_groups += run[i][1];
    }
    const unsigned long long before = bi + ii - items;
    if (splits > 1 && bi + ii <= gridDim.x) atomicMax(&n_groups, (int)(uint32_t)(bg + gg));
    if (blockIdx.x >= before && blockIdx.x < before + items) {
      const unsigned long long first = bg + gg - groups;
      found = make_item(a, pl, part, tpt, s, q, x, splits, (uint32_t)(blockIdx.x - before),
                        (uint32_t)first, (uint32_t)(first >> 32), true);
      have = 1;
    }
  }
  __syncthreads();
  if (blockIdx.x == 0 && tid == 0) *part.n_groups = n_groups;
  if (!have) return false;
  *out = found;
  return true;
}

template <typename T>
__device__ __forceinline__ bool any_nonfinite(uint32_t w) {
  constexpr uint32_t m = Elem<T>::kExpMask;
  return (w & m) == m || (w & (m << 16)) == (m << 16);
}

// A pair of elements with what is not finite replaced by 0.
template <typename T>
__device__ __forceinline__ uint32_t finite_only(uint32_t w) {
  constexpr uint32_t m = Elem<T>::kExpMask;
  if ((w & m) == m) w &= 0xffff0000u;
  if ((w & (m << 16)) == (m << 16)) w &= 0xffffu;
  return w;
}

template <typename T>
__device__ __forceinline__ void store_out(const AttnArgs& a, int row, int head, int d, float x,
                                          float y) {
  const int64_t at = row * a.o_row + head * a.o_head + d;
  if (a.out_f32)
    *reinterpret_cast<float2*>(static_cast<float*>(a.out) + at) = make_float2(x, y);
  else
    *reinterpret_cast<uint32_t*>(static_cast<T*>(a.out) + at) = Elem<T>::pack(x, y);
}

// Grid bound of one kind of tiles: unsplit tiles, and at most plan.slots() splits.
inline int64_t grid_bound(const AttnArgs& a, const Plan& pl, int64_t tiles) {
  const int64_t units = (int64_t)a.b.max_kv / pl.unit + 1;
  return std::min(tiles + (units > pl.min_units ? pl.slots() : 0), tiles * units);
}

// The tile kernel (paged_attn_tc.cu).  pdl: launched while attn_rows_kernel, on
// the same stream, still runs; it ends after it.
cudaError_t launch_attn_tiles(AttnArgs a, int dtype, int hd, bool pdl, cudaStream_t st);

}  // namespace paged
}  // namespace gb
