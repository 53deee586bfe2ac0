// sample.cu -- one token per row of logits under temperature, top-k, top-p and
// min-p, drawn with a given uniform number (gb_sample).
//
// A thread-block cluster takes a row: each CTA loads its share of the logits
// into shared memory once (the only pass over HBM), and everything after that
// works on shared memory, with the CTAs' results exchanged through distributed
// shared memory.  No workspace, one launch.
//
// The kept set is a prefix of the tokens in order (falling logit, rising id).
// The short way, for a filtered row:
//   1. a histogram, bins of 1/32 of a nat of the scaled logits on an absolute grid
//      (so that it needs no common maximum), tells from which bin on no token can be
//      kept: of counts, or, where top-p is over the whole row, of masses (a token's
//      weight relative to its bin's largest in 16 bits), whose sums give the row's
//      total weight to some 2^-15 as well;
//   2. the candidates before that bin, when they are at most kCand, go to the
//      cluster's first CTA, which sorts them, applies the filters exactly,
//      sorts the kept ones by id and draws (unless top-p's cut lies so near a border
//      that the total does not decide it).
// The middle way, for top-p over many tokens: the mass histogram gives a window of a
// bin or less for the cut, one pass sums the exact weights (for the cut and for the
// draw), and the first CTA looks for the cut among the window's tokens.
// The long way, for what remains: each filter is the search for the element at
// which a running sum -- of ones for top-k, of weights for top-p -- reaches a
// target, by histograms of 1024 bins (the second and later ones over the bits
// of the logits, down to a single value, where equal logits go by id); then all
// kept weights are summed in order of id.  An unfiltered row takes that last
// step alone.
//
// Measured, f32 rows of 201088: 15 us for one row with all filters, 35 where top-p
// keeps thousands; 128 rows 82 and 205 us, without filters 85, greedy 49 (2.1 TB/s).
// The rows are bound by instructions between some ten cluster barriers, not by memory:
// two CTAs of 113 KB on an SM take turns at loading and computing.
//
// Weights are e^z 2^45, z = (x - max) / T <= 0, rounded to integers: their sums
// are exact, so neither the order of the sums nor that of the atomics matters.
// e^z is evaluated in double precision by table and polynomial (Tang's method):
// z = n ln2 / 32 + r, |r| <= ln2 / 64, e^z = 2^(n div 32) 2^((n mod 32) / 32) P(r)
// with P the Taylor series to r^5 (the next term is below 2^-48, an eighth of the
// largest weight's resolution).
#include <cooperative_groups.h>

#include "common.cuh"
#include "moe_internal.h"
#include "ptx.cuh"

namespace gb {
namespace samp {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;      // portable
constexpr int kBins = 1024;
constexpr int kList = 512;          // elements of a bin resolved in one step
constexpr int kCand = 1024;         // candidates sorted by one CTA: two per thread
constexpr float kGrid = 32.0f;      // bins per nat
constexpr float kStep = 1.4426950408889634f / kGrid;  // a bin in powers of two
// Masses: a token's weight relative to its bin's largest, in units of 2^-16, so that a
// slice of at most 50000 tokens stays below 2^32.
constexpr float kUnit = 65536.0f;
constexpr unsigned kLeastMass = 63500;  // no mass is below: e^-1/32 2^16 = 63520, less the roundings
constexpr int kMaxVocab = 400000;   // 8 x 200 KB of shared memory
constexpr int kOneBits = 45;        // the largest weight is 2^45: 400000 of them stay below 2^64
constexpr double kNoWeight = -32.0; // e^z 2^45 rounds to 0 below -46 ln 2 = -31.9

struct Args {
  const void* logits;
  int64_t row_stride;
  int vocab, slice;  // slice: elements per CTA, a multiple of 8
  const float* u;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  int32_t* token;
  float* logprob;
};

struct Item {
  uint32_t key;
  int idx;
};

// 16-byte size: the slice lies behind it and is read as float4.
struct alignas(16) Shared {
  union {
    uint16_t count[kBins];  // the short way's histogram (a slice is below 2^16)
    uint32_t count2[kBins / 2];
    uint32_t lo[kBins];     // a bin's sum, low words (shared memory adds 32 bits natively)
    unsigned long long part[kThreads];  // weights added to the threads' parts of the slice
    Item all[kList];        // the cluster's elements of the crossing bin, once the bins are read
  };
  union {
    uint64_t cand[kCand];  // the short way's candidates: key and ~id
    struct {
      union {
        uint32_t hi[kBins];      // the bins' high words
        uint64_t weight[kList];  // of `all`
      };
      Item list[kList];  // this CTA's elements of the crossing bin
    };
  };
  double exp_table[32];
  uint64_t warp_sum[kWarps];
  float warp_sum_f[kWarps];
  uint64_t ex64[2][kMaxCluster];  // exchange slots, by parity of the exchange
  uint64_t ex64b[2][kMaxCluster];
  uint32_t ex32[2][kMaxCluster];
  uint64_t above;
  int bin, n_list, answer;
  int bin_k, bin_p, n_cand;  // the short way: bins that hold the cuts, candidates
  uint32_t key_lo, key_hi;
  float win_lo, win_hi;      // the window of cut_window, in grid units
};

static_assert(sizeof(Shared) % 16 == 0, "the slice behind Shared is read as float4");

// Logit order as unsigned order: a larger logit has the larger key.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

// The doubles nearest 2^(j / 32).
__device__ __constant__ uint64_t kExpTable[32] = {
    0x3ff0000000000000ull, 0x3ff059b0d3158574ull, 0x3ff0b5586cf9890full, 0x3ff11301d0125b51ull,
    0x3ff172b83c7d517bull, 0x3ff1d4873168b9aaull, 0x3ff2387a6e756238ull, 0x3ff29e9df51fdee1ull,
    0x3ff306fe0a31b715ull, 0x3ff371a7373aa9cbull, 0x3ff3dea64c123422ull, 0x3ff44e086061892dull,
    0x3ff4bfdad5362a27ull, 0x3ff5342b569d4f82ull, 0x3ff5ab07dd485429ull, 0x3ff6247eb03a5585ull,
    0x3ff6a09e667f3bcdull, 0x3ff71f75e8ec5f74ull, 0x3ff7a11473eb0187ull, 0x3ff82589994cce13ull,
    0x3ff8ace5422aa0dbull, 0x3ff93737b0cdc5e5ull, 0x3ff9c49182a3f090ull, 0x3ffa5503b23e255dull,
    0x3ffae89f995ad3adull, 0x3ffb7f76f2fb5e47ull, 0x3ffc199bdd85529cull, 0x3ffcb720dcef9069ull,
    0x3ffd5818dcfba487ull, 0x3ffdfc97337b9b5full, 0x3ffea4afa2a490daull, 0x3fff50765b6e4540ull};

// The integer weight of a scaled logit z <= 0 (round(e^z 2^45)); no branches, so
// that several run side by side.
__device__ __forceinline__ uint64_t weight_of(double z, const double* table) {
  constexpr double kMagic = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to an integer
  const bool none = !(z > kNoWeight);            // -inf and NaN too
  z = none ? 0.0 : z;
  const double t = fma(z, 0x1.71547652b82fep+5, kMagic);
  const int n = __double2loint(t);
  const double nd = t - kMagic;
  const double r = fma(-nd, 0x1.62e42fefa39efp-6, z);  // the constant's rounding moves z by at most 32 x 2^-53
  double p = fma(r, 1.0 / 120, 1.0 / 24);
  p = fma(p, r, 1.0 / 6);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  const double s = table[n & 31];
  const int e = (n >> 5) + kOneBits;  // -2 <= e <= 45
  const double sc = __hiloint2double(__double2hiint(s) + (e << 20), __double2loint(s));
  // + 2^52: the sum's low mantissa bits are the integer nearest to p sc
  const double w = fma(p, sc, 4503599627370496.0);
  return none ? 0 : (uint64_t)__double_as_longlong(w) & 0xfffffffffffffull;
}

__device__ __forceinline__ uint64_t shfl_xor_u64(uint64_t v, int o) {
  return __shfl_xor_sync(kFullMask, (unsigned long long)v, o);
}

// The inclusive sums of the CTA's values, two in a row per thread; total: all.
template <typename V>
__device__ __forceinline__ void block_scan2(Shared& sh, V (&v)[2], V* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  v[1] += v[0];
  V inc = v[1];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V t = __shfl_up_sync(kFullMask, inc, o);
    if (lane >= o) inc += t;
  }
  __syncthreads();
  if (lane == 31) sh.warp_sum[warp] = inc;
  __syncthreads();
  // the warps' sums, scanned by every warp for itself
  V ws = lane < kWarps ? (V)sh.warp_sum[lane] : 0;
#pragma unroll
  for (int o = 1; o < kWarps; o <<= 1) {
    const V t = __shfl_up_sync(kFullMask, ws, o);
    if (lane >= o) ws += t;
  }
  const V all = __shfl_sync(kFullMask, ws, kWarps - 1);
  const V upto = __shfl_sync(kFullMask, ws, (warp + 31) & 31);
  const V before = inc - v[1] + (warp ? upto : 0);
  v[0] += before;
  v[1] += before;
  *total = all;
}

// The grid bin of a logit: a non-decreasing function of v (each rounding is
// monotone, 0 x inf converts to 0, between the ends).
__device__ __forceinline__ int grid_of(float v, float scale) {
  const int g = __float2int_rd(v * scale);
  return max(-(1 << 28), min(1 << 28, g));
}

// The mass of a logit in its grid bin (-inf has none, also where 0 x inf puts it in a bin:
// the callers leave it out).
__device__ __forceinline__ uint32_t mass_of(float v, float scale, int bin) {
  const float frac = fminf(fmaxf(v * scale - (float)bin, 0.0f), 1.0f);
  return (uint32_t)__float2int_rn(exp2f((frac - 1.0f) * kStep) * kUnit);
}

// The relative error of a weight of a mass histogram, and of their sums: half a unit,
// and the roundings of v * scale and of scale itself, 2^-23 of it each for v and for
// the largest logit, over 32 bins per nat.
__device__ __forceinline__ float mass_slack(float top, float scale) {
  return 1.0f / 65536.0f + (fabsf(top * scale) + (float)kBins) * (1.0f / (1 << 27));
}

// A bin's mass on the scale of all bins: 2^32 is the upper edge of bin 0.
__device__ __forceinline__ unsigned long long scaled_mass(uint64_t m, int j) {
  return (unsigned long long)((double)m * (double)(exp2f(-(float)j * kStep) * 65536.0f));
}

// The window around the cut at which the running mass reaches `want`, in grid units:
// the bin with its slack, or of a bin of many the part where the cut is as a rule
// (n tokens at random are off by half their root).  v: the bin's scaled mass, before:
// that of the bins above, count: its tokens.
__device__ __forceinline__ void set_window(Shared& sh, int bin, float count, double v, double before,
                                           double want, double all) {
  const float slack = (float)(1e-5 * all / v);
  float hi = (float)(bin + 1), lo = (float)bin;
  if (count > 900.0f) {
    const float at = hi - (float)((want - before) / v), half = 2.5f * rsqrtf(count);
    lo = at - half;
    hi = at + half;
  }
  sh.win_lo = lo - slack;
  sh.win_hi = hi + slack;
}

struct Row {
  cg::cluster_group cl;
  Shared& sh;
  const float* x;  // this CTA's slice
  int n, base;     // its length and first token id
  int rank, ranks;
  int exchanges;   // exchanges made so far
  float top;       // the largest logit
  double inv_t;
  float bin_scale;
  uint32_t cut_key;  // kept: key > cut_key, or key == cut_key and id <= cut_idx
  int cut_idx;

  __device__ __forceinline__ bool kept(uint32_t k, int idx) const {
    return k > cut_key || (k == cut_key && idx <= cut_idx);
  }
  __device__ __forceinline__ uint64_t weight(float v) const {
    const uint64_t w = weight_of(((double)v - (double)top) * inv_t, sh.exp_table);
    return v == top ? 1ull << kOneBits : w;  // also where both are +inf
  }
  // The first histogram's bin: a non-decreasing function of top - v, since each
  // rounding is monotone.  NaN (0 * inf: T near 0, or infinite) converts to 0.
  __device__ __forceinline__ int bin_of(float v) const {
    if (v == top) return 0;
    const float d = (top - v) * bin_scale;
    return d < (float)(kBins - 1) ? (int)d : d == d ? kBins - 1 : 0;
  }

  // f(logit, id) over this CTA's slice, four in flight (the slice is padded with
  // -inf to a multiple of four).
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    const int n4 = (n + 3) / 4;
#pragma unroll 2
    for (int q = threadIdx.x; q < n4; q += kThreads) {
      const float4 v = reinterpret_cast<const float4*>(x)[q];
      f(v.x, base + 4 * q);
      f(v.y, base + 4 * q + 1);
      f(v.z, base + 4 * q + 2);
      f(v.w, base + 4 * q + 3);
    }
  }

  // Every CTA's values, to be read from ex64 / ex32 / ex64b[parity] until the
  // exchange after the next one.
  __device__ __forceinline__ int exchange(uint64_t a, uint32_t b, uint64_t c = 0) {
    const int par = exchanges++ & 1;
    if (threadIdx.x < ranks) {
      Shared* o = cl.map_shared_rank(&sh, threadIdx.x);
      o->ex64[par][rank] = a;
      o->ex32[par][rank] = b;
      o->ex64b[par][rank] = c;
    }
    cl.sync();
    return par;
  }

  // The CTA's sum of v, on every thread; ends with a barrier after the write
  // and begins with one, so it may be called in a row.
  __device__ __forceinline__ uint64_t block_sum(uint64_t v) {
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) v += shfl_xor_u64(v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh.warp_sum[threadIdx.x >> 5] = v;
    __syncthreads();
    uint64_t s = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) s += sh.warp_sum[w];
    return s;
  }

  // Adds v to bin j: the carry of the low word goes to the high one.
  __device__ __forceinline__ void add_bin(int j, uint64_t v) {
    const uint32_t l = (uint32_t)v;
    const uint32_t old = atomicAdd(&sh.lo[j], l);
    const uint32_t h = (uint32_t)(v >> 32) + (old + l < old ? 1u : 0u);
    if (h) atomicAdd(&sh.hi[j], h);
  }

  // After a histogram: the cluster's bins summed (every CTA does it for
  // itself), and the first bin at which `above` + the bins so far reach
  // target.  Leaves sh.bin, sh.above (the sum before that bin).
  __device__ void find_bin(uint64_t above, uint64_t target) {
    cl.sync();  // every CTA's histogram is complete
    constexpr int kPer = kBins / kThreads;
    const int j0 = threadIdx.x * kPer;
    uint64_t v[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) v[i] = 0;
    static_assert(kPer == 2, "a thread reads two bins at once");
    uint2 l[kMaxCluster], h[kMaxCluster];
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r) {  // every load before the first is used
      l[r] = h[r] = make_uint2(0, 0);
      if (r < ranks) {
        const Shared* o = cl.map_shared_rank(&sh, r);
        l[r] = *reinterpret_cast<const uint2*>(o->lo + j0);
        h[r] = *reinterpret_cast<const uint2*>(o->hi + j0);
      }
    }
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r) {
      v[0] += (uint64_t)l[r].x | ((uint64_t)h[r].x << 32);
      v[1] += (uint64_t)l[r].y | ((uint64_t)h[r].y << 32);
    }
    uint64_t mine = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) mine += v[i];
    uint64_t inc = mine;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t t = __shfl_up_sync(kFullMask, (unsigned long long)inc, o);
      if (lane >= o) inc += t;
    }
    __syncthreads();
    if (lane == 31) sh.warp_sum[warp] = inc;
    __syncthreads();
    uint64_t before = above + inc - mine;
    for (int w = 0; w < warp; ++w) before += sh.warp_sum[w];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (before < target && target <= before + v[i]) {
        sh.bin = j0 + i;
        sh.above = before;
      }
      before += v[i];
    }
    // The target is within the sum by construction; should it not be, every
    // CTA still takes the same bin.
    if (threadIdx.x == kThreads - 1 && before < target) {
      sh.bin = kBins - 1;
      sh.above = before - v[kPer - 1];
    }
    __syncthreads();
  }

  // Clears the histogram.  No other CTA still reads it: a gather, with its
  // exchange, lies between the last find_bin and this.
  __device__ __forceinline__ void clear_bins() {
    __syncthreads();
    for (int j = threadIdx.x; j < kBins; j += kThreads) sh.lo[j] = sh.hi[j] = 0;
    __syncthreads();
  }

  // Lists the cluster's elements for which pred(key, logit, id) holds in
  // sh.all (order unspecified); their number, or -1 when they are more than
  // kList.
  template <typename P>
  __device__ int gather(P pred) {
    if (threadIdx.x == 0) sh.n_list = 0;
    __syncthreads();
    each([&](float v, int id) {
      const uint32_t k = key_of(v);
      if (pred(k, v, id)) {
        const int s = atomicAdd(&sh.n_list, 1);
        if (s < kList) sh.list[s] = Item{k, id};
      }
    });
    __syncthreads();
    const int par = exchange(0, (uint32_t)sh.n_list);
    int total = 0;
    for (int r = 0; r < ranks; ++r) total = min(total + (int)min(sh.ex32[par][r], 1u << 20), 1 << 24);
    if (total > kList) return -1;
    int at = 0;
    for (int r = 0; r < ranks; ++r) {
      const int c = (int)sh.ex32[par][r];
      const Shared* o = cl.map_shared_rank(&sh, r);
      for (int i = threadIdx.x; i < c; i += kThreads) sh.all[at + i] = o->list[i];
      at += c;
    }
    __syncthreads();
    return total;
  }

  // Of the total elements in sh.all, the one at which above + the values of
  // the elements up to it (in order) reach target becomes the new cut.
  template <bool MASS>
  __device__ void resolve(int total, uint64_t above, uint64_t target) {
    uint64_t mine = 1;
    const int t = threadIdx.x;
    if (t < total) {
      if (MASS) mine = weight(logit_of(sh.all[t].key));
      sh.weight[t] = mine;
    }
    if (t == 0) {
      sh.key_lo = 0;
      sh.answer = 0x7fffffff;
    }
    __syncthreads();
    if (t < total) {
      const Item me = sh.all[t];
      uint64_t before = above;
      for (int i = 0; i < total; ++i) {
        const Item o = sh.all[i];
        if (o.key > me.key || (o.key == me.key && o.idx < me.idx)) before += sh.weight[i];
      }
      if (before < target && target <= before + mine) {
        sh.key_lo = me.key;
        sh.answer = me.idx;
      }
    }
    __syncthreads();
    cut_key = sh.key_lo;
    cut_idx = sh.answer;
  }

  // The need-th (from 1) of the kept elements with key k, by id, becomes the cut.
  __device__ void cut_tie(uint32_t k, uint64_t need) {
    // a warp counts a contiguous part, so that the parts are in order of id
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int seg = ((n + kWarps - 1) / kWarps + 31) / 32 * 32;
    const int a = min(warp * seg, n), e = min(a + seg, n);
    uint32_t c = 0;
    for (int i = a + lane; i < e; i += 32) c += key_of(x[i]) == k && kept(k, base + i);
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) c += __shfl_xor_sync(kFullMask, c, o);
    __syncthreads();
    if (lane == 0) sh.warp_sum[warp] = c;
    __syncthreads();
    uint64_t mine = 0;
    for (int w = 0; w < kWarps; ++w) mine += sh.warp_sum[w];
    int par = exchange(mine, 0);
    uint64_t before = 0;
    for (int r = 0; r < rank; ++r) before += sh.ex64[par][r];
    if (threadIdx.x == 0) sh.answer = -1;
    __syncthreads();
    for (int w = 0; w < warp; ++w) before += sh.warp_sum[w];
    if (before < need && need <= before + c) {  // the same on the whole warp
      for (int i0 = a; i0 < e; i0 += 32) {
        const int i = i0 + lane;
        const bool hit = i < e && key_of(x[i]) == k && kept(k, base + i);
        const unsigned m = __ballot_sync(kFullMask, hit);
        if (hit && before + __popc(m & ((2u << lane) - 1)) == need) sh.answer = base + i;
        before += __popc(m);
      }
    }
    __syncthreads();
    par = exchange(0, (uint32_t)(sh.answer + 1));
    int got = 0;
    for (int r = 0; r < ranks; ++r) got = max(got, (int)sh.ex32[par][r]);
    cut_key = k;
    cut_idx = got - 1;
  }

  // The first histogram is in place (bins of bin_of over the kept elements):
  // narrows the cut to the element at which the running sum reaches target.
  template <bool MASS>
  __device__ void select(uint64_t target) {
    find_bin(0, target);
    uint64_t above = sh.above;
    const int j = sh.bin;
    int total = gather([&](uint32_t k, float v, int id) { return kept(k, id) && bin_of(v) == j; });
    if (total >= 0) {
      resolve<MASS>(total, above, target);
      return;
    }
    // the bin's span of keys
    uint32_t lo = 0xffffffffu, hi = 0;
    each([&](float v, int id) {
      const uint32_t k = key_of(v);
      if (kept(k, id) && bin_of(v) == j) {
        lo = min(lo, k);
        hi = max(hi, k);
      }
    });
    lo = __reduce_min_sync(kFullMask, lo);
    hi = __reduce_max_sync(kFullMask, hi);
    if (threadIdx.x == 0) {
      sh.key_lo = 0xffffffffu;
      sh.key_hi = 0;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) {
      atomicMin(&sh.key_lo, lo);
      atomicMax(&sh.key_hi, hi);
    }
    __syncthreads();
    const int par = exchange(((uint64_t)sh.key_lo << 32) | sh.key_hi, 0);
    lo = 0xffffffffu;
    hi = 0;
    for (int r = 0; r < ranks; ++r) {
      lo = min(lo, (uint32_t)(sh.ex64[par][r] >> 32));
      hi = max(hi, (uint32_t)sh.ex64[par][r]);
    }
    // at most four rounds: each divides the span by 1024
    while (lo < hi) {
      int shift = 0;
      while (((hi - lo) >> shift) >= (uint32_t)kBins) ++shift;
      clear_bins();
      each([&](float v, int id) {
        const uint32_t k = key_of(v);
        if (k >= lo && k <= hi && kept(k, id)) {
          const uint64_t w = MASS ? weight(v) : 1;
          if (w) add_bin((int)((hi - k) >> shift), w);
        }
      });
      find_bin(above, target);
      above = sh.above;
      const uint32_t nh = hi - (min((uint32_t)sh.bin, (hi - lo) >> shift) << shift);
      const uint32_t width = (1u << shift) - 1;
      lo = nh - lo > width ? nh - width : lo;
      hi = nh;
      total = gather([&](uint32_t k, float, int id) { return k >= lo && k <= hi && kept(k, id); });
      if (total >= 0) {
        resolve<MASS>(total, above, target);
        return;
      }
    }
    uint64_t need = target - above;
    if (MASS) {
      const uint64_t w = weight(logit_of(lo));
      need = w ? (need + w - 1) / w : 1;  // w > 0: the bin crossed the target
    }
    cut_tie(lo, need);
  }

  // The window of top-p's cut over the tokens that top-k kept, by a mass histogram.
  __device__ bool find_window(float p, float scale) {
    const int tid = threadIdx.x, top_bin = grid_of(top, scale);
    __syncthreads();
    for (int j = tid; j < kBins; j += kThreads) sh.lo[j] = 0;
    if (tid == 0) sh.win_hi = -INFINITY;
    __syncthreads();
    each([&](float v, int id) {
      const int b = grid_of(v, scale), j = top_bin - b;
      if (j < kBins && v > -INFINITY && kept(key_of(v), id)) atomicAdd(&sh.lo[j], mass_of(v, scale, b));
    });
    cl.sync();
    const int j0 = 2 * tid;
    uint64_t m[2] = {0, 0};
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r)
      if (r < ranks) {
        const uint2 got = *reinterpret_cast<const uint2*>(cl.map_shared_rank(&sh, r)->lo + j0);
        m[0] += got.x;
        m[1] += got.y;
      }
    unsigned long long v[2], inc[2], all;
#pragma unroll
    for (int e = 0; e < 2; ++e) v[e] = inc[e] = scaled_mass(m[e], j0 + e);
    block_scan2(sh, inc, &all);
    const double want = (double)p * (double)all;
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if ((double)(inc[e] - v[e]) < want && want <= (double)inc[e])
        set_window(sh, top_bin - (j0 + e), (float)m[e] / kUnit, (double)v[e], (double)(inc[e] - v[e]), want,
                   (double)all);
    __syncthreads();
    return sh.win_hi > -INFINITY;
  }

  // Top-p's cut over the kept tokens with one exact pass (the middle way): sums the
  // exact weights of all and of those before the window, and lists the window's tokens
  // for the first CTA, which finds the cut among them.  The exact sums show whether the
  // cut lies in the window: when it does not (or the window's tokens are too many),
  // false, and nothing has changed.  mine: the weight, of at least min_w each, of the
  // tokens kept in the slice's part [i0, i1) that this thread sums for the draw.
  __device__ bool cut_window(float p, float scale, int part, int i0, int i1, uint64_t min_w, uint64_t& mine) {
    const int tid = threadIdx.x;
    const float win_lo = sh.win_lo, win_hi = sh.win_hi;
    if (tid == 0) sh.n_list = 0;
    __syncthreads();
    uint64_t sum = 0, above = 0, draw = 0;
#pragma unroll 4
    for (int i = i0; i < i1; ++i) {
      const float v = x[i];
      const uint32_t k = key_of(v);
      const bool in = kept(k, base + i);
      const uint64_t w = in ? weight(v) : 0;
      const float y = v * scale;
      sum += w;
      above += y > win_hi ? w : 0;
      draw += y > win_hi && w >= min_w ? w : 0;
      if (in && y <= win_hi && y >= win_lo) {
        const int s = atomicAdd(&sh.n_list, 1);
        if (s < kCand) sh.cand[s] = ((uint64_t)k << 32) | (uint32_t)~(base + i);
      }
    }
    sum = block_sum(sum);
    above = block_sum(above);
    int par = exchange(sum, (uint32_t)sh.n_list, above);
    uint64_t total = 0;
    above = 0;
    int count = 0, before_me = 0;
    for (int r = 0; r < ranks; ++r) {
      total += sh.ex64[par][r];
      above += sh.ex64b[par][r];
      if (r < rank) before_me += (int)sh.ex32[par][r];
      count += (int)sh.ex32[par][r];
    }
    const double ceiled = ceil((double)p * (double)total);
    uint64_t target = (uint64_t)ceiled;
    target = target < 1 ? 1 : target > total ? total : target;
    if (above >= target || count > kCand) return false;
    const int n_mine = sh.n_list;
    if (rank != 0) {
      Shared* o = cl.map_shared_rank(&sh, 0);
      for (int i = tid; i < n_mine; i += kThreads) o->cand[before_me + i] = sh.cand[i];
    }
    cl.sync();
    uint64_t answer = 0;
    uint32_t found = 0;
    if (rank == 0) found = find_cut(count, above, target, answer);
    par = exchange(answer, found);
    if (!sh.ex32[par][0]) return false;
    cut_key = (uint32_t)(sh.ex64[par][0] >> 32);
    cut_idx = (int)(uint32_t)sh.ex64[par][0];
    // the window's kept tokens, to the threads whose parts they are of
    sh.part[tid] = 0;
    __syncthreads();
    for (int i = tid; i < n_mine; i += kThreads) {
      const uint32_t k = (uint32_t)(sh.cand[i] >> 32);
      const int id = (int)~(uint32_t)sh.cand[i];
      if (kept(k, id)) {
        const uint64_t w = weight(logit_of(k));
        if (w >= min_w) atomicAdd(&sh.part[(id - base) / part], (unsigned long long)w);
      }
    }
    __syncthreads();
    mine = draw + sh.part[tid];
    return true;
  }

  // Of the n tokens in sh.cand, the one at which above + the weights up to it (in
  // order) reach target: its key and id in answer.  0: they do not.
  __device__ uint32_t find_cut(int n, uint64_t above, uint64_t target, uint64_t& answer) {
    uint32_t key[2] = {0, 0}, id[2] = {0, 0};
    uint64_t w[2] = {0, 0};
    uint32_t lo = 0xffffffffu, hi = 0;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = threadIdx.x + e * kThreads;
      if (i < n) {
        key[e] = (uint32_t)(sh.cand[i] >> 32);
        id[e] = ~(uint32_t)sh.cand[i];
        w[e] = weight(logit_of(key[e]));
        lo = min(lo, key[e]);
        hi = max(hi, key[e]);
      }
    }
    if (above + block_sum(w[0] + w[1]) < target) return 0;
    lo = __reduce_min_sync(kFullMask, lo);
    hi = __reduce_max_sync(kFullMask, hi);
    if (threadIdx.x == 0) {
      sh.key_lo = 0xffffffffu;
      sh.key_hi = 0;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) {
      atomicMin(&sh.key_lo, lo);
      atomicMax(&sh.key_hi, hi);
    }
    __syncthreads();
    lo = sh.key_lo;
    hi = sh.key_hi;
    // The largest key from which on the weights reach the target, by histograms of
    // kThreads bins over the keys' span, a bin per thread: low words, then high words.
    while (lo < hi) {
      int shift = 0;
      while (((hi - lo) >> shift) >= (uint32_t)kThreads) ++shift;
      sh.lo[threadIdx.x] = sh.lo[kThreads + threadIdx.x] = 0;
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (w[e] && key[e] >= lo && key[e] <= hi) {
          const int j = (hi - key[e]) >> shift;
          const uint32_t l = (uint32_t)w[e], old = atomicAdd(&sh.lo[j], l);
          const uint32_t h = (uint32_t)(w[e] >> 32) + (old + l < old ? 1u : 0u);
          if (h) atomicAdd(&sh.lo[kThreads + j], h);
        }
      __syncthreads();
      const uint64_t v = (uint64_t)sh.lo[threadIdx.x] | ((uint64_t)sh.lo[kThreads + threadIdx.x] << 32);
      unsigned long long inc[2] = {v, 0}, all;
      block_scan2(sh, inc, &all);
      const uint64_t before = above + inc[0] - v;
      if (before < target && target <= before + v) {  // one thread
        sh.bin = threadIdx.x;
        sh.above = before;
      }
      __syncthreads();
      const uint32_t edge = hi - ((uint32_t)sh.bin << shift), width = (1u << shift) - 1;
      above = sh.above;
      lo = edge - lo > width ? edge - width : lo;
      hi = edge;
    }
    // equal logits, by id: each weighs the same
    const uint64_t one = weight(logit_of(lo));
    const uint64_t need = (target - above + one - 1) / one;  // one > 0: they reach the target
    const bool is0 = key[0] == lo && threadIdx.x < n, is1 = key[1] == lo && threadIdx.x + kThreads < n;
    uint32_t first = 0, last = 0x7fffffffu;
    const uint64_t same = block_sum(((uint64_t)is0 + is1) << 40 | (is0 ? id[0] : 0) + (is1 ? id[1] : 0));
    if (same >> 40 == 1) {
      first = (uint32_t)same;  // the only one
    } else {
      while (first < last) {
        const uint32_t mid = first + (last - first) / 2;
        if (block_sum((uint64_t)(is0 && id[0] <= mid) + (is1 && id[1] <= mid)) >= need) last = mid;
        else first = mid + 1;
      }
    }
    answer = ((uint64_t)lo << 32) | first;
    return 1;
  }
};

// ---- the short way -----------------------------------------------------------

struct Settings {
  bool use_k, use_p, use_min;
  int k;
  float p, least;
};

// Descending bitonic sort of a[0, m), m a power of two of at most 2 kThreads.
__device__ __forceinline__ void sort_desc(uint64_t* a, int m) {
  for (int size = 2; size <= m; size <<= 1)
    for (int d = size >> 1; d >= 1; d >>= 1) {
      // pairs of one warp stay within its 64 elements for d <= 32
      if (d >= 32 || d == size >> 1) __syncthreads();
      else __syncwarp();
      const int t = threadIdx.x;
      if (t < m / 2) {
        const int i = (t / d) * 2 * d + (t & (d - 1)), j = i + d;
        const uint64_t x = a[i], y = a[j];
        if ((x < y) == ((i & size) == 0)) {
          a[i] = y;
          a[j] = x;
        }
      }
    }
  __syncthreads();
}

__device__ __forceinline__ int pow2_from(int n) { return n <= 2 ? 2 : 1 << (32 - __clz(n - 1)); }

// The same for few candidates (n <= kFew), a thread each: sums over the pairs
// instead of sorts, three barriers in all.
constexpr int kFew = 128;
__device__ bool finish_few(Row& R, const Settings& st, int n, double approx_total, double slack, bool all_min, float u,
                           int32_t* token, float* logprob) {
  Shared& sh = R.sh;
  const int t = threadIdx.x;
  uint64_t* w = sh.cand + kFew;      // weights
  uint64_t* wk = sh.cand + 2 * kFew;  // of the kept
  uint64_t me = 0, mine = 0;
  if (t < n) {
    me = sh.cand[t];
    mine = R.weight(logit_of((uint32_t)(me >> 32)));
    w[t] = mine;
  }
  if (t == 0) sh.above = 0;
  __syncthreads();
  int rank = 0;
  uint64_t before = 0;
  if (t < n) {
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
      const bool first = sh.cand[i] > me;
      rank += first;
      before += first ? w[i] : 0;
    }
    if (st.use_k && rank == min(st.k, n) - 1) sh.above = before + mine;  // the weight of the top k
  }
  __syncthreads();
  bool kept = false, maybe = false;
  if (t < n && !(st.use_k && rank >= st.k)) {
    double lo = INFINITY, hi = INFINITY;
    if (st.use_p) {
      const double z = (double)st.p * (st.use_k ? (double)sh.above : approx_total * (double)(1ull << kOneBits));
      lo = st.use_k ? z : z * (1.0 - slack);
      hi = st.use_k ? z : z * (1.0 + slack);
    }
    const bool big = !st.use_min || (double)mine >= (double)st.least * (double)(1ull << kOneBits);
    kept = rank == 0 || (big && (double)before < lo);
    maybe = rank == 0 || (big && (double)before < hi);
    // top-p must end within the candidates, unless min_p does
    if (st.use_p && !st.use_k && !all_min && kept && rank == n - 1 && (double)(before + mine) < hi) maybe = false;
  }
  if (t < n) wk[t] = kept ? mine : 0;
  if (__syncthreads_or(kept != maybe)) return false;
  if (kept) {
    uint64_t below = 0, all = 0;
    const uint32_t nid = (uint32_t)me;  // ~id
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
      const uint64_t v = wk[i];
      all += v;
      below += (uint32_t)sh.cand[i] > nid ? v : 0;
    }
    uint64_t at = (uint64_t)((double)u * (double)all);
    if (!(u < 1.0f) || at >= all) at = all - 1;
    if (below <= at && at < below + mine) {
      *token = (int)~nid;
      if (logprob) *logprob = (float)log((double)mine / (double)all);
    }
  }
  return true;
}

// The first CTA, with the candidates (every token from the first in order to
// some later one) in sh.cand: the filters and the draw.  approx_total: the
// row's weight in units of the largest, where top-p is over the whole row.
// all_min: every token that min_p keeps is among them.  false: the cut is too
// close to a border for that total.
__device__ bool finish(Row& R, const Settings& st, int n, double approx_total, double slack, bool all_min, float u,
                       int32_t* token, float* logprob) {
  Shared& sh = R.sh;
  const int t = threadIdx.x;
  if (n <= kFew) return finish_few(R, st, n, approx_total, slack, all_min, u, token, logprob);
  int m = pow2_from(n);
  for (int i = n + t; i < m; i += kThreads) sh.cand[i] = 0;
  sort_desc(sh.cand, m);
  // two elements per thread, in order
  unsigned long long w[2] = {0, 0}, inc[2], all;
  const int i0 = 2 * t;
#pragma unroll
  for (int e = 0; e < 2; ++e)
    if (i0 + e < n && (!st.use_k || i0 + e < st.k))
      w[e] = R.weight(logit_of((uint32_t)(sh.cand[i0 + e] >> 32)));
  inc[0] = w[0];
  inc[1] = w[1];
  block_scan2(sh, inc, &all);
  double lo = INFINITY, hi = INFINITY;  // the weight before a kept token is below lo, if not unsure
  if (st.use_p) {
    if (st.use_k) {
      lo = hi = (double)st.p * (double)all;
    } else {
      const double z = (double)st.p * approx_total * (double)(1ull << kOneBits);
      lo = z * (1.0 - slack);
      hi = z * (1.0 + slack);
    }
  }
  const double min_w = st.use_min ? (double)st.least * (double)(1ull << kOneBits) : 0.0;
  int kept = 0, maybe = 0;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int i = i0 + e;
    if (i >= n || (st.use_k && i >= st.k)) continue;
    const double before = (double)(inc[e] - w[e]);
    const bool big = (double)w[e] >= min_w;
    kept += i == 0 || (big && before < lo);
    maybe += i == 0 || (big && before < hi);
  }
  const unsigned long long sum = (unsigned long long)R.block_sum(((uint64_t)maybe << 32) | (uint32_t)kept);
  const int c = (int)(uint32_t)sum;
  if ((int)(sum >> 32) != c) return false;
  // top-p must end within the candidates, unless min_p does
  if (st.use_p && !st.use_k && !all_min && c == n && (double)all < hi) return false;
  // the kept ones by id: descending ~id
  uint64_t item[2];
#pragma unroll
  for (int e = 0; e < 2; ++e)
    item[e] = i0 + e < c ? (sh.cand[i0 + e] << 32) | (sh.cand[i0 + e] >> 32) : 0;
  m = pow2_from(c);
  __syncthreads();
#pragma unroll
  for (int e = 0; e < 2; ++e)
    if (i0 + e < m) sh.cand[i0 + e] = item[e];
  sort_desc(sh.cand, m);
  w[0] = w[1] = 0;
#pragma unroll
  for (int e = 0; e < 2; ++e)
    if (i0 + e < c) w[e] = R.weight(logit_of((uint32_t)sh.cand[i0 + e]));
  inc[0] = w[0];
  inc[1] = w[1];
  block_scan2(sh, inc, &all);
  uint64_t at = (uint64_t)((double)u * (double)all);
  if (!(u < 1.0f) || at >= all) at = all - 1;
#pragma unroll
  for (int e = 0; e < 2; ++e)
    if (i0 + e < c && inc[e] - w[e] <= at && at < inc[e]) {
      *token = (int)~(uint32_t)(sh.cand[i0 + e] >> 32);
      if (logprob) *logprob = (float)log((double)w[e] / (double)all);
    }
  return true;
}

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }

// NaN counts as -inf; -0 becomes +0, so that equal logits have equal keys.
__device__ __forceinline__ float clean(float v) { return v == v ? v + 0.0f : -INFINITY; }

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const __grid_constant__ Args a) {
  extern __shared__ __align__(16) unsigned char smem[];
  Shared& sh = *reinterpret_cast<Shared*>(smem);
  float* xs = reinterpret_cast<float*>(smem + sizeof(Shared));
  cg::cluster_group cl = cg::this_cluster();
  const int rank = cl.block_rank(), ranks = cl.num_blocks();
  const int row = blockIdx.x / ranks;
  const int base = min(rank * a.slice, a.vocab), n = min(base + a.slice, a.vocab) - base;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  // the slice, with its largest logit
  float top = -INFINITY;
  {
    const T* src = static_cast<const T*>(a.logits) + row * a.row_stride + base;
    constexpr int kVec = 16 / sizeof(T);
    const int nv = (reinterpret_cast<uintptr_t>(src) & 15) ? 0 : n / kVec;
#pragma unroll 4
    for (int i = tid; i < nv; i += kThreads) {
      const uint4 r = ld_stream_u4(src + (int64_t)i * kVec);
      T e[kVec];
      *reinterpret_cast<uint4*>(e) = r;
#pragma unroll
      for (int j = 0; j < kVec; j += 4) {
        float4 f;
        f.x = clean(to_f32<T>(e[j]));
        f.y = clean(to_f32<T>(e[j + 1]));
        f.z = clean(to_f32<T>(e[j + 2]));
        f.w = clean(to_f32<T>(e[j + 3]));
        top = fmaxf(fmaxf(top, fmaxf(f.x, f.y)), fmaxf(f.z, f.w));
        *reinterpret_cast<float4*>(xs + i * kVec + j) = f;
      }
    }
    for (int i = nv * kVec + tid; i < n; i += kThreads) {
      const float f = clean(to_f32<T>(src[i]));
      top = fmaxf(top, f);
      xs[i] = f;
    }
  }
  for (int i = n + tid; i < (n + 3) / 4 * 4; i += kThreads) xs[i] = -INFINITY;
  const float t = a.temperature ? a.temperature[row] : 1.0f;
  Settings st;
  st.k = a.top_k ? a.top_k[row] : 0;
  st.p = a.top_p ? a.top_p[row] : 1.0f;
  st.least = a.min_p ? a.min_p[row] : 0.0f;
  const bool greedy = !(t > 0.0f) || st.k == 1 || st.p <= 0.0f || st.least > 1.0f;
  st.use_k = st.k > 0 && st.k < a.vocab;
  st.use_p = st.p < 1.0f;
  st.use_min = st.least > 0.0f;
  const bool filtered = !greedy && (st.use_k || st.use_p || st.use_min);
  float u = a.u[row];
  u = u > 0.0f ? u : 0.0f;
  for (int j = tid; j < kBins; j += kThreads) sh.lo[j] = 0;
  if (tid < 32) sh.exp_table[tid] = __longlong_as_double((long long)kExpTable[tid]);
  if (tid == 0) {
    sh.n_list = 0;
    sh.bin_k = sh.bin_p = 0x7fffffff;
    sh.win_hi = -INFINITY;
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, o));
  if (lane == 0) sh.warp_sum_f[warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sh.warp_sum_f[w]);
  Row R{cl, sh, xs, n, base, rank, ranks, 0, 0.0f, 0.0, 0.0f, 0u, 0x7fffffff};

  // The short way's histogram, from the slice's own largest logit down: of masses
  // where top-p is over the whole row, else of counts.
  const float grid = kGrid / t;
  const int my_top = grid_of(top, grid);
  const bool whole_p = filtered && st.use_p && !st.use_k;
  if (whole_p) {
    R.each([&](float v, int) {
      const int b = grid_of(v, grid), j = my_top - b;
      if (j < kBins && v > -INFINITY) atomicAdd(&sh.lo[j], mass_of(v, grid, b));
    });
  } else if (filtered) {
    R.each([&](float v, int) {
      const int b = my_top - grid_of(v, grid);
      if (b < kBins) atomicAdd(&sh.count2[b >> 1], 1u << ((b & 1) * 16));
    });
  }
  int par = R.exchange(0, __float_as_uint(top));
  for (int r = 0; r < ranks; ++r) top = fmaxf(top, __uint_as_float(sh.ex32[par][r]));
  R.top = top;

  // no token can be drawn, or the first in order is the answer
  const bool none = top == -INFINITY;
  if (none || greedy) {
    uint32_t first = 0x7fffffff;
    if (!none)
      for (int i = tid; i < n; i += kThreads)
        if (xs[i] == top) {
          first = base + i;
          break;
        }
    first = __reduce_min_sync(kFullMask, first);
    __syncthreads();
    if (lane == 0) sh.warp_sum[warp] = first;
    __syncthreads();
    for (int w = 0; w < kWarps; ++w) first = min(first, (uint32_t)sh.warp_sum[w]);
    par = R.exchange(0, first);
    for (int r = 0; r < ranks; ++r) first = min(first, sh.ex32[par][r]);
    if (rank == 0 && tid == 0) {
      a.token[row] = none ? -1 : (int)first;
      if (a.logprob) a.logprob[row] = none ? -INFINITY : 0.0f;
    }
    return;
  }
  R.inv_t = 1.0 / (double)t;
  R.bin_scale = 32.0f / t;

  const float slack = mass_slack(top, grid);
  // A grid so fine (t below 10^-37) that a bin has no number puts a logit of 0 nowhere.
  if (filtered && top < INFINITY && grid < INFINITY && (!whole_p || slack < 0.01f)) {
    const int top_bin = grid_of(top, grid);
    // the cluster's bins, two per thread, every load before the first is used
    const int j0 = 2 * tid;
    uint32_t got[2 * kMaxCluster];
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r) {
      got[2 * r] = got[2 * r + 1] = 0;
      if (r < ranks) {
        const int j = j0 - (top_bin - grid_of(__uint_as_float(sh.ex32[par][r]), grid));
        const Shared* o = cl.map_shared_rank(&sh, r);
        // bins j and j + 1: of counts, one word, or the halves of two
        if (j + 1 >= 0) {
          const int q = whole_p ? j + 1 : (j + 1) >> 1;
          got[2 * r + 1] = o->lo[q];
          if (j >= 0 && (whole_p || (j & 1))) got[2 * r] = o->lo[q - 1];
        }
      }
    }
    int upto[2];  // tokens up to the bin's end; where masses are summed, a bound of them
    double total = 0.0;
    if (whole_p) {
      uint64_t m[2] = {0, 0};
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r) {
        m[0] += got[2 * r];
        m[1] += got[2 * r + 1];
      }
      unsigned long long inc[2] = {m[0], m[1]}, all;
      block_scan2(sh, inc, &all);
#pragma unroll
      for (int e = 0; e < 2; ++e) upto[e] = (int)min(inc[e] / kLeastMass, 1ull << 24) + 1;
      unsigned long long v[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) v[e] = inc[e] = scaled_mass(m[e], j0 + e);
      block_scan2(sh, inc, &all);
      // in units of the largest weight
      total = (double)all * (double)(exp2f(((float)(top_bin + 1) - top * grid) * kStep) * (1.0f / 4294967296.0f));
      const double cut = (double)st.p * (double)all, want = cut * (1.0 + 4.0 * (double)slack);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const double before = (double)(inc[e] - v[e]);
        if (before < want && want <= (double)inc[e]) sh.bin_p = j0 + e;
        if (before < cut && cut <= (double)inc[e])
          set_window(sh, top_bin - (j0 + e), (float)m[e] / kUnit, (double)v[e], before, cut, (double)all);
      }
    } else {
      uint32_t cnt[2] = {0, 0}, inc[2], all;
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r) {
        if (r < ranks) {
          const int j = j0 - (top_bin - grid_of(__uint_as_float(sh.ex32[par][r]), grid));
          const bool odd = j & 1;
          cnt[0] += odd ? got[2 * r] >> 16 : j >= 0 ? got[2 * r + 1] & 0xffffu : 0u;
          cnt[1] += odd ? got[2 * r + 1] & 0xffffu : got[2 * r + 1] >> 16;
        }
      }
      inc[0] = cnt[0];
      inc[1] = cnt[1];
      block_scan2(sh, inc, &all);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        upto[e] = (int)inc[e];
        if (st.use_k && inc[e] - cnt[e] < (uint32_t)st.k && (uint32_t)st.k <= inc[e]) sh.bin_k = j0 + e;
      }
    }
    __syncthreads();
    // the last bin that min_p keeps a token of, with room for the roundings
    int bin_min = 0x7fffffff;
    if (st.use_min) {
      float v = top + t * logf(st.least);
      v -= 1e-6f * (fabsf(top) + fabsf(v));
      bin_min = max(0, min(1 << 28, top_bin - grid_of(v, grid) + 1));
    }
    int j = st.use_k ? sh.bin_k : whole_p ? sh.bin_p : 0x7fffffff;
    const bool all_min = st.use_min && bin_min <= j;
    if (all_min && !(st.use_k && st.use_p)) j = bin_min;
    if (j < kBins) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (j0 + e == j) sh.n_cand = upto[e];
      __syncthreads();
      const int n_cand = sh.n_cand;
      if (n_cand <= kCand) {
        const int from = top_bin - j;
        // floor(y) >= from <=> y >= from, where `from` is a float
        const bool plain = abs(from) < (1 << 24);
        const float from_f = (float)from;
        R.each([&](float v, int id) {
          if ((plain ? v * grid >= from_f : grid_of(v, grid) >= from) && v > -INFINITY) {
            const int s = atomicAdd(&sh.n_list, 1);
            if (s < kCand) sh.cand[s] = ((uint64_t)key_of(v) << 32) | (uint32_t)~id;
          }
        });
        __syncthreads();
        if (rank != 0) {  // to the first CTA
          const int mine = min(sh.n_list, kCand);
          Shared* o = cl.map_shared_rank(&sh, 0);
          if (tid == 0) sh.answer = mine ? atomicAdd(&o->n_list, mine) : 0;
          __syncthreads();
          const int at = sh.answer;
          for (int i = tid; i < mine && at + i < kCand; i += kThreads) o->cand[at + i] = sh.cand[i];
        }
        cl.sync();
        bool done = true;
        if (rank == 0)
          done = finish(R, st, min(sh.n_list, kCand), total, (double)slack, all_min, u, a.token + row,
                        a.logprob ? a.logprob + row : nullptr);
        if (!whole_p) return;  // nothing of another CTA is read any more
        par = R.exchange(0, done);
        if (sh.ex32[par][0]) return;
      }
    }
    R.exchange(0, 0);  // the counts are read no more
  }

  if (st.use_k) {
    R.clear_bins();
    R.each([&](float v, int) { atomicAdd(&sh.lo[R.bin_of(v)], 1u); });
    R.select<false>((uint64_t)st.k);
  }
  // A thread sums a contiguous part of the slice for the draw (an odd number of
  // elements: no bank conflicts), so the parts are in order of id.
  const int part = ((n + kThreads - 1) / kThreads) | 1;
  const int i0 = min(tid * part, n), i1 = min(i0 + part, n);
  // weights are whole numbers: at least `least` of the largest is at least this
  const uint64_t min_w = st.use_min ? (uint64_t)ceil((double)st.least * (double)(1ull << kOneBits)) : 0;
  uint64_t mine = 0;
  // The middle way: the window is known where top-p is over the whole row.  A window
  // says nothing of a row whose logits are infinite or whose grid is too coarse.
  bool summed = false;
  if (st.use_p && top < INFINITY && slack < 0.01f)
    summed = (st.use_k ? R.find_window(st.p, grid) : sh.win_hi > -INFINITY) &&
             R.cut_window(st.p, grid, part, i0, i1, min_w, mine);
  if (st.use_p && !summed) {
    R.clear_bins();
    // Tokens that even together weigh less than (1 - p) of the largest cannot
    // hold the crossing: they count into the total alone.
    const double skip = 0.999 * (1.0 - (double)st.p) * (double)(1ull << kOneBits) / a.vocab;
    const uint64_t floor_w = (uint64_t)skip;
    uint64_t sum = 0;
    R.each([&](float v, int id) {
      const uint64_t w = R.kept(key_of(v), id) ? R.weight(v) : 0;
      sum += w;
      if (w > floor_w) R.add_bin(R.bin_of(v), w);
    });
    sum = R.block_sum(sum);
    par = R.exchange(sum, 0);
    uint64_t total = 0;
    for (int r = 0; r < ranks; ++r) total += sh.ex64[par][r];
    const double want = ceil((double)st.p * (double)total);
    uint64_t target = (uint64_t)want;
    target = target < 1 ? 1 : target > total ? total : target;
    R.select<true>(target);
  }

  // The draw.
  // the scaled logit below which min_p surely drops a token
  const double z_min = st.use_min ? log((double)st.least) - 1e-6 : -INFINITY;
  auto final_weight = [&](int i) -> uint64_t {
    const float v = xs[i];
    if (!filtered) return R.weight(v);
    if (!R.kept(key_of(v), base + i)) return 0;
    if (v != top && ((double)v - (double)top) * R.inv_t < z_min) return 0;
    const uint64_t w = R.weight(v);
    return w >= min_w ? w : 0;
  };
  if (summed) {
    // cut_window has done it
  } else if (filtered) {
#pragma unroll 2
    for (int i = i0; i < i1; ++i) mine += final_weight(i);
  } else {
#pragma unroll 4
    for (int i = i0; i < i1; ++i) mine += R.weight(xs[i]);
  }
  uint64_t inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t v = __shfl_up_sync(kFullMask, (unsigned long long)inc, o);
    if (lane >= o) inc += v;
  }
  __syncthreads();
  if (lane == 31) sh.warp_sum[warp] = inc;
  __syncthreads();
  uint64_t before = inc - mine, slice_sum = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += sh.warp_sum[w];
    slice_sum += sh.warp_sum[w];
  }
  par = R.exchange(slice_sum, 0);
  uint64_t total = 0;
  for (int r = 0; r < ranks; ++r) {
    if (r < rank) before += sh.ex64[par][r];
    total += sh.ex64[par][r];
  }
  uint64_t at = (uint64_t)((double)u * (double)total);  // cumulative > u total <=> cumulative > at
  if (!(u < 1.0f) || at >= total) at = total - 1;
  const bool owner = before <= at && at < before + mine;
  const unsigned owners = __ballot_sync(kFullMask, owner);
  if (owners) {  // the owner's part again, by its warp
    const int o = __ffs(owners) - 1;
    const int b0 = __shfl_sync(kFullMask, i0, o), b1 = __shfl_sync(kFullMask, i1, o);
    uint64_t run = __shfl_sync(kFullMask, (unsigned long long)before, o);
    for (int c = b0; c < b1; c += 32) {
      const int i = c + lane;
      const uint64_t w = i < b1 ? final_weight(i) : 0;
      uint64_t s = w;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const uint64_t v = __shfl_up_sync(kFullMask, (unsigned long long)s, d);
        if (lane >= d) s += v;
      }
      if (run + s - w <= at && at < run + s) {
        a.token[row] = base + i;
        if (a.logprob) a.logprob[row] = (float)log((double)w / (double)total);
      }
      run += __shfl_sync(kFullMask, (unsigned long long)s, 31);
    }
  }
  cl.sync();  // no CTA leaves while another may read its shared memory
}

template <typename T>
cudaError_t launch(Args a, int rows, cudaStream_t st) {
  // Eight CTAs for a long row; fewer for a short one, a slice of at least
  // 2048 logits each.
  int c = kMaxCluster;
  while (c > 1 && a.vocab <= 2048 * (c / 2)) c /= 2;
  a.slice = ((a.vocab + c - 1) / c + 7) / 8 * 8;
  const size_t smem = sizeof(Shared) + (size_t)a.slice * sizeof(float);
  auto kern = sample_kernel<T>;
  cudaError_t e = set_smem_limit(kern, sizeof(Shared) + ((size_t)kMaxVocab / kMaxCluster + 8) * sizeof(float));
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(rows * c));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)c;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, a);
}

}  // namespace samp
}  // namespace gb

extern "C" int gb_sample(const gb_sample_args* args, void* stream) {
  using namespace gb;
  if (!args) return set_error(GB_ERR_INVALID_ARG, "args is null");
  if (args->struct_size != sizeof(gb_sample_args))
    return set_error(GB_ERR_INVALID_ARG, "gb_sample_args: struct_size %u, expected %zu",
                     args->struct_size, sizeof(gb_sample_args));
  const int dt = args->dtype;
  if (dt != GB_DTYPE_F32 && dt != GB_DTYPE_BF16 && dt != GB_DTYPE_F16)
    return set_error(GB_ERR_INVALID_ARG, "unknown dtype %d", dt);
  if (args->rows < 0 || args->rows > (1 << 24))
    return set_error(GB_ERR_INVALID_ARG, "rows %d not in 0..2^24", args->rows);
  if (args->vocab < 1) return set_error(GB_ERR_INVALID_ARG, "vocab %d < 1", args->vocab);
  if (args->vocab > samp::kMaxVocab)
    return set_error(GB_ERR_UNSUPPORTED, "vocab %d above %d", args->vocab, samp::kMaxVocab);
  if (args->rows > 1 && args->row_stride < args->vocab)
    return set_error(GB_ERR_INVALID_ARG, "row_stride %lld < vocab %d", (long long)args->row_stride,
                     args->vocab);
  if (args->rows == 0) return GB_OK;
  if (!args->logits_dev || !args->u_dev || !args->token_dev)
    return set_error(GB_ERR_INVALID_ARG, "logits, u and token must not be null");
  const int es = dt == GB_DTYPE_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(args->logits_dev) % es)
    return set_error(GB_ERR_INVALID_ARG, "logits must be aligned to their elements");
  samp::Args a{};
  a.logits = args->logits_dev;
  a.row_stride = args->row_stride;
  a.vocab = args->vocab;
  a.u = args->u_dev;
  a.temperature = args->temperature_dev;
  a.top_k = args->top_k_dev;
  a.top_p = args->top_p_dev;
  a.min_p = args->min_p_dev;
  a.token = args->token_dev;
  a.logprob = args->logprob_dev;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dt == GB_DTYPE_F32    ? samp::launch<float>(a, args->rows, st)
                        : dt == GB_DTYPE_BF16 ? samp::launch<__nv_bfloat16>(a, args->rows, st)
                                              : samp::launch<__half>(a, args->rows, st);
  if (e != cudaSuccess) return set_error(GB_ERR_CUDA, "sample launch: %s", cudaGetErrorString(e));
  return GB_OK;
}
