// sample.cu -- one token per row of logits under temperature, top-k, top-p and
// min-p, drawn with a given uniform number (gb_sample).
//
// A thread-block cluster takes a row: each CTA loads its share of the logits
// into shared memory once (the only pass over HBM), and everything after that
// works on shared memory, with the CTAs' results exchanged through distributed
// shared memory.  No workspace, one launch.
//
// The kept set of top-k and top-p is a prefix of the tokens in order (falling
// logit, rising id), so each filter is the search for the element at which a
// running sum -- of ones for top-k, of weights for top-p -- reaches a target:
//   1. a histogram of 1024 bins over (max - x), 1/32 of a nat of the scaled
//      logits each, finds the bin that crosses the target;
//   2. that bin's elements (tens, usually) are listed on every CTA, and each
//      thread sums what stands before its element; one of them crosses.
// A bin of more than kList elements is split again by the bits of its
// elements' keys, down to a single key, where equal logits go by id.
//
// Weights are e^z 2^45, z = (x - max) / T <= 0, rounded to integers: their sums
// are exact, so neither the order of the sums nor that of the atomics matters.
// e^z is evaluated in double precision by table and polynomial (Tang's method):
// z = n ln2 / 32 + r, |r| <= ln2 / 64, e^z = 2^(n div 32) 2^((n mod 32) / 32) P(r)
// with P the Taylor series to r^6 (the next term is below 2^-58).
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

struct Shared {
  union {
    struct {  // a bin's sum: 64 bits in two words, because shared memory adds 32 bits natively
      uint32_t lo[kBins], hi[kBins];
    };
    struct {  // after the histogram has been read (gather's exchange)
      Item all[kList];  // the cluster's elements of the crossing bin
      uint64_t weight[kList];
    };
  };
  Item list[kList];  // this CTA's elements of the crossing bin
  double exp_table[32];
  uint64_t warp_sum[kWarps];
  uint64_t ex64[2][kMaxCluster];  // exchange slots, by parity of the exchange
  uint32_t ex32[2][kMaxCluster];
  uint64_t above;
  int bin, n_list, answer;
  uint32_t key_lo, key_hi;
};

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

// The integer weight of a scaled logit z <= 0 (round(e^z 2^45)).
__device__ __forceinline__ uint64_t weight_of(double z, const double* table) {
  if (!(z > kNoWeight)) return 0;  // -inf and NaN too
  constexpr double kMagic = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to an integer
  const double t = fma(z, 0x1.71547652b82fep+5, kMagic);
  const int n = __double2loint(t);
  const double nd = t - kMagic;
  double r = fma(-nd, 0x1.62e42fef00000p-6, z);
  r = fma(-nd, 0x1.473de6af278edp-39, r);
  double p = fma(r, 1.0 / 720, 1.0 / 120);
  p = fma(p, r, 1.0 / 24);
  p = fma(p, r, 1.0 / 6);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  const double s = table[n & 31];
  const int e = (n >> 5) + kOneBits;  // -2 <= e <= 45
  const double sc = __hiloint2double(__double2hiint(s) + (e << 20), __double2loint(s));
  // + 2^52: the sum's low mantissa bits are the integer nearest to p sc
  const double w = fma(p, sc, 4503599627370496.0);
  return (uint64_t)__double_as_longlong(w) & 0xfffffffffffffull;
}

__device__ __forceinline__ uint64_t shfl_xor_u64(uint64_t v, int o) {
  return __shfl_xor_sync(kFullMask, (unsigned long long)v, o);
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
    if (v == top) return 1ull << kOneBits;  // also where both are +inf
    return weight_of(((double)v - (double)top) * inv_t, sh.exp_table);
  }
  // The first histogram's bin: a non-decreasing function of top - v, since each
  // rounding is monotone.  NaN (0 * inf: T near 0, or infinite) converts to 0.
  __device__ __forceinline__ int bin_of(float v) const {
    if (v == top) return 0;
    const float d = (top - v) * bin_scale;
    return d < (float)(kBins - 1) ? (int)d : d == d ? kBins - 1 : 0;
  }

  // Every CTA's value, to be read from ex64[parity] / ex32[parity] until the
  // exchange after the next one.
  __device__ __forceinline__ int exchange(uint64_t a, uint32_t b) {
    const int par = exchanges++ & 1;
    if (threadIdx.x < ranks) {
      Shared* o = cl.map_shared_rank(&sh, threadIdx.x);
      o->ex64[par][rank] = a;
      o->ex32[par][rank] = b;
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
    for (int r = 0; r < ranks; ++r) {
      const Shared* o = cl.map_shared_rank(&sh, r);
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        v[i] += (uint64_t)o->lo[j0 + i] | ((uint64_t)o->hi[j0 + i] << 32);
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
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const float v = x[i];
      const uint32_t k = key_of(v);
      if (pred(k, v, base + i)) {
        const int s = atomicAdd(&sh.n_list, 1);
        if (s < kList) sh.list[s] = Item{k, base + i};
      }
    }
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
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const float v = x[i];
      const uint32_t k = key_of(v);
      if (kept(k, base + i) && bin_of(v) == j) {
        lo = min(lo, k);
        hi = max(hi, k);
      }
    }
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
      for (int i = threadIdx.x; i < n; i += kThreads) {
        const float v = x[i];
        const uint32_t k = key_of(v);
        if (k >= lo && k <= hi && kept(k, base + i)) {
          const uint64_t w = MASS ? weight(v) : 1;
          if (w) add_bin((int)((hi - k) >> shift), w);
        }
      }
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
};

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
  const float t = a.temperature ? a.temperature[row] : 1.0f;
  const int k = a.top_k ? a.top_k[row] : 0;
  const float p = a.top_p ? a.top_p[row] : 1.0f;
  const float least = a.min_p ? a.min_p[row] : 0.0f;
  for (int j = tid; j < kBins; j += kThreads) sh.lo[j] = sh.hi[j] = 0;
  if (tid < 32) sh.exp_table[tid] = __longlong_as_double((long long)kExpTable[tid]);
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, o));
  if (lane == 0) sh.warp_sum[warp] = __float_as_uint(top);
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, __uint_as_float((uint32_t)sh.warp_sum[w]));
  Row R{cl, sh, xs, n, base, rank, ranks, 0, 0.0f, 0.0, 0.0f, 0u, 0x7fffffff};
  int par = R.exchange(0, __float_as_uint(top));
  for (int r = 0; r < ranks; ++r) top = fmaxf(top, __uint_as_float(sh.ex32[par][r]));
  R.top = top;

  // no token can be drawn, or the first in order is the answer
  const bool none = top == -INFINITY;
  if (none || !(t > 0.0f) || k == 1 || p <= 0.0f || least > 1.0f) {
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

  if (k > 0 && k < a.vocab) {
    for (int i = tid; i < n; i += kThreads) atomicAdd(&sh.lo[R.bin_of(xs[i])], 1u);
    R.select<false>((uint64_t)k);
    R.clear_bins();
  }
  if (p < 1.0f) {
    // Tokens that even together weigh less than (1 - p) of the largest cannot
    // hold the crossing: they count into the total alone.
    const double skip = 0.999 * (1.0 - (double)p) * (double)(1ull << kOneBits) / a.vocab;
    const uint64_t floor_w = (uint64_t)skip;
    uint64_t sum = 0;
    for (int i = tid; i < n; i += kThreads) {
      const float v = xs[i];
      if (R.kept(key_of(v), base + i)) {
        const uint64_t w = R.weight(v);
        sum += w;
        if (w > floor_w) R.add_bin(R.bin_of(v), w);
      }
    }
    sum = R.block_sum(sum);
    par = R.exchange(sum, 0);
    uint64_t total = 0;
    for (int r = 0; r < ranks; ++r) total += sh.ex64[par][r];
    const double want = ceil((double)p * (double)total);
    uint64_t target = (uint64_t)want;
    target = target < 1 ? 1 : target > total ? total : target;
    R.select<true>(target);
  }

  // The draw.  A thread sums a contiguous part of the slice (an odd number of
  // elements: no bank conflicts), so the parts are in order of id.
  const int part = ((n + kThreads - 1) / kThreads) | 1;
  const int i0 = min(tid * part, n), i1 = min(i0 + part, n);
  const double min_w = (double)least * (double)(1ull << kOneBits);
  // the scaled logit below which min_p surely drops a token
  const double z_min = least > 0.0f ? log((double)least) - 1e-6 : -INFINITY;
  auto final_weight = [&](int i) -> uint64_t {
    const float v = xs[i];
    if (!R.kept(key_of(v), base + i)) return 0;
    if (v != top && ((double)v - (double)top) * R.inv_t < z_min) return 0;
    const uint64_t w = R.weight(v);
    return (double)w >= min_w ? w : 0;
  };
  uint64_t mine = 0;
  for (int i = i0; i < i1; ++i) mine += final_weight(i);
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
  float u = a.u[row];
  u = u > 0.0f ? u : 0.0f;
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
