// paged_attn.cu -- causal attention of a ragged batch's new rows over their
// sequences' pages (gb_paged_attention).
//
//   o = sum_j e^(s_j - m) v_j / (e^(sink - m) + sum_j e^(s_j - m)),  s_j = scale (q . k_j)
//
// in one pass over K and V with a running maximum and sum.
//
// Work.  The query heads that share a KV head are rows of one tile, so each
// key is read once for all of them: kRows rows = (kRows / group) tokens x
// group heads.  A tile's keys are split over several CTAs when the batch has
// too few tiles to fill the GPU, each split writes its unnormalised sum with
// its maximum and its sum of weights, and a second kernel joins them in the
// order of the splits.  The lengths are on the device, so every CTA works out
// its own item from them (a scan over the sequences), and the grid is sized
// from the host's bounds.
#include <algorithm>

#include "paged.cuh"
#include "ptx.cuh"

namespace gb {
namespace paged {
namespace {

// 2^x by the hardware's approximation (relative error 2^-22); 2^-inf = 0.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kTargetItems = 296;              // two CTAs on each of 148 SMs
constexpr int kMaxSlots = 2 * kTargetItems;    // items of split tiles, at most (see Plan)
constexpr int kUnit = 64;                      // keys per unit of work
constexpr int kMinUnits = 2;                   // units per split, at least
constexpr int kRows = 16;                      // rows of a tile
constexpr int kThreads = 128;
constexpr int kMaxGroup = 16;                  // query heads per KV head

struct Group {  // a split tile, for the joining kernel
  int row0, tokens, g, slot0, splits;
};

struct AttnArgs {
  Batch b;
  int nh, group, window, out_f32;
  float scale;  // scale * log2 e
  const void* q;
  int64_t q_row, q_head;
  const void *k_pool, *v_pool;
  const float* sinks;
  void* out;
  int64_t o_row, o_head;
  // workspace
  int* n_groups;
  Group* groups;       // [kTargetItems]
  float2* part_ml;     // [kMaxSlots][kRows]: maximum (log2), sum
  float* part_o;       // [kMaxSlots][kRows][head_dim]
};

size_t workspace_layout(int head_dim, char* base, AttnArgs* a) {
  size_t at = 0;
  auto take = [&](size_t bytes) {
    char* p = base ? base + at : nullptr;
    at += (bytes + 255) & ~(size_t)255;
    return p;
  };
  char* n = take(sizeof(int));
  char* g = take(sizeof(Group) * kTargetItems);
  char* ml = take(sizeof(float2) * kMaxSlots * kRows);
  char* o = take(sizeof(float) * (size_t)kMaxSlots * kRows * head_dim);
  if (a) {
    a->n_groups = reinterpret_cast<int*>(n);
    a->groups = reinterpret_cast<Group*>(g);
    a->part_ml = reinterpret_cast<float2*>(ml);
    a->part_o = reinterpret_cast<float*>(o);
  }
  return at;
}

// What a CTA does: rows of `tokens` tokens from row `row0`, the first at
// position pos0, KV head g, units [u0, u1) of kUnit keys.
struct Item {
  int seq, row0, tokens, pos0, g, u0, u1;
  int slot;  // of the partial result, -1: the tile is not split
};

// Splitting.  n = the units a sequence's rows see, t = ceil(W / kTargetItems)
// units per split (W: the units of all tiles), so a sequence has ceil(n / t)
// splits.  Tiles with more than one split have n > t, hence at most W / t such
// tiles and at most 2 W / t <= kMaxSlots of their splits.
struct SeqWork {
  int tiles, units;
};
__device__ __forceinline__ int first_unit(int pos, int window) {
  return window > 0 && pos >= window ? (pos - window + 1) / kUnit : 0;
}
__device__ __forceinline__ SeqWork seq_work(const Seq& q, int tpt, int window) {
  SeqWork w{0, 0};
  w.tiles = (q.q_len + tpt - 1) / tpt;
  const int last = q.kv_len - 1;
  if (w.tiles && last >= 0)
    w.units = last / kUnit - first_unit(max(q.kv_len - q.q_len, 0), window) + 1;
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

// Finds the CTA's item; false: there is none.  Called by the whole CTA.
__device__ bool find_item(const AttnArgs& a, int tpt, Item* out) {
  __shared__ unsigned long long red[kThreads / 32];
  __shared__ unsigned long long run[kThreads / 32][2];
  __shared__ Item found;
  __shared__ int have;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Batch& b = a.b;
  Seq mine{0, 0, 0};  // of the first kThreads sequences
  unsigned long long w = 0;
  for (int s = tid; s < b.n_seqs; s += kThreads) {
    const Seq q = load_seq(b, s, blockIdx.x == 0);
    if (s == tid) mine = q;
    const SeqWork x = seq_work(q, tpt, a.window);
    w += (unsigned long long)x.tiles * x.units;
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) w += __shfl_xor_sync(kFullMask, w, o);
  if (lane == 0) red[warp] = w;
  if (tid == 0) have = 0;
  __syncthreads();
  w = 0;
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) w += red[i];
  w *= b.nkv;
  const unsigned long long t64 = (w + kTargetItems - 1) / kTargetItems;
  const int t = (int)(t64 < kMinUnits ? kMinUnits : t64 > (1u << 30) ? (1u << 30) : t64);
  // prefixes over the sequences: items (low half) and split items; split tiles
  unsigned long long base_items = 0, base_groups = 0;
  for (int s0 = 0; s0 < b.n_seqs; s0 += kThreads) {
    const int s = s0 + tid;
    Seq q{0, 0, 0};
    if (s < b.n_seqs) q = s0 ? load_seq(b, s, false) : mine;
    const SeqWork x = seq_work(q, tpt, a.window);
    const int splits = max(1, (x.units + t - 1) / t);
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
    for (int i = 0; i < kThreads / 32; ++i) {
      if (i < warp) {
        bi += run[i][0];
        bg += run[i][1];
      }
      base_items += run[i][0];
      base_groups += run[i][1];
    }
    const unsigned long long before = bi + ii - items;
    if (blockIdx.x >= before && blockIdx.x < before + items) {
      const unsigned long long j = blockIdx.x - before;
      const unsigned long long gb = bg + gg - groups;
      Item it;
      it.seq = s;
      it.g = (int)(j % b.nkv);
      const unsigned long long js = j / b.nkv;
      const int split = (int)(js % splits), tile = (int)(js / splits);
      it.row0 = q.row0 + tile * tpt;
      it.tokens = min(tpt, q.q_len - tile * tpt);
      it.pos0 = q.kv_len - q.q_len + tile * tpt;
      const int last = it.pos0 + it.tokens - 1;
      const int lo = first_unit(it.pos0, a.window);
      const int n = last < 0 ? 0 : last / kUnit - lo + 1;
      const int per = (n + splits - 1) / splits;
      it.u0 = lo + min(split * per, n);
      it.u1 = lo + min((split + 1) * per, n);
      it.slot = -1;
      if (splits > 1) {
        const int group = (int)(uint32_t)gb + tile * b.nkv + it.g;
        const int slot0 = (int)(gb >> 32) + (tile * b.nkv + it.g) * splits;
        it.slot = slot0 + split;
        if (split == 0) a.groups[group] = Group{it.row0, it.tokens, it.g, slot0, splits};
      }
      found = it;
      have = 1;
    }
  }
  if (blockIdx.x == 0 && tid == 0) *a.n_groups = (int)(uint32_t)base_groups;
  __syncthreads();
  if (!have) return false;
  *out = found;
  return true;
}

// ---- mma.sync building blocks (16 rows) --------------------------------------
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4],
                                                        uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                                 uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
// 16 bytes global -> shared; `bytes` 0 fills the destination with zeros and reads nothing.
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <typename T>
__device__ __forceinline__ bool any_nonfinite(uint32_t w) {
  constexpr uint32_t m = Elem<T>::kExpMask;
  return (w & m) == m || (w & (m << 16)) == (m << 16);
}

// Keys per warp and step; a CTA's four warps take a unit of 64.
constexpr int kStep = 16;

template <int HD>
constexpr int stages() { return HD == 64 ? 6 : HD == 128 ? 5 : 3; }
template <int HD>
constexpr int warp_bytes() { return stages<HD>() * 2 * kStep * HD * 2; }
template <int HD>
constexpr int q_bytes() { return kRows * HD * 2; }
template <int HD>
constexpr int smem_bytes() { return 4 * warp_bytes<HD>() + q_bytes<HD>(); }

template <typename T>
__device__ __forceinline__ void store_out(const AttnArgs& a, int row, int head, int d, float x,
                                          float y) {
  const int64_t at = row * a.o_row + head * a.o_head + d;
  if (a.out_f32)
    *reinterpret_cast<float2*>(static_cast<float*>(a.out) + at) = make_float2(x, y);
  else
    *reinterpret_cast<uint32_t*>(static_cast<T*>(a.out) + at) = Elem<T>::pack(x, y);
}

// A CTA per item: four warps, each with keys of its own (16 of every unit) and
// its own pipeline of cp.async stages, so no barrier stands in the loop; their
// results are joined in shared memory at the end.
template <typename T, int HD>
__global__ void __launch_bounds__(kThreads) attn_rows_kernel(const __grid_constant__ AttnArgs a) {
  extern __shared__ __align__(128) unsigned char sm[];
  constexpr int kStages = stages<HD>();
  constexpr int C = HD / 8;                 // 16-byte pieces of a row
  constexpr int kStageBytes = 2 * kStep * HD * 2;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int tpt = kRows / a.group;
  Item it;
  const bool have = find_item(a, tpt, &it);
  pdl_trigger();
  if (!have) return;
  const int n_rows = it.tokens * a.group;
  unsigned char* qs = sm + 4 * warp_bytes<HD>();
  // Q rows, piece c of row r at c ^ (r & 7): ldmatrix reads 8 rows without bank conflicts
  for (int i = tid; i < kRows * C; i += kThreads) {
    const int r = i / C, c = i % C;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (r < n_rows) {
      const int tok = r / a.group, h = it.g * a.group + r - tok * a.group;
      v = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) +
                                          (it.row0 + tok) * a.q_row + h * a.q_head + c * 8);
    }
    *reinterpret_cast<uint4*>(qs + r * HD * 2 + ((c ^ (r & 7)) << 4)) = v;
  }
  __syncthreads();
  const uint32_t qbase = smem_u32(qs);
  const uint32_t wbase = smem_u32(sm) + warp * warp_bytes<HD>();
  constexpr bool kQInRegs = HD <= 128;
  uint32_t qf[kQInRegs ? HD / 16 : 1][4];
  auto load_q = [&](int ks, uint32_t(&f)[4]) {
    const int r = lane & 15, c = ks * 2 + (lane >> 4);
    ldsm4(f, qbase + r * HD * 2 + ((c ^ (r & 7)) << 4));
  };
  if constexpr (kQInRegs) {
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) load_q(ks, qf[ks]);
  }
  // this lane's two rows
  const int r0 = lane >> 2, r1 = r0 + 8;
  const int p0 = it.pos0 + r0 / a.group, p1 = it.pos0 + r1 / a.group;
  const int window = a.window > 0 ? a.window : 0x7fffffff;
  const int last = it.pos0 + it.tokens - 1;
  const int key_lo = max(0, a.window > 0 ? it.pos0 - a.window + 1 : 0);
  // keys that every row sees lie in [all_lo, it.pos0]
  const int all_lo = max(0, a.window > 0 ? last - a.window + 1 : 0);
  float acc[HD / 8][4];
#pragma unroll
  for (int i = 0; i < HD / 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;

  const int n = it.u1 - it.u0;
  const T* kp = static_cast<const T*>(a.k_pool) + it.g * a.b.head_stride;
  const T* vp = static_cast<const T*>(a.v_pool) + it.g * a.b.head_stride;
  const int32_t* table = a.b.table + it.seq * a.b.table_stride;
  const int page_mask = (1 << a.b.page_shift) - 1;
  // the element offset of key lane & 15 of step u; -1: not to be read, -2: its page is bad
  auto key_offset = [&](int u) -> int64_t {
    const int key = (it.u0 + u) * kUnit + warp * kStep + (lane & 15);
    if (u >= n || key < key_lo || key > last) return -1;
    const int page = __ldg(table + (key >> a.b.page_shift));
    if ((unsigned)page >= (unsigned)a.b.n_pages) {
      flag(a.b, GB_PAGED_BAD_PAGE);
      return -2;
    }
    return page * a.b.page_stride + (key & page_mask) * a.b.slot_stride;
  };
  __shared__ unsigned bad_keys[4][kStages];  // of each stage, a bit per key
  auto issue = [&](int u, int64_t off) {
    const uint32_t dst = wbase + (u % kStages) * kStageBytes;
    constexpr int kRowsPer = 32 / C > 0 ? 32 / C : 1;
    const unsigned bad = __ballot_sync(kFullMask, off == -2) & 0xffffu;
    if (lane == 0) bad_keys[warp][u % kStages] = bad;
#pragma unroll
    for (int i = 0; i < kStep / kRowsPer; ++i) {
      const int r = i * kRowsPer + lane / C, c = lane % C;
      const int64_t o = __shfl_sync(kFullMask, (long long)off, r);
      const uint32_t bytes = o >= 0 ? 16u : 0u;
      const int64_t e = o >= 0 ? o + c * 8 : 0;
      const uint32_t d = dst + r * HD * 2 + ((c ^ (r & 7)) << 4);
      cp16(d, kp + e, bytes);
      cp16(d + kStep * HD * 2, vp + e, bytes);
    }
  };
#pragma unroll
  for (int u = 0; u < kStages - 1; ++u) {
    if (u < n) issue(u, key_offset(u));
    cp_commit();
  }
  int64_t next_off = key_offset(kStages - 1);
  for (int u = 0; u < n; ++u) {
    if (u + kStages - 1 < n) issue(u + kStages - 1, next_off);
    cp_commit();
    next_off = key_offset(u + kStages);
    cp_wait<kStages - 1>();
    __syncwarp();
    const uint32_t ks_ = wbase + (u % kStages) * kStageBytes, vs_ = ks_ + kStep * HD * 2;
    const int key0 = (it.u0 + u) * kUnit + warp * kStep;
    if (key0 <= last && key0 + kStep > key_lo) {  // the same on the whole warp
      float s[2][4];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = 0.0f;
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks) {
        uint32_t kf[4], qt[4];
        // keys 0-7 / 8-15, dims 0-7 / 8-15 of the step
        const int r = (lane & 7) + ((lane >> 4) << 3), c = ks * 2 + ((lane >> 3) & 1);
        ldsm4(kf, ks_ + r * HD * 2 + ((c ^ (r & 7)) << 4));
        if constexpr (kQInRegs) {
          mma16816<T>(s[0], qf[ks], kf[0], kf[1]);
          mma16816<T>(s[1], qf[ks], kf[2], kf[3]);
        } else {
          load_q(ks, qt);
          mma16816<T>(s[0], qt, kf[0], kf[1]);
          mma16816<T>(s[1], qt, kf[2], kf[3]);
        }
      }
      const unsigned bad = bad_keys[warp][u % kStages];
      const bool masked = key0 + kStep - 1 > it.pos0 || key0 < all_lo || bad;
      uint32_t seen = 0xffu;  // bit nt * 4 + j: score s[nt][j] is visible
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[nt][j] *= a.scale;
      if (masked) {
        seen = 0;
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int kk = nt * 8 + (lane & 3) * 2 + (j & 1), key = key0 + kk;
            const int p = j < 2 ? p0 : p1;
            if (key <= p && p - key < window && !((bad >> kk) & 1))
              seen |= 1u << (nt * 4 + j);
            else
              s[nt][j] = -INFINITY;
          }
      }
      float x0 = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1]));
      float x1 = fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3]));
      x0 = fmaxf(x0, __shfl_xor_sync(kFullMask, x0, 1));
      x1 = fmaxf(x1, __shfl_xor_sync(kFullMask, x1, 1));
      x0 = fmaxf(x0, __shfl_xor_sync(kFullMask, x0, 2));
      x1 = fmaxf(x1, __shfl_xor_sync(kFullMask, x1, 2));
      // The reference (a maximum less kTop) moves only when a score passes the
      // maximum by 2^6: the weights then stay below 2^(kTop + 6), which the
      // 16-bit types hold as exactly as 1.
      constexpr float kTop = Elem<T>::kTop;
      if (__any_sync(kFullMask, x0 > m0 + (kTop + 6.0f) || x1 > m1 + (kTop + 6.0f))) {
        const float n0 = fmaxf(m0, x0 - kTop), n1 = fmaxf(m1, x1 - kTop);
        const float c0 = n0 == -INFINITY ? 1.0f : ex2(m0 - n0);
        const float c1 = n1 == -INFINITY ? 1.0f : ex2(m1 - n1);
        m0 = n0;
        m1 = n1;
        l0 *= c0;
        l1 *= c1;
#pragma unroll
        for (int i = 0; i < HD / 8; ++i) {
          acc[i][0] *= c0;
          acc[i][1] *= c0;
          acc[i][2] *= c1;
          acc[i][3] *= c1;
        }
      }
      const float u0 = m0 == -INFINITY ? 0.0f : m0, u1 = m1 == -INFINITY ? 0.0f : m1;
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        s[nt][0] = ex2(s[nt][0] - u0);
        s[nt][1] = ex2(s[nt][1] - u0);
        s[nt][2] = ex2(s[nt][2] - u1);
        s[nt][3] = ex2(s[nt][3] - u1);
        l0 += s[nt][0] + s[nt][1];
        l1 += s[nt][2] + s[nt][3];
      }
      const uint32_t pf[4] = {Elem<T>::pack(s[0][0], s[0][1]), Elem<T>::pack(s[0][2], s[0][3]),
                              Elem<T>::pack(s[1][0], s[1][1]), Elem<T>::pack(s[1][2], s[1][3])};
#pragma unroll
      for (int dt = 0; dt < HD / 16; ++dt) {
        uint32_t vf[4];
        const int r = (lane & 7) + (((lane >> 3) & 1) << 3), c = dt * 2 + (lane >> 4);
        ldsm4_t(vf, vs_ + r * HD * 2 + ((c ^ (r & 7)) << 4));
        if (masked && __any_sync(kFullMask, any_nonfinite<T>(vf[0]) || any_nonfinite<T>(vf[1]) ||
                                                any_nonfinite<T>(vf[2]) || any_nonfinite<T>(vf[3]))) {
          // 0 x inf is NaN: add the visible products alone, key by key
          for (int kk = 0; kk < kStep; ++kk) {
            const int own = (lane & ~3) | ((kk & 7) >> 1), nt = kk >> 3;
            const uint32_t sb = __shfl_sync(kFullMask, seen, own) >> (nt * 4 + (kk & 1));
            const uint32_t a0 = __shfl_sync(kFullMask, pf[nt * 2], own);
            const uint32_t a1 = __shfl_sync(kFullMask, pf[nt * 2 + 1], own);
            const float2 f0 = Elem<T>::unpack(a0), f1 = Elem<T>::unpack(a1);
            const float w0 = kk & 1 ? f0.y : f0.x, w1 = kk & 1 ? f1.y : f1.x;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int col = dt * 16 + h * 8 + (lane & 3) * 2;
              const uint32_t vw = *reinterpret_cast<const uint32_t*>(
                  sm + (vs_ - smem_u32(sm)) + kk * HD * 2 + (((col >> 3) ^ (kk & 7)) << 4) +
                  (col & 7) * 2);
              const float2 v = Elem<T>::unpack(vw);
              if (sb & 1) {
                acc[dt * 2 + h][0] += w0 * v.x;
                acc[dt * 2 + h][1] += w0 * v.y;
              }
              if (sb & 4) {
                acc[dt * 2 + h][2] += w1 * v.x;
                acc[dt * 2 + h][3] += w1 * v.y;
              }
            }
          }
        } else {
          mma16816<T>(acc[dt * 2], pf, vf[0], vf[1]);
          mma16816<T>(acc[dt * 2 + 1], pf, vf[2], vf[3]);
        }
      }
    }
    __syncwarp();  // the stage is read before the next issue overwrites it
  }
  cp_wait<0>();
  l0 += __shfl_xor_sync(kFullMask, l0, 1);
  l1 += __shfl_xor_sync(kFullMask, l1, 1);
  l0 += __shfl_xor_sync(kFullMask, l0, 2);
  l1 += __shfl_xor_sync(kFullMask, l1, 2);
  // join the four warps
  __shared__ float wm[4][kRows], wl[4][kRows];
  __syncthreads();  // the stages are free
  float* os = reinterpret_cast<float*>(sm);  // [4][kRows][HD]
  if ((lane & 3) == 0) {
    wm[warp][r0] = m0;
    wm[warp][r1] = m1;
    wl[warp][r0] = l0;
    wl[warp][r1] = l1;
  }
#pragma unroll
  for (int i = 0; i < HD / 8; ++i) {
    const int d = i * 8 + (lane & 3) * 2;
    *reinterpret_cast<float2*>(os + (warp * kRows + r0) * HD + d) = make_float2(acc[i][0], acc[i][1]);
    *reinterpret_cast<float2*>(os + (warp * kRows + r1) * HD + d) = make_float2(acc[i][2], acc[i][3]);
  }
  __syncthreads();
  for (int i = tid; i < n_rows * (HD / 2); i += kThreads) {
    const int r = i / (HD / 2), d = (i % (HD / 2)) * 2;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) M = fmaxf(M, wm[w][r]);
    const int tok = r / a.group, h = it.g * a.group + r - tok * a.group;
    float sink = -INFINITY;
    if (it.slot < 0 && a.sinks) sink = a.sinks[h] * kLog2e;
    M = fmaxf(M, sink);
    float L = M == -INFINITY ? 0.0f : ex2(sink - M), x = 0.0f, y = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if (wm[w][r] == -INFINITY) continue;
      const float f = ex2(wm[w][r] - M);
      const float2 o = *reinterpret_cast<const float2*>(os + (w * kRows + r) * HD + d);
      L += wl[w][r] * f;
      x += o.x * f;
      y += o.y * f;
    }
    if (it.slot >= 0) {
      *reinterpret_cast<float2*>(a.part_o + ((int64_t)it.slot * kRows + r) * HD + d) =
          make_float2(x, y);
      if (d == 0) a.part_ml[it.slot * kRows + r] = make_float2(M, L);
    } else {
      const float inv = L == 0.0f ? 0.0f : 1.0f / L;
      store_out<T>(a, it.row0 + tok, h, d, x * inv, y * inv);
    }
  }
}

// Joins a split tile: a warp per row, its splits in order.
template <typename T, int HD>
__global__ void __launch_bounds__(kRows * 32) attn_join_kernel(const __grid_constant__ AttnArgs a) {
  pdl_wait();
  if ((int)blockIdx.x >= __ldcg(a.n_groups)) return;
  const Group g = a.groups[blockIdx.x];
  const int r = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (r >= g.tokens * a.group) return;
  const int tok = r / a.group, h = g.g * a.group + r - tok * a.group;
  const float sink = a.sinks ? a.sinks[h] * kLog2e : -INFINITY;
  float M = sink;
  for (int s = lane; s < g.splits; s += 32) M = fmaxf(M, a.part_ml[(g.slot0 + s) * kRows + r].x);
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) M = fmaxf(M, __shfl_xor_sync(kFullMask, M, o));
  float L = M == -INFINITY ? 0.0f : ex2(sink - M);
  float acc[HD / 32];
#pragma unroll
  for (int i = 0; i < HD / 32; ++i) acc[i] = 0.0f;
  for (int s = 0; s < g.splits; ++s) {
    const int64_t at = (int64_t)(g.slot0 + s) * kRows + r;
    const float2 ml = a.part_ml[at];
    if (ml.x == -INFINITY) continue;
    const float f = ex2(ml.x - M);
    L += ml.y * f;
#pragma unroll
    for (int i = 0; i < HD / 64; ++i) {
      const float2 o = *reinterpret_cast<const float2*>(a.part_o + at * HD + i * 64 + lane * 2);
      acc[2 * i] += o.x * f;
      acc[2 * i + 1] += o.y * f;
    }
  }
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
  for (int i = 0; i < HD / 64; ++i)
    store_out<T>(a, g.row0 + tok, h, i * 64 + lane * 2, acc[2 * i] * inv, acc[2 * i + 1] * inv);
}

template <typename T, int HD>
cudaError_t launch_attn(const AttnArgs& a, cudaStream_t st) {
  const int tpt = kRows / a.group;
  // tiles: a sequence's last one may be partial
  const int64_t tiles = std::min<int64_t>((int64_t)a.b.total_q / tpt + a.b.n_seqs, a.b.total_q) * a.b.nkv;
  // items (see Plan): unsplit tiles, and at most 2 kTargetItems splits
  const int64_t units = (int64_t)a.b.max_kv / kUnit + 1;
  const bool splits = units > kMinUnits;
  const int64_t grid = std::min(tiles + (splits ? kMaxSlots : 0), tiles * units);
  if (grid > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  auto kern = attn_rows_kernel<T, HD>;
  cudaError_t e = set_smem_limit(kern, smem_bytes<HD>());
  if (e != cudaSuccess) return e;
  kern<<<(unsigned)grid, kThreads, smem_bytes<HD>(), st>>>(a);
  e = cudaGetLastError();
  if (e != cudaSuccess || !splits) return e;
  return launch_pdl(attn_join_kernel<T, HD>, dim3(kTargetItems), dim3(kRows * 32), 0, st, a);
}

template <typename T>
cudaError_t launch_attn_hd(const AttnArgs& a, int hd, cudaStream_t st) {
  if (hd == 64) return launch_attn<T, 64>(a, st);
  if (hd == 128) return launch_attn<T, 128>(a, st);
  return launch_attn<T, 256>(a, st);
}

}  // namespace
}  // namespace paged
}  // namespace gb

extern "C" int gb_paged_attention_workspace(const gb_paged_batch* batch, int32_t n_heads,
                                            int64_t* bytes) {
  using namespace gb;
  using namespace gb::paged;
  if (!bytes) return set_error(GB_ERR_INVALID_ARG, "bytes is null");
  *bytes = 0;
  Batch b;
  const int rc = check_batch(batch, &b);
  if (rc) return rc;
  if (n_heads < 1 || n_heads % batch->n_kv_heads)
    return set_error(GB_ERR_INVALID_ARG, "n_heads %d is not a multiple of n_kv_heads %d", n_heads,
                     batch->n_kv_heads);
  *bytes = (int64_t)workspace_layout(batch->head_dim, nullptr, nullptr);
  return GB_OK;
}

extern "C" int gb_paged_attention(const gb_paged_batch* batch, const gb_attn_args* args,
                                  void* stream) {
  using namespace gb;
  using namespace gb::paged;
  AttnArgs a{};
  const int rc = check_batch(batch, &a.b);
  if (rc) return rc;
  if (!args) return set_error(GB_ERR_INVALID_ARG, "args is null");
  if (args->struct_size != sizeof(gb_attn_args))
    return set_error(GB_ERR_INVALID_ARG, "gb_attn_args: struct_size %u, expected %zu",
                     args->struct_size, sizeof(gb_attn_args));
  if (args->n_heads < 1 || args->n_heads % batch->n_kv_heads)
    return set_error(GB_ERR_INVALID_ARG, "n_heads %d is not a multiple of n_kv_heads %d",
                     args->n_heads, batch->n_kv_heads);
  a.group = args->n_heads / batch->n_kv_heads;
  if (a.group > kMaxGroup)
    return set_error(GB_ERR_UNSUPPORTED, "%d query heads per KV head: at most %d", a.group, kMaxGroup);
  if (args->window < 0) return set_error(GB_ERR_INVALID_ARG, "window < 0");
  if (args->out_dtype != GB_DTYPE_F32 && args->out_dtype != batch->dtype)
    return set_error(GB_ERR_UNSUPPORTED, "out_dtype %d: F32 or the pool's", args->out_dtype);
  if (!(args->scale > 0.0f) || !(args->scale < INFINITY))
    return set_error(GB_ERR_INVALID_ARG, "scale must be positive and finite");
  if (batch->n_seqs == 0 || batch->total_q == 0) return GB_OK;
  if (!args->q_dev || !args->out_dev || !args->k_pool_dev || !args->v_pool_dev || !args->workspace_dev)
    return set_error(GB_ERR_INVALID_ARG, "q, out, the pools and the workspace must not be null");
  const int64_t os = args->out_dtype == GB_DTYPE_F32 ? 4 : 2;
  if (!aligned16(args->q_dev) || !aligned16(args->out_dev) || !aligned16(args->k_pool_dev) ||
      !aligned16(args->v_pool_dev) || !stride_ok(args->q_row_stride, 2) ||
      !stride_ok(args->q_head_stride, 2) || !stride_ok(args->out_row_stride, os) ||
      !stride_ok(args->out_head_stride, os))
    return set_error(GB_ERR_INVALID_ARG,
                     "buffers must be 16-byte aligned, strides non-negative multiples of 16 bytes");
  if (args->out_dev == args->q_dev) return set_error(GB_ERR_INVALID_ARG, "out must not be q");
  if (reinterpret_cast<uintptr_t>(args->workspace_dev) & 255)
    return set_error(GB_ERR_INVALID_ARG, "the workspace must be 256-byte aligned");
  const int64_t need = (int64_t)workspace_layout(batch->head_dim, nullptr, nullptr);
  if (args->workspace_bytes < need)
    return set_error(GB_ERR_INVALID_ARG, "workspace of %lld bytes, %lld needed",
                     (long long)args->workspace_bytes, (long long)need);
  workspace_layout(batch->head_dim, static_cast<char*>(args->workspace_dev), &a);
  a.nh = args->n_heads;
  a.window = args->window;
  a.out_f32 = args->out_dtype == GB_DTYPE_F32;
  a.scale = args->scale * kLog2e;
  a.q = args->q_dev;
  a.q_row = args->q_row_stride, a.q_head = args->q_head_stride;
  a.k_pool = args->k_pool_dev, a.v_pool = args->v_pool_dev;
  a.sinks = args->sinks_dev;
  a.out = args->out_dev;
  a.o_row = args->out_row_stride, a.o_head = args->out_head_stride;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = batch->dtype == GB_DTYPE_BF16
                            ? launch_attn_hd<__nv_bfloat16>(a, batch->head_dim, st)
                            : launch_attn_hd<__half>(a, batch->head_dim, st);
  if (e != cudaSuccess)
    return set_error(GB_ERR_CUDA, "attention launch: %s", cudaGetErrorString(e));
  return GB_OK;
}
