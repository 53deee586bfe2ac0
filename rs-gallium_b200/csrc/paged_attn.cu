// paged_attn.cu -- causal attention of a ragged batch's new rows over their
// sequences' pages (gb_paged_attention): the kernel of decoding sequences, the
// joining kernel, and the entry points.
#include "paged_attn.cuh"

namespace gb {
namespace paged {
namespace {

constexpr int kThreads = 128;

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

// Keys per warp and step.
constexpr int kStep = 16;
constexpr int kWarps = kThreads / 32;

// Few stages for many warps: a step is a chain of some 370 instructions, and with two
// warps on each scheduler (six stages of 4 KB at head_dim 64) the chains, not the
// memory, were the bound (3.9 TB/s).
template <int HD>
constexpr int stages() { return HD == 128 ? 2 : 3; }
template <int HD>
constexpr int warp_bytes() { return stages<HD>() * 2 * kStep * HD * 2; }
// the stages, Q where registers do not hold it, and
// the join of the warps' sums
template <int HD, int HPC>
constexpr int smem_bytes() {
  return kWarps * warp_bytes<HD>() + (HD == 256 ? kRows * HD * 2 : 0) + HPC * kRows * HD * 4;
}

// Where a CTA's share begins: the units of the decoding sequences' pairs (a sequence and
// HPC of its KV heads, `pairs` per sequence) in a row, cut into equal shares of `share`
// units.
struct Share {
  int64_t begin, units;  // begin < 0: none
  int64_t share, total;
  int seq;               // of the first unit
  int64_t offset;        // of the first unit from the sequence's first
};

// The units of one of the sequence's pairs; a sequence with rows that see nothing
// has one, in which its zeros are written.
__device__ __forceinline__ int pair_units(const AttnArgs& a, const Plan& pl, const Seq& q) {
  const SeqWork x = seq_work<true>(a, pl, q, kRows / a.group);
  return x.tiles ? max(x.units, 1) : 0;
}

__device__ __forceinline__ void set_share(const AttnArgs& a, const Plan& pl, unsigned long long total,
                                          Share* sh) {
  const int64_t t = (int64_t)((total + pl.target - 1) / (unsigned)pl.target);
  sh->share = t < pl.min_units ? pl.min_units : t;
  sh->total = (int64_t)total;
  sh->begin = blockIdx.x * sh->share;
  sh->units = min(sh->share, sh->total - sh->begin);
  if (sh->units <= 0) sh->begin = -1;
}

// Up to 128 sequences each warp holds them all, one in 32 a lane (mine); else the CTA
// works out its share together and sequences are read when they are needed.
__device__ __forceinline__ Share find_share(const AttnArgs& a, const Plan& pl, int pairs, Seq (&mine)[4]) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Batch& b = a.b;
  Share sh;
  sh.seq = 0;
  sh.offset = 0;
  if (b.n_seqs <= kLaneSeqs) {
    unsigned long long w[4], upto[4], total = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      mine[i] = Seq{0, 0, 0};
      w[i] = upto[i] = 0;
      if (32 * i >= b.n_seqs) continue;
      const int s = 32 * i + lane;
      if (s < b.n_seqs) mine[i] = load_seq(b, s, blockIdx.x == 0 && warp == 0);
      w[i] = (unsigned long long)pair_units(a, pl, mine[i]) * pairs;
      upto[i] = total + warp_inclusive(w[i]);
      total = __shfl_sync(kFullMask, upto[i], 31);
    }
    set_share(a, pl, total, &sh);
    int seq = -1;
    int64_t off = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t before = (int64_t)(upto[i] - w[i]);
      if (sh.begin >= before && sh.begin < (int64_t)upto[i]) {
        seq = 32 * i + lane;
        off = sh.begin - before;
      }
    }
    const unsigned m = __ballot_sync(kFullMask, seq >= 0);
    if (m) {
      sh.seq = __shfl_sync(kFullMask, seq, __ffs(m) - 1);
      sh.offset = __shfl_sync(kFullMask, (long long)off, __ffs(m) - 1);
    }
    return sh;
  }
  __shared__ unsigned long long part[kWarps];
  __shared__ int first;
  __shared__ long long first_off;
  unsigned long long sum = 0;
  for (int s = tid; s < b.n_seqs; s += kThreads)
    sum += pair_units(a, pl, load_seq(b, s, blockIdx.x == 0));
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) sum += __shfl_xor_sync(kFullMask, sum, o);
  if (lane == 0) part[warp] = sum;
  __syncthreads();
  sum = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) sum += part[i];
  set_share(a, pl, sum * pairs, &sh);
  if (sh.begin < 0) return sh;
  unsigned long long base = 0;
  for (int s0 = 0; s0 < b.n_seqs; s0 += kThreads) {
    const int s = s0 + tid;
    const unsigned long long w =
        s < b.n_seqs ? (unsigned long long)pair_units(a, pl, load_seq(b, s, false)) * pairs : 0;
    const unsigned long long inc = warp_inclusive(w);
    __syncthreads();
    if (lane == 31) part[warp] = inc;
    __syncthreads();
    unsigned long long before = base + inc - w;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      if (i < warp) before += part[i];
      base += part[i];
    }
    if (sh.begin >= (int64_t)before && sh.begin < (int64_t)(before + w)) {
      first = s;
      first_off = sh.begin - (int64_t)before;
    }
    if ((int64_t)base > sh.begin) break;  // the same in every thread
  }
  __syncthreads();
  sh.seq = first;
  sh.offset = first_off;
  return sh;
}

// A place in the row of units.
struct Cursor {
  int seq, g, u, units, lo;  // pair of the sequence, unit of it, its units, its first key unit
  Seq q;
};

// Every CTA takes an equal share of the units of all decoding sequences, whatever
// their lengths; where it cuts a pair, both sides leave partial sums for the
// joining kernel.  Four warps, each with 16 keys of every unit of one of the pair's HPC
// heads, and its own pipeline of cp.async stages, which runs on across the pairs; the
// warps of a head join their results in shared memory at the end of each pair.
// mma.sync suits it: 16 rows fill one, and memory is the floor.  Measured with 64 query
// and 8 KV heads of 64: 64 sequences of 512 to 8192 keys 102 us, 4.3 TB/s; 256 of 2000
// 217 us, 4.8 TB/s, and 5.8 where a page's slots of a head lie together, since the rows
// of a head are 128-byte pieces a slot apart.  TMA boxes in place of cp.async were no
// faster (106 us; with the 256-byte L2 promotion, which fetches the next head too, 127).
// Two heads side by side at head_dim 128, whose rows of a slot DRAM then gives together
// (512 bytes of the [page][slot][head][dim] layout): 32 sequences of 100 to 4000 keys 51
// us against 67, 256 of 300 76 against 87, 32 of 4000 the same.  Four at 64 lost as often
// as they gained (64 sequences of 300 keys 31 us against 18, 256 of 2000 204 against 217).
template <typename T, int HD, int HPC>
__global__ void __launch_bounds__(kThreads, rows_plan<HD, HPC>().target / 148)
    attn_rows_kernel(const __grid_constant__ AttnArgs a) {
  extern __shared__ __align__(128) unsigned char sm[];
  constexpr Plan kPlan = rows_plan<HD, HPC>();
  constexpr int kStages = stages<HD>();
  constexpr int KW = kWarps / HPC;          // warps per head
  constexpr int C = HD / 8;                 // 16-byte pieces of a row
  constexpr int kStageBytes = 2 * kStep * HD * 2;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  Seq held[4];
  const int hw = warp / KW, kw = warp % KW, pairs = a.b.nkv / HPC;
  const Share share = find_share(a, kPlan, pairs, held);
  pdl_trigger();
  // the pair that begins in this share and ends in a later one, if there is one
  if (kw == 0 && lane == 0) a.rows.groups[blockIdx.x * HPC + hw].splits = 0;
  if (share.begin < 0) return;
  auto seq_at = [&](int s) -> Seq {  // the same in every lane
    if (a.b.n_seqs > kLaneSeqs) return load_seq(a.b, s, false);
    Seq q = held[0];
#pragma unroll
    for (int i = 1; i < 4; ++i)
      if ((s >> 5) == i) q = held[i];
    return Seq{__shfl_sync(kFullMask, q.row0, s & 31), __shfl_sync(kFullMask, q.q_len, s & 31),
               __shfl_sync(kFullMask, q.kv_len, s & 31)};
  };
  auto enter = [&](Cursor& c) {  // c.seq and c.q are set
    c.units = pair_units(a, kPlan, c.q);
    c.lo = first_unit(max(c.q.kv_len - c.q.q_len, 0), a.window, kPlan.unit);
  };
  auto next_pair = [&](Cursor& c) {
    c.u = 0;
    if (++c.g < pairs) return;
    c.g = 0;
    do {
      if (++c.seq >= a.b.n_seqs) return;  // past the last unit: not used
      c.q = seq_at(c.seq);
      enter(c);
    } while (!c.units);
  };
  Cursor at;
  at.seq = share.seq;
  at.q = seq_at(at.seq);
  enter(at);
  at.g = (int)(share.offset / at.units);
  at.u = (int)(share.offset - (int64_t)at.g * at.units);
  const int total = (int)share.units;

  constexpr bool kQInRegs = HD <= 128;
  unsigned char* qs = sm + kWarps * warp_bytes<HD>();
  float* os = reinterpret_cast<float*>(qs + (kQInRegs ? 0 : kRows * HD * 2)) + hw * kRows * HD;  // [kRows][HD]
  __shared__ unsigned bad_keys[kWarps][kStages];  // of each stage, a bit per key
  __shared__ float wm[kWarps][kRows], wl[kWarps][kRows];
  const uint32_t qbase = smem_u32(qs);
  const uint32_t wbase = smem_u32(sm) + warp * warp_bytes<HD>();
  const T* kp = static_cast<const T*>(a.k_pool);
  const T* vp = static_cast<const T*>(a.v_pool);
  const int page_mask = (1 << a.b.page_shift) - 1;

  // The loads run kStages - 1 steps ahead, their page numbers one more.
  Cursor ld = at;
  int looked = 0;  // steps whose pages were looked up
  // the element offset of key lane & 15 of the next step; -1: not to be read, -2: its page is bad
  auto look_up = [&]() -> int64_t {
    if (looked >= total) return -1;
    ++looked;
    const int key = (ld.lo + ld.u) * kPlan.unit + kw * kStep + (lane & 15);
    const int first = a.window > 0 ? max(0, ld.q.kv_len - ld.q.q_len - a.window + 1) : 0;
    int64_t off = -1;
    if (key >= first && key < ld.q.kv_len) {
      const int page = __ldg(a.b.table + ld.seq * a.b.table_stride + (key >> a.b.page_shift));
      if ((unsigned)page < (unsigned)a.b.n_pages) {
        off = page * a.b.page_stride + (key & page_mask) * a.b.slot_stride + (ld.g * HPC + hw) * a.b.head_stride;
      } else {
        flag(a.b, GB_PAGED_BAD_PAGE);
        off = -2;
      }
    }
    if (++ld.u == ld.units && looked < total) next_pair(ld);
    return off;
  };
  auto issue = [&](int slot, int64_t off) {
    const uint32_t dst = wbase + slot * kStageBytes;
    constexpr int kRowsPer = 32 / C;
    const unsigned bad = __ballot_sync(kFullMask, off == -2) & 0xffffu;
    if (lane == 0) bad_keys[warp][slot] = bad;
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
    const int64_t off = look_up();
    if (u < total) issue(u, off);
    cp_commit();
  }
  int64_t next_off = look_up();

  int done = 0, slot = 0, fill = kStages - 1;  // steps computed; stages of the next step and load
  while (done < total) {
    // ---- a pair, or what of it is in this share
    const int len = min(at.units - at.u, total - done);
    const int n_rows = at.q.q_len * a.group, pos0 = at.q.kv_len - at.q.q_len;
    const int last = at.q.kv_len - 1;
    const int head0 = (at.g * HPC + hw) * a.group;  // the KV head's first query head
    auto q_row = [&](int r) -> const T* {
      const int tok = r / a.group;
      return static_cast<const T*>(a.q) + (at.q.row0 + tok) * a.q_row + (head0 + r - tok * a.group) * a.q_head;
    };
    uint32_t qf[kQInRegs ? HD / 16 : 1][4];
    auto load_q = [&](int ks, uint32_t(&f)[4]) {
      const int r = lane & 15, c = ks * 2 + (lane >> 4);
      ldsm4(f, qbase + r * HD * 2 + ((c ^ (r & 7)) << 4));
    };
    if constexpr (kQInRegs) {
      // the MMA's fragments: rows lane / 4 and + 8, two columns, and the two 8 on
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = (lane >> 2) + h * 8;
        const uint32_t* src = reinterpret_cast<const uint32_t*>(q_row(r < n_rows ? r : 0)) + (lane & 3);
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks) {
          qf[ks][h] = r < n_rows ? __ldg(src + ks * 8) : 0;
          qf[ks][2 + h] = r < n_rows ? __ldg(src + ks * 8 + 4) : 0;
        }
      }
    } else {
      __syncthreads();  // the pair before is done with Q
      // piece c of row r at c ^ (r & 7): ldmatrix reads 8 rows without bank conflicts
      for (int i = tid; i < kRows * C; i += kThreads) {
        const int r = i / C, c = i % C;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (r < n_rows) v = *reinterpret_cast<const uint4*>(q_row(r) + c * 8);
        *reinterpret_cast<uint4*>(qs + r * HD * 2 + ((c ^ (r & 7)) << 4)) = v;
      }
      __syncthreads();
    }
    // this lane's two rows
    const int r0 = lane >> 2, r1 = r0 + 8;
    const int p0 = pos0 + r0 / a.group, p1 = pos0 + r1 / a.group;
    const int window = a.window > 0 ? a.window : 0x7fffffff;
    const int key_lo = max(0, a.window > 0 ? pos0 - a.window + 1 : 0);
    // keys that every row sees lie in [all_lo, pos0]
    const int all_lo = max(0, a.window > 0 ? last - a.window + 1 : 0);
    float acc[HD / 8][4];
#pragma unroll
    for (int i = 0; i < HD / 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;

    for (int k = 0; k < len; ++k) {
      // heads side by side stay in step, so that DRAM sees their rows together
      if constexpr (HPC > 1) __syncthreads();
      if (done + k + kStages - 1 < total) issue(fill, next_off);
      cp_commit();
      next_off = look_up();
      cp_wait<kStages - 1>();
      __syncwarp();
      const uint32_t ks_ = wbase + slot * kStageBytes, vs_ = ks_ + kStep * HD * 2;
      const int key0 = (at.lo + at.u + k) * kPlan.unit + kw * kStep;
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
        const unsigned bad = bad_keys[warp][slot];
        const bool masked = key0 + kStep - 1 > pos0 || key0 < all_lo || bad;
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
        // 16-bit types hold as exactly as 1.  Each row's moves by itself, so that no
        // other row has a part in its rounding.
        constexpr float kTop = Elem<T>::kTop;
        const bool moves0 = x0 > m0 + (kTop + 6.0f), moves1 = x1 > m1 + (kTop + 6.0f);
        if (__any_sync(kFullMask, moves0 || moves1)) {
          const float c0 = moves0 ? ex2(m0 - (x0 - kTop)) : 1.0f;
          const float c1 = moves1 ? ex2(m1 - (x1 - kTop)) : 1.0f;
          m0 = moves0 ? x0 - kTop : m0;
          m1 = moves1 ? x1 - kTop : m1;
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
        // P in the pool's type, as the MMA takes it beside V: half a step of that type per
        // weight, where the sums of weights keep f32.
        const uint32_t pf[4] = {Elem<T>::pack(s[0][0], s[0][1]), Elem<T>::pack(s[0][2], s[0][3]),
                                Elem<T>::pack(s[1][0], s[1][1]), Elem<T>::pack(s[1][2], s[1][3])};
#pragma unroll
        for (int dt = 0; dt < HD / 16; ++dt) {
          uint32_t vf[4];
          const int r = (lane & 7) + (((lane >> 3) & 1) << 3), c = dt * 2 + (lane >> 4);
          ldsm4_t(vf, vs_ + r * HD * 2 + ((c ^ (r & 7)) << 4));
          if (masked && __any_sync(kFullMask, any_nonfinite<T>(vf[0]) || any_nonfinite<T>(vf[1]) ||
                                                  any_nonfinite<T>(vf[2]) || any_nonfinite<T>(vf[3]))) {
            // 0 x inf is NaN: what is not finite is left out of the MMAs (whose sums round
            // the same without it) and added key by key to the rows that see it
#pragma unroll
            for (int i = 0; i < 4; ++i) vf[i] = finite_only<T>(vf[i]);
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
                constexpr uint32_t em = Elem<T>::kExpMask;
                const bool bx = (vw & em) == em, by = (vw & (em << 16)) == (em << 16);
                if (sb & 1) {
                  if (bx) acc[dt * 2 + h][0] += w0 * v.x;
                  if (by) acc[dt * 2 + h][1] += w0 * v.y;
                }
                if (sb & 4) {
                  if (bx) acc[dt * 2 + h][2] += w1 * v.x;
                  if (by) acc[dt * 2 + h][3] += w1 * v.y;
                }
              }
            }
          }
          mma16816<T>(acc[dt * 2], pf, vf[0], vf[1]);
          mma16816<T>(acc[dt * 2 + 1], pf, vf[2], vf[3]);
        }
      }
      __syncwarp();  // the stage is read before a later issue overwrites it
      fill = slot;
      slot = slot + 1 == kStages ? 0 : slot + 1;
    }
    l0 += __shfl_xor_sync(kFullMask, l0, 1);
    l1 += __shfl_xor_sync(kFullMask, l1, 1);
    l0 += __shfl_xor_sync(kFullMask, l0, 2);
    l1 += __shfl_xor_sync(kFullMask, l1, 2);
    const bool whole = len == at.units;
    // A partial result's slot: a share has at most two, in its first pair and its last.
    const int part = (2 * blockIdx.x + (done ? 1 : 0)) * HPC + hw;
    // Two elements of row r, and its statistics: a result, or a part of one.
    auto put = [&](int r, int d, float2 o, float top, float L) {
      if (!whole) {
        *reinterpret_cast<float2*>(a.rows.o + ((int64_t)part * kRows + r) * HD + d) = o;
        if (d == 0) a.rows.ml[part * kRows + r] = make_float2(top, L);
        return;
      }
      const int tok = r / a.group, h = head0 + r - tok * a.group;
      float f = 1.0f;
      if (a.sinks) {
        const float sink = a.sinks[h] * kLog2e, M = fmaxf(top, sink);
        f = part_factor(top, L, M);
        L = L * f + (M == -INFINITY ? 0.0f : ex2(sink - M));
      }
      const float inv = L == 0.0f ? 0.0f : f / L;
      store_out<T>(a, at.q.row0 + tok, h, d, o.x * inv, o.y * inv);
    };
    // ---- the head's warps' sums, added in their order
    __syncthreads();  // the pair before is read
    if ((lane & 3) == 0) {
      wm[warp][r0] = m0;
      wm[warp][r1] = m1;
      wl[warp][r0] = l0;
      wl[warp][r1] = l1;
    }
    __syncthreads();
    float M0 = -INFINITY, M1 = -INFINITY;
#pragma unroll
    for (int w = 0; w < KW; ++w) {
      M0 = fmaxf(M0, wm[hw * KW + w][r0]);
      M1 = fmaxf(M1, wm[hw * KW + w][r1]);
    }
    const float f0 = part_factor(m0, l0, M0), f1 = part_factor(m1, l1, M1);
    for (int w = 0; w < KW; ++w) {
      if (w == kw) {
#pragma unroll
        for (int i = 0; i < HD / 8; ++i) {
          const int d = i * 8 + (lane & 3) * 2;
          float2* o0 = reinterpret_cast<float2*>(os + r0 * HD + d);
          float2* o1 = reinterpret_cast<float2*>(os + r1 * HD + d);
          // a warp that saw nothing of a row adds nothing to it, not 0 x its sums
          float2 x = w ? *o0 : make_float2(0.0f, 0.0f), y = w ? *o1 : make_float2(0.0f, 0.0f);
          if (f0 != 0.0f) {
            x.x += acc[i][0] * f0;
            x.y += acc[i][1] * f0;
          }
          if (f1 != 0.0f) {
            y.x += acc[i][2] * f1;
            y.y += acc[i][3] * f1;
          }
          *o0 = x;
          *o1 = y;
        }
      }
      __syncthreads();
    }
    for (int i = kw * 32 + lane; i < n_rows * (HD / 2); i += KW * 32) {
      const int r = i / (HD / 2), d = (i % (HD / 2)) * 2;
      float M = -INFINITY, L = 0.0f;
#pragma unroll
      for (int w = 0; w < KW; ++w) M = fmaxf(M, wm[hw * KW + w][r]);
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        const float l = wl[hw * KW + w][r];
        L += l * part_factor(wm[hw * KW + w][r], l, M);
      }
      put(r, d, *reinterpret_cast<const float2*>(os + r * HD + d), M, L);
    }
    if (!whole && at.u == 0 && kw == 0 && lane == 0) {
      const int64_t end = share.begin + done + at.units - 1;  // the pair's last unit
      // sequences that share rows (q_start going back) may want more CTAs than there are
      const int last_cta = (int)min(end / share.share, (int64_t)gridDim.x - 1);
      a.rows.groups[blockIdx.x * HPC + hw] =
          Group{at.q.row0, n_rows, at.g * HPC + hw, part, 2 * (int)blockIdx.x * HPC + hw, 2 * HPC,
                last_cta - (int)blockIdx.x + 1};
    }
    done += len;
    if (done < total) next_pair(at);
  }
  cp_wait<0>();
}

// Joins the split tiles: a warp per row, its splits in order.  Both kinds of
// tiles in pieces of kRows rows, a CTA per piece in turn.
template <typename T, int HD>
__global__ void __launch_bounds__(kRows * 32) attn_join_kernel(const __grid_constant__ AttnArgs a) {
  pdl_wait();
  constexpr int kTileRows = tile_plan<HD>().tile_rows, kParts = kTileRows / kRows;
  const int n_small = a.all_tiles ? 0 : a.rows_grid * a.side;
  const int n_tiles = a.tiles.n_groups ? __ldcg(a.tiles.n_groups) : 0;
  const int lane = threadIdx.x & 31;
  for (int i = blockIdx.x; i < n_small + n_tiles * kParts; i += gridDim.x) {
    const bool small = i < n_small;
    const Partials& part = small ? a.rows : a.tiles;
    const int rows = small ? kRows : kTileRows;
    const Group g = part.groups[small ? i : (i - n_small) / kParts];
    const int r = (small ? 0 : (i - n_small) % kParts * kRows) + (threadIdx.x >> 5);
    if (!g.splits || r >= g.rows) continue;  // nothing else of g is written without splits
    const int tok = r / a.group, h = g.g * a.group + r - tok * a.group;
    // A large tile's rows are in sub-tiles of 128, each of whole tokens.
    const int per = small ? kRows : 128 / a.group * a.group;
    const int at_row = r / per * 128 + r % per;
    const float sink = a.sinks ? a.sinks[h] * kLog2e : -INFINITY;
    float M = sink;
    // row of partial result s
    auto at_part = [&](int s) -> int64_t {
      return (int64_t)(s ? g.slot1 + s * g.step : g.slot0) * rows + at_row;
    };
    float2 ml = make_float2(-INFINITY, 0.0f);  // of split `lane`, later of the chunk's
    if (lane < g.splits) ml = part.ml[at_part(lane)];
    M = fmaxf(M, ml.x);
    for (int s = lane + 32; s < g.splits; s += 32) M = fmaxf(M, part.ml[at_part(s)].x);
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) M = fmaxf(M, __shfl_xor_sync(kFullMask, M, o));
    float L = M == -INFINITY ? 0.0f : ex2(sink - M);
    float acc[HD / 32];
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) acc[i] = 0.0f;
    for (int s0 = 0; s0 < g.splits; s0 += 32) {
      if (s0) {
        ml = make_float2(-INFINITY, 0.0f);
        if (s0 + lane < g.splits) ml = part.ml[at_part(s0 + lane)];
      }
      // an empty split's sums were written as well, but its weight is 0
      const float fl = part_factor(ml.x, ml.y, M), ll = ml.y * fl;
      constexpr int kU = HD == 64 ? 16 : HD == 128 ? 8 : 4;  // splits whose loads are in flight
      const int n = min(32, g.splits - s0);
      for (int s = 0; s < n; s += kU) {
        float2 o[kU][HD / 64];
#pragma unroll
        for (int u = 0; u < kU; ++u)
#pragma unroll
          for (int i = 0; i < HD / 64; ++i)
            o[u][i] = s + u < n ? *reinterpret_cast<const float2*>(
                                      part.o + at_part(s0 + s + u) * HD + i * 64 + lane * 2)
                                : make_float2(0.0f, 0.0f);
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          const float f = __shfl_sync(kFullMask, fl, (s + u) & 31), lu = __shfl_sync(kFullMask, ll, (s + u) & 31);
          if (s + u >= n || f == 0.0f) continue;
          L += lu;
#pragma unroll
          for (int i = 0; i < HD / 64; ++i) {
            acc[2 * i] += o[u][i].x * f;
            acc[2 * i + 1] += o[u][i].y * f;
          }
        }
      }
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
    for (int i = 0; i < HD / 64; ++i)
      store_out<T>(a, g.row0 + tok, h, i * 64 + lane * 2, acc[2 * i] * inv, acc[2 * i + 1] * inv);
  }
}

size_t workspace_layout(int head_dim, char* base, AttnArgs* a) {
  size_t at = 0;
  auto take = [&](size_t bytes) {
    char* p = base ? base + at : nullptr;
    at += (bytes + 255) & ~(size_t)255;
    return p;
  };
  auto part = [&](const Plan& pl, int side, Partials* p) {
    char* n = take(sizeof(int));
    char* g = take(sizeof(Group) * pl.target * side);
    char* ml = take(sizeof(float2) * pl.slots() * side * pl.tile_rows);
    char* o = take(sizeof(float) * (size_t)pl.slots() * side * pl.tile_rows * head_dim);
    if (p)
      *p = Partials{reinterpret_cast<int*>(n), reinterpret_cast<Group*>(g),
                    reinterpret_cast<float2*>(ml), reinterpret_cast<float*>(o)};
  };
  Partials* rows = a ? &a->rows : nullptr;
  if (head_dim == 64) part(rows_plan<64, 1>(), heads_side<64>(), rows);
  else if (head_dim == 128) part(rows_plan<128, 1>(), heads_side<128>(), rows);
  else part(rows_plan<256, 1>(), heads_side<256>(), rows);
  part(head_dim == 64 ? tile_plan<64>() : head_dim == 128 ? tile_plan<128>() : tile_plan<256>(), 1,
       a ? &a->tiles : nullptr);
  return at;
}

template <typename T, int HD, int HPC>
cudaError_t launch_rows(AttnArgs& a, cudaStream_t st) {
  // shares, but no more than min_units each would make
  constexpr Plan pl = rows_plan<HD, HPC>();
  const int64_t most =
      (int64_t)std::min(a.b.n_seqs, a.b.total_q) * (a.b.nkv / HPC) * (a.b.max_kv / pl.unit + 1);
  a.rows_grid = (int)std::min<int64_t>(pl.target, (most + pl.min_units - 1) / pl.min_units);
  auto kern = attn_rows_kernel<T, HD, HPC>;
  cudaError_t e = set_smem_limit(kern, smem_bytes<HD, HPC>());
  if (e != cudaSuccess) return e;
  kern<<<(unsigned)a.rows_grid, kThreads, smem_bytes<HD, HPC>(), st>>>(a);
  return cudaGetLastError();
}

template <typename T, int HD>
cudaError_t launch_attn(AttnArgs a, int dtype, cudaStream_t st) {
  constexpr Plan tp = tile_plan<HD>();
  // Chunks: some sequence may have more than kRows rows.  Decoding sequences:
  // some may have fewer, since not all can be as long as the longest.
  const bool tiles = (int64_t)a.b.max_q * a.group > kRows;
  const int64_t least = a.b.total_q - (int64_t)(a.b.n_seqs - 1) * a.b.max_q;
  a.all_tiles = tiles && least * a.group > kRows;
  if (!tiles) a.tiles.n_groups = nullptr;
  cudaError_t e;
  if (!a.all_tiles) {
    constexpr int kSide = heads_side<HD>();
    a.side = a.b.nkv % kSide == 0 ? kSide : 1;
    e = a.side == kSide ? launch_rows<T, HD, kSide>(a, st) : launch_rows<T, HD, 1>(a, st);
    if (e != cudaSuccess) return e;
  }
  if (tiles && (e = launch_attn_tiles(a, dtype, HD, !a.all_tiles, st)) != cudaSuccess) return e;
  // One share cuts no pair; no tile is split when the longest sequence has too few keys.
  const bool join = (!a.all_tiles && a.rows_grid > 1) || (tiles && a.b.max_kv / tp.unit + 1 > tp.min_units);
  if (!join) return cudaSuccess;
  return launch_pdl(attn_join_kernel<T, HD>, dim3(592), dim3(kRows * 32), 0, st, a);
}

template <typename T>
cudaError_t launch_attn_hd(const AttnArgs& a, int hd, cudaStream_t st) {
  const int dt = Elem<T>::kType;
  if (hd == 64) return launch_attn<T, 64>(a, dt, st);
  if (hd == 128) return launch_attn<T, 128>(a, dt, st);
  return launch_attn<T, 256>(a, dt, st);
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
  const int64_t hd = batch->head_dim;
  if ((batch->total_q > 1 && (args->q_row_stride < hd || args->out_row_stride < hd)) ||
      (args->n_heads > 1 && (args->q_head_stride < hd || args->out_head_stride < hd)))
    return set_error(GB_ERR_INVALID_ARG, "row and head strides must be at least head_dim");
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
