// paged_attn_tc.cu -- attention of chunks of new tokens (gb_paged_attention's
// sequences of more than 16 rows) on the 5th-generation tensor cores.
//
// A CTA takes NT row tiles of 128 rows (tokens x the query heads of one KV
// head) and streams the keys they see in tiles of KT:
//   S_w = Q_w K^T            tcgen05.mma, A and B in shared memory, S in TMEM
//   P_w = 2^(S_w scale - m)  a warpgroup per row tile, a thread per row: S from
//                            TMEM into registers, P back over S as 16-bit pairs
//   O_w += P_w V             tcgen05.mma, A in TMEM, V as stored (its keys are
//                            the MMA's K: B is "MN-major")
// The tensor cores work on one row tile while another is in its softmax: two
// tiles of one CTA at head_dim 128 (each K and V tile is read once for both), two or
// four CTAs of an SM at 64, which also hide each other's start and end.  Where TMEM
// has room (256, and 64 with two CTAs), S has two buffers, so that the next tile's S
// is there when a softmax ends.  K and V
// tiles come by TMA from the pages as stored: a box per page and 64 columns (the
// 128-byte swizzle), the page number read by a lane of the producer warp; a page
// that is not needed, or bad, is read as out of range, which TMA fills with zeros.
//
// The reference maximum of a row moves only when a score passes the maximum by
// 2^6 (the weights stay below 2^(kTop + 6)); then the row's warpgroup scales O
// in TMEM, after its last MMA.  Sums of weights are f32, P is rounded to the
// pool's type, O accumulates in f32 in TMEM.
//
// A tile that some row sees only in part is masked score by score, and its V
// rows are looked over in shared memory first: rows that no row of the CTA sees
// are cleared (0 x NaN is NaN), and values that are not finite are cleared and
// noted: the rows that do see them add them at the end.
//
// Warps: four per row tile, then the TMA producer and the MMA issuer.  Every wait
// is bounded, as in the expert GEMMs.
//
// Measured, in a captured step: a chunk of 1000 tokens behind 16 K keys, 32 heads of 128,
// f16, 247-249 us, 1100 TFLOP/s (276-292 alone with cold caches; 1268 TFLOP/s behind 32
// K); head_dim 256 1160 and head_dim 64 680 TFLOP/s behind 32 K; four prompts of 2 K, 64
// heads of 64, 240-246 us, 520-534 TFLOP/s.  Bound at head_dim 64 by the
// softmax between the MMAs: 16 exponentials per clock and SM would take 127 us there,
// half the time.  Two threads per row, and exponentials as polynomials, were no faster.
#include "paged_attn.cuh"
#include "umma.cuh"

namespace gb {
namespace paged {
namespace {

// MANY, at head_dim 64: four CTAs on an SM with one S buffer and a short ring each,
// instead of two that reach further ahead.  A CTA spends some 8 us on its start and
// end, which more neighbours hide.
template <int HD, bool MANY = false>
struct Cfg {
  static constexpr int NT = HD == 128 ? 2 : 1;            // row tiles
  static constexpr int KT = HD == 128 ? 128 : 64;         // keys per tile
  static constexpr int kBufs = HD == 128 || MANY ? 1 : 2;  // S buffers per row tile
  static constexpr int kCtas = MANY ? 4 : HD == 64 ? 2 : 1;  // per SM
  static constexpr int kSub = HD / 64;                    // 64-column blocks
  static constexpr int kQBytes = NT * 128 * HD * 2;
  static constexpr int kTileBytes = KT * HD * 2;          // a K or V tile
  static constexpr int kRing = MANY ? 4 : HD == 64 ? 9 : HD == 128 ? 4 : 5;  // K and V tiles in flight
  static constexpr int kSoftmax = NT * 128;               // softmax threads
  // head_dim 128 holds 128 scores per thread: its softmax warps take registers
  // from the other warpgroup, which two idle warps fill (3 x 168 = 2 x 216 + 72).
  static constexpr bool kShift = HD == 128;
  static constexpr int kThreads = kSoftmax + (kShift ? 128 : 64);
  static constexpr int kBarBytes = 512;
  static constexpr int kSmem = 1024 + kQBytes + kRing * kTileBytes + kBarBytes;
  // TMEM columns: S of row tile w, buffer b at (w kBufs + b) KT; O at kOCol + w HD
  static constexpr int kTmem = 512 / kCtas;
  static constexpr int kOCol = NT * kBufs * KT;
  static_assert(kOCol + NT * HD <= kTmem && kCtas * kTmem <= 512, "S and O in TMEM");
  static_assert((2 * kRing + 1 + 8 * NT) * 8 <= kBarBytes, "barriers");
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z,
                                            int w, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}

// Low words of shared-memory descriptors (128-byte swizzle, 8-row groups 1024
// bytes apart).  K-major (Q, K): rows of 64 elements along the MMA's K.  MN-major
// (V): rows of 64 elements along N, `lbo` bytes between blocks of 64; the groups
// of 8 rows lie along the MMA's K.
__device__ __forceinline__ uint32_t k_major_lo(uint32_t saddr) {
  return ((saddr & 0x3FFFFu) >> 4) | (1u << 16);
}
__device__ __forceinline__ uint32_t mn_major_lo(uint32_t saddr, uint32_t lbo) {
  return ((saddr & 0x3FFFFu) >> 4) | ((lbo >> 4) << 16);
}

// kind::f16, D = f32, A and B of type T, M = 128, N = n; mn: B is MN-major.
template <typename T>
__device__ __forceinline__ constexpr uint32_t idesc(int n, bool mn) {
  const uint32_t t = Elem<T>::kType == GB_DTYPE_BF16 ? 1u : 0u;
  return (1u << 4) | (t << 7) | (t << 10) | ((mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(128 >> 4) << 24);
}

// The MMA warp runs converged, on values that are the same in every lane (so
// that descriptors stay in uniform registers: a lone lane in a divergent branch
// took 60 to 100 clocks per MMA to move them there), and one elected lane issues.
__device__ __forceinline__ bool elect() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(kFullMask, v, 0); }
// A 128-byte-swizzle descriptor from its low word (address and LBO); see sw128_desc.
__device__ __forceinline__ uint64_t desc_of(uint32_t lo) {
  constexpr uint32_t hi = (1024u >> 4) | (1u << 14) | (2u << 29);
  return ((uint64_t)hi << 32) | lo;
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(id), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(id), "r"(acc)
      : "memory");
}

#define GB_R8(v, o) "=r"(v[o]), "=r"(v[o + 1]), "=r"(v[o + 2]), "=r"(v[o + 3]), "=r"(v[o + 4]), \
                    "=r"(v[o + 5]), "=r"(v[o + 6]), "=r"(v[o + 7])
#define GB_W8(v, o) "r"(v[o]), "r"(v[o + 1]), "r"(v[o + 2]), "r"(v[o + 3]), "r"(v[o + 4]), \
                    "r"(v[o + 5]), "r"(v[o + 6]), "r"(v[o + 7])
// 32 columns of the thread's TMEM lane.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : GB_R8(v, 0), GB_R8(v, 8), GB_R8(v, 16), GB_R8(v, 24)
      : "r"(addr));
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
      "%14,%15};" ::GB_W8(v, 0),
      GB_W8(v, 8), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld8(uint32_t addr, uint32_t* v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : GB_R8(v, 0)
               : "r"(addr));
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::GB_W8(v, 0),
               "r"(addr)
               : "memory");
}
__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// ---- pairs of f32 (one instruction for both) -----------------------------------
__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// Element (row, column) of a K or V tile: blocks of 64 columns, 128-byte rows,
// 16-byte pieces swizzled by the row.
template <int HD>
__device__ __forceinline__ uint32_t tile_offset(int row, int piece) {
  return (uint32_t)((piece >> 3) * (Cfg<HD>::KT * 128) + row * 128 + (((piece & 7) ^ (row & 7)) << 4));
}

template <typename T, int HD, bool MANY>
__global__ void __launch_bounds__(Cfg<HD, MANY>::kThreads, Cfg<HD, MANY>::kCtas)
    attn_tile_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                     const __grid_constant__ CUtensorMap map_v, const __grid_constant__ AttnArgs a) {
  using C = Cfg<HD, MANY>;
  constexpr int NT = C::NT, KT = C::KT, kBufs = C::kBufs;
  constexpr int kHalves = kBufs == 1 ? 2 : 1;  // P handed over in parts
  // the buffer of a row tile's step, and the phase of its barriers
  auto buf_of = [](int w, int step) { return w * kBufs + (kBufs == 2 ? step & 1 : 0); };
  auto phase_of = [](int step) { return kBufs == 2 ? step >> 1 : step; };
  constexpr Plan kPlan = tile_plan<HD>();
  extern __shared__ uint8_t smem_raw[];
  const int tid = threadIdx.x, lane = tid & 31, warp = uniform(tid >> 5);
  const int tpt = 128 / a.group;  // tokens per row tile
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* ring = smem + C::kQBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + C::kRing * C::kTileBytes);
  uint64_t* kv_full = bars;                // [kRing]
  uint64_t* kv_empty = bars + C::kRing;    // [kRing]
  uint64_t* q_full = bars + 2 * C::kRing;
  uint64_t* s_full = q_full + 1;           // [2 NT]: row tile and buffer
  uint64_t* p_full = s_full + 2 * NT;      // [2 NT]: row tile, and buffer or half
  uint64_t* o_done = p_full + 2 * NT;      // [2 NT]: the PVs of a row tile in turn
  uint64_t* v_clean = o_done + 2 * NT;     // [2 NT]: a row tile's edge tiles in turn
  __shared__ uint32_t tmem_slot;
  // The bad pages of key tile j, a bit each, at j % 8: written by the producer once a slot
  // is free for K of j, when every softmax warp is within the ring of it (at most four
  // tiles behind), and read where S of j is there.
  __shared__ volatile uint32_t bad_pages[8];
  __shared__ int abort_word, poisoned;
  volatile int* abort_flag = &abort_word;

  if (tid == 0) {
    for (int i = 0; i < C::kRing; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
    }
    mbar_init(q_full, 1);
    for (int i = 0; i < 2 * NT; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 128);
      mbar_init(&o_done[i], 1);
      mbar_init(&v_clean[i], 128);
    }
    abort_word = poisoned = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) tmem_alloc(&tmem_slot, C::kTmem);
  // the item, while the barriers are set up and TMEM is allocated
  Item it;
  const bool have = find_item<false, C::kThreads>(a, kPlan, a.tiles, NT * tpt, &it);
  pdl_trigger();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (!have) {
    if (warp == 0) tmem_dealloc(tmem_slot, C::kTmem);
    pdl_wait();  // this grid ends after the kernel it was launched beside
    return;
  }

  // The tiles: row tile w has tokens [w tpt, w tpt + n_w); key tiles [u0, u1).
  const int n0 = min(it.tokens, tpt), n1 = it.tokens - n0;
  const int last = it.pos0 + it.tokens - 1;
  const int key_lo = a.window > 0 ? max(0, it.pos0 - a.window + 1) : 0;
  const int all_lo = a.window > 0 ? max(0, last - a.window + 1) : 0;
  // key tiles that row tile w sees any key of
  const int hi0 = min(it.u1, it.pos0 + n0 - 1 < 0 ? 0 : (it.pos0 + n0 - 1) / KT + 1);
  const int lo1 = max(it.u0, first_unit(it.pos0 + tpt, a.window, KT));
  auto active = [&](int w, int j) {
    return w == 0 ? j < hi0 : n1 > 0 && j >= lo1;
  };
  // a tile with a key that some row does not see
  const int32_t* table = a.b.table + it.seq * a.b.table_stride;
  const int page_size = 1 << a.b.page_shift;
  auto edge = [&](int j) { return j * KT + KT - 1 > it.pos0 || j * KT < all_lo; };

  const uint32_t tmem = tmem_slot;
  // A bounded wait of a whole warp, with one result for it: where it has run out, or
  // another warp's has, some lanes may still have seen the phase end, and none may go on
  // alone to what the warp does together (TMEM accesses, votes).
  auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
    if (__all_sync(kFullMask, mbar_try_wait(bar, parity & 1))) return true;
    const uint64_t t0 = globaltimer();
    while (!__all_sync(kFullMask, mbar_try_wait(bar, parity & 1)))
      if (__any_sync(kFullMask, *abort_flag || globaltimer() - t0 > a.wait_ns)) {
        *abort_flag = 1;
        return false;
      }
    return true;
  };

  if (warp < C::kSoftmax / 32) {
    if constexpr (C::kShift) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // ---------------- softmax: thread = row ---------------------------------------
    const int w = NT == 1 ? 0 : warp >> 2;  // row tile
    const int r = tid & 127;               // row of the tile
    const int tok = r / a.group;           // token of the tile
    const bool live = tok < (w ? n1 : n0) && r < tpt * a.group;
    const int head = it.g * a.group + r - tok * a.group;
    const int pos = live ? it.pos0 + w * tpt + tok : -1;
    const int first = live && a.window > 0 ? max(0, pos - a.window + 1) : 0;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t o_addr = tmem + C::kOCol + w * HD + lane_base;
    constexpr float kTop = Elem<T>::kTop;
    // PV of the row tile's step n done.  A parity tells a phase only from its
    // neighbours: S of a step comes after PV of the step two before, so with two
    // barriers in turn the phase before n's is always complete.
    auto wait_o = [&](int n) { return wait(&o_done[2 * w + (n & 1)], n >> 1); };
    // Reference maximum, sum of weights.  A row that is no token's holds whatever queries,
    // or shared memory, were there: its reference never moves.
    float m = live ? -INFINITY : INFINITY, l = 0.0f;
    // the key tiles that the row tile sees any key of
    const int j0 = w ? lo1 : it.u0, j1 = w ? (n1 > 0 ? it.u1 : lo1) : hi0;
    const int all_steps = max(j1 - j0, 0);
    int edges = 0;
    bool ok = true;
    for (int j = j0; j < j1; ++j) {
      const int steps = j - j0;
      const bool at_edge = edge(j);
      const int buf = buf_of(w, steps);
      const uint32_t s_addr = tmem + buf * KT + lane_base;
      ok = wait(&s_full[buf], phase_of(steps));
      if (!ok) break;
      if (at_edge) {
        // Look over this thread's share of the V tile (S of the tile is there, so the
        // ring is at most at this V).
        const int t = 2 * (j - it.u0) + 1;
        ok = wait(&kv_full[t % C::kRing], (t / C::kRing) & 1);
        if (!ok) break;
        uint8_t* v = ring + (t % C::kRing) * C::kTileBytes;
        constexpr int kPieces = HD / 8;
        bool found = false;
        const bool both = NT == 2 && active(w ^ 1, j);
        for (int i = both ? tid : r; i < KT * kPieces; i += both ? 256 : 128) {
          const int row = i / kPieces, key = j * KT + row;
          uint4* p = reinterpret_cast<uint4*>(v + tile_offset<HD>(row, i % kPieces));
          if (key > last || key < key_lo) {
            *p = make_uint4(0, 0, 0, 0);
          } else {
            const uint4 x = *p;
            if (any_nonfinite<T>(x.x) || any_nonfinite<T>(x.y) || any_nonfinite<T>(x.z) ||
                any_nonfinite<T>(x.w)) {
              *p = make_uint4(finite_only<T>(x.x), finite_only<T>(x.y), finite_only<T>(x.z),
                              finite_only<T>(x.w));
              found = true;
            }
          }
        }
        if (found) *(volatile int*)&poisoned = 1;
        fence_proxy_async_smem();
        mbar_arrive(&v_clean[2 * w + (edges++ & 1)]);
      }
      tc_fence_after();
      const unsigned bad = bad_pages[j & 7];
      uint32_t sb[KT];
#pragma unroll
      for (int c = 0; c < KT; c += 32) tmem_ld32(s_addr + c, sb + c);
      tmem_wait_ld();
      float* s = reinterpret_cast<float*>(sb);
      if (at_edge || bad) {
        const int hi = pos - j * KT, lo = first - j * KT;
#pragma unroll
        for (int i = 0; i < KT; ++i)
          if (i > hi || i < lo) s[i] = -INFINITY;
        for (unsigned left = bad; left; left &= left - 1) {
          const int b0 = (__ffs(left) - 1) << a.b.page_shift, b1 = b0 + page_size;
#pragma unroll
          for (int i = 0; i < KT; ++i)
            if (i >= b0 && i < b1) s[i] = -INFINITY;
        }
      }
      float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
      for (int i = 4; i < KT; i += 4)
#pragma unroll
        for (int c = 0; c < 4; ++c) mx[c] = fmaxf(mx[c], s[i + c]);
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale - kTop;
      const bool moves = top > m + 6.0f;
      if (__any_sync(kFullMask, moves)) {  // only the row that must: its rounding is its own
        const float f = moves ? ex2(m - top) : 1.0f;
        m = moves ? top : m;
        l *= f;
        if (steps) {  // after the last MMAs into this O
          ok = wait_o(steps - 1);
          if (!ok) break;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < HD; c += 8) {
            uint32_t o[8];
            tmem_ld8(o_addr + c, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            tmem_st8(o_addr + c, o);
          }
          tmem_wait_st();
        }
      }
      const float ref = m == -INFINITY ? 0.0f : m;
      const uint64_t scale2 = pair(a.scale, a.scale), ref2 = pair(-ref, -ref);
      uint64_t sum[2] = {0, 0};
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {  // the MMAs of a half start while the next is computed
#pragma unroll
        for (int c = h * (KT / 2 / kHalves); c < (h + 1) * (KT / 2 / kHalves); c += 16) {
          uint32_t p[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int e = 2 * (c + i);
            float2 v = unpair(fma2(pair(s[e], s[e + 1]), scale2, ref2));
            v.x = ex2(v.x);
            v.y = ex2(v.y);
            sum[i & 1] = add2(sum[i & 1], pair(v.x, v.y));
            p[i] = Elem<T>::pack(v.x, v.y);
          }
          tmem_st16(s_addr + c, p);
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&p_full[kHalves == 2 ? 2 * w + h : buf]);
      }
      {
        const float2 v = unpair(add2(sum[0], sum[1]));
        l += v.x + v.y;
      }
    }
    // ---- the row's result
    if (ok && all_steps) {
      ok = wait_o(all_steps - 1);
      tc_fence_after();
    }
    if (!__any_sync(kFullMask, *abort_flag) && ok && (w == 0 || n1 > 0)) {
      const bool split = it.slot >= 0;
      float M = m, L = l, inv;
      if (!split && a.sinks && live) {
        const float sink = a.sinks[head] * kLog2e;
        M = fmaxf(m, sink);
        L = l * part_factor(m, l, M) + (M == -INFINITY ? 0.0f : ex2(sink - M));
      }
      inv = split ? 1.0f : L == 0.0f ? 0.0f : part_factor(m, l, M) / L;
      const int out_row = it.row0 + w * tpt + tok;
      const int64_t part_row = split ? (int64_t)it.slot * kPlan.tile_rows + w * 128 + r : 0;
      if (split && live) a.tiles.ml[part_row] = make_float2(m, l);
      const bool poison = *(volatile int*)&poisoned != 0;
#pragma unroll(HD == 64 ? 2 : 1)
      for (int c = 0; c < HD; c += 32) {
        uint32_t o[32];
        __syncwarp();  // rows that are not live skip the stores
        if (all_steps) {
          tmem_ld32(o_addr + c, o);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0;
        }
        if (!live) continue;
        if (poison) {
          // values that are not finite, of the keys this row sees in edge tiles
          for (int key = max(first, it.u0 * KT); key <= min(pos, it.u1 * KT - 1); ++key) {
            if (!edge(key / KT)) continue;
            const int page = __ldg(table + (key >> a.b.page_shift));
            if ((unsigned)page >= (unsigned)a.b.n_pages) continue;
            const uint32_t* v = reinterpret_cast<const uint32_t*>(
                static_cast<const T*>(a.v_pool) + page * a.b.page_stride +
                (key & (page_size - 1)) * a.b.slot_stride + it.g * a.b.head_stride + c);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const uint32_t x = __ldg(v + i);
              if (!any_nonfinite<T>(x)) continue;
              const float2 f = Elem<T>::unpack(x);
              constexpr uint32_t em = Elem<T>::kExpMask;
              if ((x & em) == em) o[2 * i] = __float_as_uint(__uint_as_float(o[2 * i]) + f.x);
              if ((x & (em << 16)) == (em << 16))
                o[2 * i + 1] = __float_as_uint(__uint_as_float(o[2 * i + 1]) + f.y);
            }
          }
        }
        if (split) {
          float4* d = reinterpret_cast<float4*>(a.tiles.o + part_row * HD + c);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            d[i] = make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]),
                               __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3]));
        } else {
          const int64_t at = out_row * a.o_row + head * a.o_head + c;
          float y[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) y[i] = __uint_as_float(o[i]) * inv;
          if (a.out_f32) {
            float4* d = reinterpret_cast<float4*>(static_cast<float*>(a.out) + at);
#pragma unroll
            for (int i = 0; i < 8; ++i)
              d[i] = make_float4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
          } else {
            uint4* d = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + at);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              d[i] = make_uint4(Elem<T>::pack(y[8 * i], y[8 * i + 1]),
                                Elem<T>::pack(y[8 * i + 2], y[8 * i + 3]),
                                Elem<T>::pack(y[8 * i + 4], y[8 * i + 5]),
                                Elem<T>::pack(y[8 * i + 6], y[8 * i + 7]));
          }
        }
      }
    }
  } else {
    if constexpr (C::kShift) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == C::kSoftmax / 32) {
      // ---------------- TMA producer: Q, then K and V tiles in turn ---------------
      bool ok = true;
      if (lane == 0 && !(a.withhold_q && blockIdx.x == 0)) {
        // a box holds the tokens of a row tile with the group's heads: row = token * group + head
        const uint32_t bytes = (uint32_t)(n1 > 0 ? 2 : 1) * C::kSub * tpt * a.group * 128;
        mbar_arrive_expect_tx(q_full, bytes);
        for (int w = 0; w < (n1 > 0 ? 2 : 1); ++w)
          for (int s = 0; s < C::kSub; ++s)
            tma_load_3d(smem + (w * C::kSub + s) * 128 * 128, &map_q, s * 64, it.g * a.group,
                        it.row0 + w * tpt, q_full);
      }
      const int box = min(page_size, KT);            // keys per copy
      const int boxes = KT / box;                    // per 64 columns
      int slot = 0;
      uint32_t phase = 0;
      for (int j = it.u0; j < it.u1 && ok; ++j) {
        // lane b holds the page of the tile's keys [b box, b box + box)
        int page = a.b.n_pages, in_page = 0;
        bool bad = false;
        {
          const int key = j * KT + lane * box;
          in_page = key & (page_size - 1);
          if (lane < boxes && key <= last && key + box > key_lo) {
            const int p = __ldg(table + (key >> a.b.page_shift));
            if ((unsigned)p < (unsigned)a.b.n_pages) {
              page = p;
            } else {
              bad = true;
              flag(a.b, GB_PAGED_BAD_PAGE);
            }
          }
        }
        const unsigned bad_mask = __ballot_sync(kFullMask, bad);
        for (int kv = 0; kv < 2 && ok; ++kv) {
          ok = wait(&kv_empty[slot], phase ^ 1);
          if (!ok) break;
          if (lane == 0) {
            if (kv == 0) bad_pages[j & 7] = bad_mask;
            mbar_arrive_expect_tx(&kv_full[slot], C::kTileBytes);
          }
          __syncwarp();
          const uint32_t dst = smem_u32(ring + slot * C::kTileBytes);
          const CUtensorMap* map = kv ? &map_v : &map_k;
          if (lane < boxes) {
#pragma unroll
            for (int s = 0; s < C::kSub; ++s)
              tma_load_4d(dst + s * KT * 128 + lane * box * 128, map, s * 64, in_page, it.g, page,
                          &kv_full[slot]);
          }
          if (++slot == C::kRing) {
            slot = 0;
            phase ^= 1;
          }
        }
      }
      if (!ok) {  // copies in flight land within microseconds
        const uint64_t t0 = globaltimer();
        while (globaltimer() - t0 < 2000000ull) {
        }
      }
    } else if (warp == C::kSoftmax / 32 + 1) {
      // ---------------- MMA issuer -------------------------------------------------
      const int u0 = uniform(it.u0), n = uniform(it.u1) - u0;
      const int act0 = uniform(hi0) - u0;                            // row tile 0: j < act0
      const int act1 = uniform(n1 > 0 ? lo1 - it.u0 : 0x7fffffff);   // row tile 1: j >= act1
      // edge tiles: those from edge_hi on, and those before edge_lo
      const int edge_hi = uniform((it.pos0 + 1) / KT) - u0;
      const int edge_lo = uniform((all_lo + KT - 1) / KT) - u0;
      const uint32_t t_base = (uint32_t)uniform((int)tmem);
      const uint32_t q_lo = k_major_lo(smem_u32(smem)), ring_base = smem_u32(ring);
      auto on = [&](int w, int j) { return w == 0 ? j < act0 : j >= act1; };
      auto at_edge = [&](int j) { return j >= edge_hi || j < edge_lo; };
      bool ok = wait(q_full, 0);
      // Ring tile t (K of key tile j: 2 j, V: 2 j + 1) is in slot t % kRing, of phase t / kRing.
      int k_slot = 0, v_slot = 1;
      uint32_t k_phase = 0, v_phase = 0;
      auto advance = [&](int& slot, uint32_t& phase) {
        slot += 2;
        if (slot >= C::kRing) {
          slot -= C::kRing;
          phase ^= 1;
        }
      };
      int edges[2] = {0, 0};
      int s_steps[2] = {0, 0}, p_steps[2] = {0, 0};  // S issued, P taken, per row tile
      auto issue_s = [&](int w, uint32_t k_lo) {
        const int buf = buf_of(w, s_steps[w]++);
        const uint32_t d = t_base + buf * KT, q = q_lo + w * (C::kSub * 128 * 128 >> 4);
        if (elect()) {
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk)
            mma_ss(d, desc_of(q + (((kk >> 2) * 128 * 128 + (kk & 3) * 32) >> 4)),
                   desc_of(k_lo + (((kk >> 2) * KT * 128 + (kk & 3) * 32) >> 4)), idesc<T>(KT, false),
                   kk != 0);
          mma_commit(&s_full[buf]);
        }
        __syncwarp();
      };
      auto issue_pv = [&](int w, uint32_t v_lo) -> bool {
        const int step = p_steps[w]++, buf = buf_of(w, step);
        const uint32_t first = step ? 1u : 0u;
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
          if (!wait(&p_full[kHalves == 2 ? 2 * w + h : buf], phase_of(step))) return false;
          tc_fence_after();
          if (elect()) {
#pragma unroll
            for (int i = 0; i < KT / 16 / kHalves; ++i) {
              const int kk = h * (KT / 16 / kHalves) + i;
              mma_ts(t_base + C::kOCol + w * HD, t_base + buf * KT + kk * 8,
                     desc_of(v_lo + kk * (2048 >> 4)), idesc<T>(HD, true), kk != 0 ? 1u : first);
            }
            if (h == kHalves - 1) mma_commit(&o_done[2 * w + (step & 1)]);
          }
          __syncwarp();
        }
        return true;
      };
      auto free_slot = [&](int& slot, uint32_t& phase) {  // once the MMAs issued so far are done
        if (elect()) mma_commit(&kv_empty[slot]);
        __syncwarp();
        advance(slot, phase);
      };
      auto k_tile = [&](uint32_t* k_lo) -> bool {
        if (!wait(&kv_full[k_slot], k_phase)) return false;
        tc_fence_after();
        *k_lo = k_major_lo(ring_base + k_slot * C::kTileBytes);
        return true;
      };
      uint32_t k_lo = 0;
      if (ok && n > 0 && (ok = k_tile(&k_lo))) {
#pragma unroll
        for (int w = 0; w < NT; ++w)
          if (on(w, 0)) issue_s(w, k_lo);
        free_slot(k_slot, k_phase);
      }
      for (int j = 0; j < n && ok; ++j) {
        const bool more = j + 1 < n;
        ok = wait(&kv_full[v_slot], v_phase);
        if (at_edge(j)) {
#pragma unroll
          for (int w = 0; w < NT; ++w)
            if (on(w, j)) {
              ok = ok && wait(&v_clean[2 * w + (edges[w] & 1)], edges[w] >> 1);
              ++edges[w];
            }
        }
        ok = ok && (!more || k_tile(&k_lo));
        if (!ok) break;
        const uint32_t v_lo = mn_major_lo(ring_base + v_slot * C::kTileBytes, KT * 128);
        // With two buffers the next S goes before this P V: its buffer's last reader, PV
        // of j - 1, is issued.  (Never before v_clean of j: a row tile's softmax cannot
        // then reach edge tile j + 2 before that phase is seen.)  With one buffer, after.
        if (kBufs == 2 && more) {
#pragma unroll
          for (int w = 0; w < NT; ++w)
            if (on(w, j + 1)) issue_s(w, k_lo);
          free_slot(k_slot, k_phase);
        }
#pragma unroll
        for (int w = 0; w < NT; ++w) {
          if (on(w, j)) ok = ok && issue_pv(w, v_lo);
          if (kBufs == 1 && more && on(w, j + 1) && ok) issue_s(w, k_lo);
        }
        if (!ok) break;
        free_slot(v_slot, v_phase);
        if (kBufs == 1 && more) free_slot(k_slot, k_phase);
      }
      if (!ok) {  // issued MMAs read shared memory and TMEM: let them finish
        const uint64_t t0 = globaltimer();
        while (globaltimer() - t0 < 2000000ull) {
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tmem_dealloc(tmem, C::kTmem);
  if (tid == 0 && *abort_flag) flag(a.b, GB_PAGED_TIMEOUT);
  pdl_wait();
}

cudaError_t make_map(CUtensorMap* m, int dtype, const void* base, int rank, const cuuint64_t* dims,
                     const cuuint64_t* strides, const cuuint32_t* box) {
  auto encode = tensor_map_encoder();
  if (!encode) return cudaErrorNotSupported;
  const cuuint32_t ones[4] = {1, 1, 1, 1};
  const CUresult r = encode(
      m, dtype == GB_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
      rank, const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
      CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

template <typename T, int HD, bool MANY = false>
cudaError_t launch(const AttnArgs& a, bool pdl, cudaStream_t st) {
  using C = Cfg<HD, MANY>;
  const int tpt = 128 / a.group;
  constexpr int dt = Elem<T>::kType;
  CUtensorMap mq, mk, mv;
  const int page_size = 1 << a.b.page_shift;
  // A dimension of one has no stride of its own; the encoder wants a valid one.
  auto stride = [](int64_t s, int64_t n) { return (cuuint64_t)(n > 1 ? s * 2 : HD * 2); };
  {
    const cuuint64_t dims[3] = {HD, (cuuint64_t)a.nh, (cuuint64_t)a.b.total_q};
    const cuuint64_t strides[2] = {stride(a.q_head, a.nh), stride(a.q_row, a.b.total_q)};
    const cuuint32_t box[3] = {64, (cuuint32_t)a.group, (cuuint32_t)tpt};
    const cudaError_t e = make_map(&mq, dt, a.q, 3, dims, strides, box);
    if (e != cudaSuccess) return e;
  }
  for (int v = 0; v < 2; ++v) {
    const cuuint64_t dims[4] = {HD, (cuuint64_t)page_size, (cuuint64_t)a.b.nkv,
                                (cuuint64_t)a.b.n_pages};
    const cuuint64_t strides[3] = {stride(a.b.slot_stride, page_size), stride(a.b.head_stride, a.b.nkv),
                                   stride(a.b.page_stride, a.b.n_pages)};
    const cuuint32_t box[4] = {64, (cuuint32_t)std::min(page_size, C::KT), 1, 1};
    const cudaError_t e = make_map(v ? &mv : &mk, dt, v ? a.v_pool : a.k_pool, 4, dims, strides, box);
    if (e != cudaSuccess) return e;
  }
  const int64_t per = (int64_t)C::NT * tpt;
  const int64_t tiles = std::min<int64_t>(a.b.total_q / per + a.b.n_seqs, a.b.total_q) * a.b.nkv;
  const int64_t grid = grid_bound(a, tile_plan<HD>(), tiles);
  if (grid > (a.b.n_seqs <= kLaneSeqs ? (int64_t)kMaxItems : 0x7fffffffll))
    return cudaErrorInvalidConfiguration;
  auto kern = attn_tile_kernel<T, HD, MANY>;
  cudaError_t e = set_smem_limit(kern, C::kSmem);
  if (e != cudaSuccess) return e;
  if (pdl)
    return launch_pdl(kern, dim3((unsigned)grid), dim3(C::kThreads), C::kSmem, st, mq, mk, mv, a);
  kern<<<(unsigned)grid, C::kThreads, C::kSmem, st>>>(mq, mk, mv, a);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_hd(const AttnArgs& a, int hd, bool pdl, cudaStream_t st) {
  // Four CTAs per SM from two waves of two on, unless rows see many keys (64 query and 8
  // KV heads): 1184 tiles of 4 K keys 283 us against 297, 2368 of up to 5 K 262 against
  // 297, with a window of 128 75 against 86; but 296 tiles of 4 K keys 83 against 70, and
  // 1184 of 30 K keys 1731 against 1665.  Decoding sequences have no tiles: of the host's
  // bounds, there are as many chunks as the rows need when every other sequence has one.
  // While keys are few, though, the small CTAs start sooner beside those of many decoding
  // sequences, which then count like tiles: 250 of 500 keys and a chunk of 200 behind 1 K
  // keys 124 us against 134 (of 500 behind 100: 112 against 122), behind 2 K, of 350 145
  // against 155, of 500 148 against 140.  With more keys they lose the more, the more tiles
  // there are: 74 of 2 K and a chunk of 280 behind 4 K 167 against 142, of 500 202 against
  // 147, behind 8 K 296 against 194 (but 74 of 300 keys, 200 behind 4 K, 91 against 97).
  const int64_t chunks = std::min<int64_t>(
      a.b.n_seqs, std::max<int64_t>(1, (a.b.total_q - a.b.n_seqs + a.b.max_q - 2) / (a.b.max_q - 1)));
  const int64_t rows = std::max<int64_t>(0, a.b.total_q - (a.b.n_seqs - chunks));
  const int64_t keys = a.window > 0 ? std::min<int64_t>(a.window, a.b.max_kv) : a.b.max_kv;
  int64_t tiles = (rows * a.group / 128 + chunks) * a.b.nkv;
  if (keys <= (tiles < 222 ? 4096 : 2048)) tiles += (a.b.n_seqs - chunks) * a.b.nkv;
  if (hd == 64 && tiles >= 592 && keys <= 8192) return launch<T, 64, true>(a, pdl, st);
  if (hd == 64) return launch<T, 64>(a, pdl, st);
  if (hd == 128) return launch<T, 128>(a, pdl, st);
  return launch<T, 256>(a, pdl, st);
}

}  // namespace

namespace {
thread_local uint64_t t_wait_ns = kMbarWaitNs;
thread_local bool t_withhold_q = false;
}  // namespace

cudaError_t launch_attn_tiles(AttnArgs a, int dtype, int hd, bool pdl, cudaStream_t st) {
  a.wait_ns = t_wait_ns;
  a.withhold_q = t_withhold_q;
  return dtype == GB_DTYPE_BF16 ? launch_hd<__nv_bfloat16>(a, hd, pdl, st)
                                : launch_hd<__half>(a, hd, pdl, st);
}

}  // namespace paged
}  // namespace gb

extern "C" int gb_paged_set_test_hooks(int64_t wait_limit_us, int32_t withhold_q) {
  using namespace gb;
  if (wait_limit_us < 0 || wait_limit_us > 10000000)
    return set_error(GB_ERR_INVALID_ARG, "wait_limit_us %lld outside [0, 1e7]", (long long)wait_limit_us);
  paged::t_wait_ns = wait_limit_us ? (uint64_t)wait_limit_us * 1000ull : kMbarWaitNs;
  paged::t_withhold_q = withhold_q != 0;
  return GB_OK;
}
