// paged_rope.cu -- the paged cache's memory-bound operators: norm + rotation +
// page append of a batch's new rows (gb_paged_rope_append), page copies
// (gb_paged_copy), and the batch descriptor's checks.
#include <algorithm>
#include <vector>

#include "paged.cuh"
#include "ptx.cuh"

namespace gb {
namespace paged {

int check_batch(const gb_paged_batch* d, Batch* b) {
  if (!d) return set_error(GB_ERR_INVALID_ARG, "batch is null");
  if (d->struct_size != sizeof(gb_paged_batch))
    return set_error(GB_ERR_INVALID_ARG, "gb_paged_batch: struct_size %u, expected %zu",
                     d->struct_size, sizeof(gb_paged_batch));
  if (d->dtype != GB_DTYPE_BF16 && d->dtype != GB_DTYPE_F16)
    return set_error(GB_ERR_UNSUPPORTED, "pool dtype %d: BF16 or F16", d->dtype);
  if (d->head_dim != 64 && d->head_dim != 128 && d->head_dim != 256)
    return set_error(GB_ERR_UNSUPPORTED, "head_dim %d: 64, 128 or 256", d->head_dim);
  if (d->page_size < 8 || d->page_size > 1024 || (d->page_size & (d->page_size - 1)))
    return set_error(GB_ERR_UNSUPPORTED, "page_size %d: a power of two from 8 to 1024",
                     d->page_size);
  if (d->n_kv_heads < 1 || d->n_kv_heads > 1024 || d->n_pages < 1)
    return set_error(GB_ERR_INVALID_ARG, "n_kv_heads must be 1..1024 and n_pages >= 1");
  if (d->n_seqs < 0 || d->total_q < 0 || d->max_q_len < 0 || d->max_kv_len < 0)
    return set_error(GB_ERR_INVALID_ARG,
                     "n_seqs, total_q, max_q_len and max_kv_len must be >= 0");
  if (d->n_seqs > (1 << 20)) return set_error(GB_ERR_UNSUPPORTED, "more than 2^20 sequences");
  const int64_t row = d->head_dim;
  if (!stride_ok(d->page_stride, 2) || !stride_ok(d->slot_stride, 2) ||
      !stride_ok(d->head_stride, 2) || (d->page_size > 1 && d->slot_stride < row) ||
      (d->n_kv_heads > 1 && d->head_stride < row) || (d->n_pages > 1 && d->page_stride < row))
    return set_error(GB_ERR_INVALID_ARG,
                     "pool strides must be multiples of 8 elements, at least head_dim");
  if (d->table_stride < 0) return set_error(GB_ERR_INVALID_ARG, "table_stride < 0");
  if (d->n_seqs > 0 && (!d->q_start_dev || !d->kv_len_dev || !d->page_table_dev))
    return set_error(GB_ERR_INVALID_ARG, "q_start, kv_len and page_table must not be null");
  b->n_seqs = d->n_seqs;
  b->total_q = d->total_q;
  b->max_q = d->max_q_len;
  b->max_kv = d->max_kv_len;
  b->nkv = d->n_kv_heads;
  b->page_shift = 31 - __builtin_clz((unsigned)d->page_size);
  b->n_pages = d->n_pages;
  b->page_stride = d->page_stride;
  b->slot_stride = d->slot_stride;
  b->head_stride = d->head_stride;
  b->q_start = d->q_start_dev;
  b->kv_len = d->kv_len_dev;
  b->table = d->page_table_dev;
  b->table_stride = d->table_stride;
  b->err = d->error_dev;
  return GB_OK;
}

namespace {

// ---- norm + rotation + page append -----------------------------------------
// One pass over q, k and v: y = x / sqrt(mean(x^2) + eps) * w over a head, then
// the halves-layout rotation, q to q_out, k and v to their pages.  A group of
// head_dim / 8 lanes takes a head of a row, 8 elements (16 bytes of a 2-byte type)
// a lane, so a warp's loads and stores are whole 128-byte lines.  The rotation
// pairs element j with j + rot / 2, which another lane of the group holds at a
// fixed lane distance (rot / 16), so one shuffle per element exchanges them.  Each
// element is read once and written once; memory is the floor.

constexpr int kRopeThreads = 256;
constexpr int kRopeRows = 64;  // rows per CTA, at most

struct RopeArgs {
  Batch b;
  int nh, hd, rot;
  int64_t units;
  const void *q, *k, *v;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;
  void* q_out;
  int64_t o_row, o_head;
  const float *q_norm, *k_norm, *cos_t, *sin_t;
  int64_t table_rows;
  void *k_pool, *v_pool;
  float eps;
};

struct RowInfo {
  int pos;      // -1: no sequence owns the row, or its position is unusable
  int slot;     // slot in the page
  int64_t page; // element offset of the page, -1: no page (the stores are dropped)
};

// The warp finds row r's sequence: the largest s with q_start[s] <= r.
__device__ __forceinline__ RowInfo find_row(const Batch& b, int r, int64_t table_rows, int lane) {
  RowInfo info{-1, 0, -1};
  if (r >= min(max(__ldg(b.q_start + b.n_seqs), 0), b.total_q)) return info;
  int lo = 0, n = b.n_seqs;  // the answer is in [lo, lo + n)
  while (n > 1) {
    const int step = (n + 31) / 32;
    const int s = lo + lane * step;
    const bool le = lane * step < n && __ldg(b.q_start + s) <= r;
    const unsigned m = __ballot_sync(kFullMask, le);
    if (!m) break;  // q_start[0] > r: not ascending from 0
    const int hit = 31 - __clz(m);
    const int left = n - hit * step;
    lo += hit * step;
    n = min(step, left);
  }
  const Seq q = load_seq(b, lo, lane == 0);
  const int i = r - q.row0;
  if (i < 0 || i >= q.q_len) return info;
  const int pos = q.kv_len - q.q_len + i;
  if (pos < 0 || pos >= table_rows) {
    if (lane == 0) flag(b, GB_PAGED_BAD_POSITION);
    return info;
  }
  info.pos = pos;
  info.slot = pos & ((1 << b.page_shift) - 1);
  const int page = __ldg(b.table + lo * b.table_stride + (pos >> b.page_shift));
  if ((unsigned)page < (unsigned)b.n_pages)
    info.page = page * b.page_stride;
  else if (lane == 0)
    flag(b, GB_PAGED_BAD_PAGE);
  return info;
}

template <typename In>
struct Load8;
template <typename T2>
struct Load8Half {
  uint4 r;
  __device__ __forceinline__ void load(const void* p, int64_t off) {
    r = *reinterpret_cast<const uint4*>(static_cast<const T2*>(p) + off);
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = Elem<T2>::unpack(w[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
};
template <>
struct Load8<__nv_bfloat16> : Load8Half<__nv_bfloat16> {};
template <>
struct Load8<__half> : Load8Half<__half> {};
template <>
struct Load8<float> {
  float4 a, c;
  __device__ __forceinline__ void load(const void* p, int64_t off) {
    const float4* s = reinterpret_cast<const float4*>(static_cast<const float*>(p) + off);
    a = s[0];
    c = s[1];
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
    x[4] = c.x, x[5] = c.y, x[6] = c.z, x[7] = c.w;
  }
};

// Norm and rotation of a head, 8 elements a lane.  w: norm weights or null (norms:
// some head of the call has them, so the sums are taken by every lane); cs, sn: the
// lane's cosines and sines, sn negative in the first half of the rotated elements;
// rotates: this lane's elements are rotated.
template <int HD>
__device__ __forceinline__ void norm_rotate(float (&y)[8], bool norms, const float* w, int d, float eps,
                                            bool rotation, bool rotates, int partner,
                                            const float (&cs)[8], const float (&sn)[8]) {
  if (norms) {
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = __fmaf_rn(y[i], y[i], ss);
#pragma unroll
    for (int o = HD / 16; o >= 1; o >>= 1) ss += __shfl_xor_sync(kFullMask, ss, o);
    if (w) {
      const float inv = rsqrtf(__fmaf_rn(ss, 1.0f / HD, eps));
      const float4 w0 = __ldg(reinterpret_cast<const float4*>(w + d));
      const float4 w1 = __ldg(reinterpret_cast<const float4*>(w + d + 4));
      const float ws[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = y[i] * inv * ws[i];
    }
  }
  if (rotation) {
    float other[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) other[i] = __shfl_sync(kFullMask, y[i], partner);
    if (rotates) {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = __fmaf_rn(y[i], cs[i], other[i] * sn[i]);
    }
  }
}

// cs and sn of a lane whose elements start at d, for a row at `pos`.
__device__ __forceinline__ void load_turn(const RopeArgs& a, int pos, int half, int d, float (&cs)[8],
                                          float (&sn)[8]) {
  const bool first = d < half;
  const int64_t at = (int64_t)pos * half + (first ? d : d - half);
  const float4* c4 = reinterpret_cast<const float4*>(a.cos_t + at);
  const float4* s4 = reinterpret_cast<const float4*>(a.sin_t + at);
  const float4 c0 = __ldg(c4), c1 = __ldg(c4 + 1), s0 = __ldg(s4), s1 = __ldg(s4 + 1);
  cs[0] = c0.x, cs[1] = c0.y, cs[2] = c0.z, cs[3] = c0.w;
  cs[4] = c1.x, cs[5] = c1.y, cs[6] = c1.z, cs[7] = c1.w;
  sn[0] = s0.x, sn[1] = s0.y, sn[2] = s0.z, sn[3] = s0.w;
  sn[4] = s1.x, sn[5] = s1.y, sn[6] = s1.z, sn[7] = s1.w;
#pragma unroll
  for (int i = 0; i < 8; ++i) sn[i] = first ? -sn[i] : sn[i];
}

template <typename Out>
__device__ __forceinline__ uint4 pack8(const float (&y)[8]) {
  return make_uint4(Elem<Out>::pack(y[0], y[1]), Elem<Out>::pack(y[2], y[3]),
                    Elem<Out>::pack(y[4], y[5]), Elem<Out>::pack(y[6], y[7]));
}

// Few (row, head) units: one per lane group, over as many CTAs as that takes.  The
// rows' sequences and slots are looked up while the units' loads are in flight.  Bound
// by the chain of those loads: one row of 80 heads of 64 takes 2.7 us with its launch,
// 61 rows of 48 heads of 128 3.8.
template <typename In, typename Out, int HD>
__global__ void __launch_bounds__(kRopeThreads) rope_units_kernel(const __grid_constant__ RopeArgs a) {
  constexpr int L = HD / 8;                // lanes per unit
  constexpr int G = kRopeThreads / L;      // units of the CTA
  __shared__ RowInfo rows[G];
  const int heads = a.nh + 2 * a.b.nkv;
  const int64_t unit0 = (int64_t)blockIdx.x * G, last = min(unit0 + G, a.units) - 1;
  const int row0 = (int)(unit0 / heads), n_rows = (int)(last / heads) - row0 + 1;
  const int d = threadIdx.x % L * 8, lane = threadIdx.x & 31;
  const int64_t unit = unit0 + threadIdx.x / L;
  const bool live = unit <= last;
  const int row = live ? (int)(unit / heads) : row0;
  const int h = live ? (int)(unit - (int64_t)row * heads) : 0;
  const bool is_q = h < a.nh, is_v = h >= a.nh + a.b.nkv;
  Load8<In> x;
  if (live) {
    if (is_q)
      x.load(a.q, row * a.q_row + h * a.q_head + d);
    else if (!is_v)
      x.load(a.k, row * a.k_row + (h - a.nh) * a.k_head + d);
    else
      x.load(a.v, row * a.v_row + (h - a.nh - a.b.nkv) * a.v_head + d);
  }
  for (int i = threadIdx.x >> 5; i < n_rows; i += kRopeThreads / 32) {
    const RowInfo r = find_row(a.b, row0 + i, a.rot ? a.table_rows : INT64_MAX, lane);
    if (lane == 0) rows[i] = r;
  }
  __syncthreads();
  const RowInfo info = live ? rows[row - row0] : RowInfo{-1, 0, -1};
  const int half = a.rot / 2, gap = half / 8;  // lanes to the rotation's partner
  const int partner = d < half ? lane + gap : d < a.rot ? lane - gap : lane;
  const bool rotates = !is_v && d < a.rot && info.pos >= 0;
  float y[8] = {}, cs[8] = {}, sn[8] = {};
  if (live) x.get(y);
  if (rotates) load_turn(a, info.pos, half, d, cs, sn);
  norm_rotate<HD>(y, a.q_norm || a.k_norm, is_v ? nullptr : is_q ? a.q_norm : a.k_norm, d, a.eps, half,
                  rotates, partner, cs, sn);
  if (!live || info.pos < 0) return;
  const uint4 o = pack8<Out>(y);
  if (is_q) {
    *reinterpret_cast<uint4*>(static_cast<Out*>(a.q_out) + row * a.o_row + h * a.o_head + d) = o;
  } else if (info.page >= 0) {
    const int g = is_v ? h - a.nh - a.b.nkv : h - a.nh;
    Out* pool = static_cast<Out*>(is_v ? a.v_pool : a.k_pool);
    *reinterpret_cast<uint4*>(pool + info.page + info.slot * a.b.slot_stride + g * a.b.head_stride + d) = o;
  }
}

// Many rows: a CTA takes `per` of them (at most kRopeRows).  `across` lane groups
// share a row, each with its heads in turn, so that a row's cosines, sines, page
// and addresses are worked out once for them; the groups' other rows run beside.
// 8150 rows of 48 heads of 128 with both norms: 54-55 us, 3.6 TB/s (82 with a unit at a
// time over the whole batch, 62 with the loads a pass ahead).  With room for three CTAs
// 16-bit rows still take 64 registers, so that four fit; f32 rows take more, three fit,
// 72 us.  Bounded to four, 56, and 69 with 40 bytes of spills.  59 % of the issue slots
// and about half of DRAM are busy: neither bounds it alone, and what the warps wait for
// between has not been told apart.
template <typename In, typename Out, int HD>
__global__ void __launch_bounds__(kRopeThreads, 3)
    rope_rows_kernel(const __grid_constant__ RopeArgs a, int per, int across) {
  constexpr int L = HD / 8;
  constexpr int G = kRopeThreads / L;
  constexpr int U = 3;  // heads whose loads are in flight
  __shared__ RowInfo rows[kRopeRows];
  const int heads = a.nh + 2 * a.b.nkv;
  const int row0 = blockIdx.x * per, n_rows = min(per, a.b.total_q - row0);
  const int lane = threadIdx.x & 31;
  for (int i = threadIdx.x >> 5; i < n_rows; i += kRopeThreads / 32) {
    const RowInfo r = find_row(a.b, row0 + i, a.rot ? a.table_rows : INT64_MAX, lane);
    if (lane == 0) rows[i] = r;
  }
  __syncthreads();
  const int d = threadIdx.x % L * 8;
  const int grp = threadIdx.x / L, beside = G / across;  // rows at a time
  const int sub = grp / across, h0 = grp - sub * across;
  const int half = a.rot / 2, gap = half / 8;
  const int partner = d < half ? lane + gap : d < a.rot ? lane - gap : lane;
  const bool norms = a.q_norm || a.k_norm;
  for (int i0 = 0; i0 < n_rows; i0 += beside) {  // the same passes in every lane
    const int i = i0 + sub;
    const RowInfo info = sub < beside && i < n_rows ? rows[i] : RowInfo{-1, 0, -1};
    const bool on = info.pos >= 0;
    float cs[8] = {}, sn[8] = {};
    if (on && d < a.rot) load_turn(a, info.pos, half, d, cs, sn);
    const int64_t r = row0 + i;
    const int64_t q_at = r * a.q_row + d, k_at = r * a.k_row + d, v_at = r * a.v_row + d;
    const int64_t o_at = r * a.o_row + d;
    const int64_t p_at = info.page < 0 ? -1 : info.page + info.slot * a.b.slot_stride + d;
    for (int hb = 0; hb < heads; hb += across * U) {
      Load8<In> x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int h = hb + u * across + h0;
        if (!on || h >= heads) continue;
        if (h < a.nh)
          x[u].load(a.q, q_at + h * a.q_head);
        else if (h < a.nh + a.b.nkv)
          x[u].load(a.k, k_at + (h - a.nh) * a.k_head);
        else
          x[u].load(a.v, v_at + (h - a.nh - a.b.nkv) * a.v_head);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (hb + u * across >= heads) break;  // for every group
        const int h = hb + u * across + h0;
        const bool live = on && h < heads, is_q = h < a.nh, is_v = h >= a.nh + a.b.nkv;
        float y[8] = {};
        if (live) x[u].get(y);
        norm_rotate<HD>(y, norms, is_v ? nullptr : is_q ? a.q_norm : a.k_norm, d, a.eps, half,
                        live && !is_v && d < a.rot, partner, cs, sn);
        if (!live) continue;
        const uint4 o = pack8<Out>(y);
        if (is_q) {
          *reinterpret_cast<uint4*>(static_cast<Out*>(a.q_out) + o_at + h * a.o_head) = o;
        } else if (p_at >= 0) {
          const int g = is_v ? h - a.nh - a.b.nkv : h - a.nh;
          *reinterpret_cast<uint4*>(static_cast<Out*>(is_v ? a.v_pool : a.k_pool) + p_at +
                                    g * a.b.head_stride) = o;
        }
      }
    }
  }
}

template <typename In, typename Out, int HD>
cudaError_t launch_rope(const RopeArgs& a, cudaStream_t st) {
  constexpr int G = kRopeThreads / (HD / 8);
  const int heads = a.nh + 2 * a.b.nkv;
  if (a.units <= (int64_t)G * 148 * 4) {
    rope_units_kernel<In, Out, HD><<<(unsigned)((a.units + G - 1) / G), kRopeThreads, 0, st>>>(a);
  } else {
    // Several CTAs an SM, a few rows each: the look-ups of a row are some 1.5 us of
    // dependent loads, which other CTAs' rows hide.
    const int64_t rows = a.units / heads;
    const int per = (int)std::max<int64_t>(1, std::min<int64_t>(kRopeRows, rows / (148 * 4 * 4)));
    rope_rows_kernel<In, Out, HD>
        <<<(unsigned)((rows + per - 1) / per), kRopeThreads, 0, st>>>(a, per, std::min(heads, G));
  }
  return cudaGetLastError();
}

template <typename In, typename Out>
cudaError_t launch_rope_hd(const RopeArgs& a, cudaStream_t st) {
  if (a.hd == 64) return launch_rope<In, Out, 64>(a, st);
  if (a.hd == 128) return launch_rope<In, Out, 128>(a, st);
  return launch_rope<In, Out, 256>(a, st);
}

template <typename Out>
cudaError_t launch_rope_in(const RopeArgs& a, int in_dtype, cudaStream_t st) {
  if (in_dtype == GB_DTYPE_F32) return launch_rope_hd<float, Out>(a, st);
  if (in_dtype == GB_DTYPE_BF16) return launch_rope_hd<__nv_bfloat16, Out>(a, st);
  return launch_rope_hd<__half, Out>(a, st);
}

// ---- page copies -------------------------------------------------------------
// (pool, page pair) x pieces of kCopyPiece bytes, a piece per CTA: every thread
// issues its loads before its stores.  The pools' addresses and the pairs are
// kernel parameters (constant memory), so the call needs no device list whose
// lifetime a caller would have to mind.  Bound by memory: each byte read once
// and written once.
constexpr int kCopyThreads = 256;
constexpr int kCopyVecs = 4;
constexpr int64_t kCopyPiece = (int64_t)kCopyThreads * kCopyVecs * 16;

template <int POOLS, int PAIRS>
struct CopyArgs {
  char* pool[POOLS];
  int2 pair[PAIRS];
  int64_t page_bytes, page_stride;
  int n_pairs, pieces;  // pieces per page
};

template <int POOLS, int PAIRS>
__global__ void __launch_bounds__(kCopyThreads)
    copy_pages_kernel(const __grid_constant__ CopyArgs<POOLS, PAIRS> a) {
  const unsigned unit = blockIdx.x / a.pieces, piece = blockIdx.x - unit * a.pieces;
  const unsigned p = unit / a.n_pairs, i = unit - p * a.n_pairs;
  const int2 pr = a.pair[i];
  const int64_t off = piece * kCopyPiece + threadIdx.x * 16;
  const char* src = a.pool[p] + pr.x * a.page_stride + off;
  char* dst = a.pool[p] + pr.y * a.page_stride + off;
  uint4 v[kCopyVecs];
#pragma unroll
  for (int j = 0; j < kCopyVecs; ++j)
    if (off + j * kCopyThreads * 16 < a.page_bytes)
      v[j] = ld_stream_u4(src + j * kCopyThreads * 16);
#pragma unroll
  for (int j = 0; j < kCopyVecs; ++j)
    if (off + j * kCopyThreads * 16 < a.page_bytes)
      __stcs(reinterpret_cast<uint4*>(dst + j * kCopyThreads * 16), v[j]);
}

template <int POOLS, int PAIRS>
cudaError_t launch_copy(void* const* pools, int n_pools, int64_t page_bytes, int64_t page_stride,
                        const int32_t* src, const int32_t* dst, int n, cudaStream_t st) {
  CopyArgs<POOLS, PAIRS> a;
  a.page_bytes = page_bytes;
  a.page_stride = page_stride;
  a.pieces = (int)((page_bytes + kCopyPiece - 1) / kCopyPiece);
  for (int i0 = 0; i0 < n; i0 += PAIRS) {
    a.n_pairs = std::min(PAIRS, n - i0);
    for (int i = 0; i < a.n_pairs; ++i) a.pair[i] = make_int2(src[i0 + i], dst[i0 + i]);
    // pools per launch: the grid's x stays below 2^31
    const int64_t per_pool = (int64_t)a.n_pairs * a.pieces;
    const int most = (int)std::min<int64_t>(POOLS, std::max<int64_t>(1, 0x7fffffffll / per_pool));
    for (int p0 = 0; p0 < n_pools; p0 += most) {
      const int np = std::min(most, n_pools - p0);
      for (int p = 0; p < np; ++p) a.pool[p] = static_cast<char*>(pools[p0 + p]);
      copy_pages_kernel<POOLS, PAIRS><<<(unsigned)(np * per_pool), kCopyThreads, 0, st>>>(a);
      const cudaError_t e = cudaGetLastError();
      if (e != cudaSuccess) return e;
    }
  }
  return cudaSuccess;
}

}  // namespace
}  // namespace paged
}  // namespace gb

extern "C" int gb_paged_rope_append(const gb_paged_batch* batch, const gb_rope_args* args,
                                    void* stream) {
  using namespace gb;
  using namespace gb::paged;
  RopeArgs a{};
  const int rc = check_batch(batch, &a.b);
  if (rc) return rc;
  if (!args) return set_error(GB_ERR_INVALID_ARG, "args is null");
  if (args->struct_size != sizeof(gb_rope_args))
    return set_error(GB_ERR_INVALID_ARG, "gb_rope_args: struct_size %u, expected %zu",
                     args->struct_size, sizeof(gb_rope_args));
  const int in = args->in_dtype;
  if (in != GB_DTYPE_F32 && in != GB_DTYPE_BF16 && in != GB_DTYPE_F16)
    return set_error(GB_ERR_INVALID_ARG, "unknown in_dtype %d", in);
  if (args->n_heads < 0 || args->n_heads > 16384)
    return set_error(GB_ERR_INVALID_ARG, "n_heads %d not in 0..16384", args->n_heads);
  if (args->rot_dim < 0 || args->rot_dim % 16 || args->rot_dim > batch->head_dim)
    return set_error(GB_ERR_UNSUPPORTED, "rot_dim %d: a multiple of 16 from 0 to head_dim %d",
                     args->rot_dim, batch->head_dim);
  if (!(args->eps >= 0.0f)) return set_error(GB_ERR_INVALID_ARG, "eps must be >= 0");
  if (args->table_rows < 0) return set_error(GB_ERR_INVALID_ARG, "table_rows < 0");
  if (batch->n_seqs == 0 || batch->total_q == 0) return GB_OK;
  const bool q = args->n_heads > 0;
  if ((q && (!args->q_dev || !args->q_out_dev)) || !args->k_dev || !args->v_dev ||
      !args->k_pool_dev || !args->v_pool_dev)
    return set_error(GB_ERR_INVALID_ARG, "q, q_out, k, v and the pools must not be null");
  if (args->rot_dim && (!args->cos_dev || !args->sin_dev))
    return set_error(GB_ERR_INVALID_ARG, "rot_dim %d needs cos and sin", args->rot_dim);
  const int64_t es = in == GB_DTYPE_F32 ? 4 : 2;
  if ((q && (!aligned16(args->q_dev) || !aligned16(args->q_out_dev))) || !aligned16(args->k_dev) ||
      !aligned16(args->v_dev) || !aligned16(args->k_pool_dev) || !aligned16(args->v_pool_dev) ||
      !aligned16(args->q_norm_dev) || !aligned16(args->k_norm_dev) || !aligned16(args->cos_dev) ||
      !aligned16(args->sin_dev))
    return set_error(GB_ERR_INVALID_ARG, "every buffer must be 16-byte aligned");
  if ((q && (!stride_ok(args->q_row_stride, es) || !stride_ok(args->q_head_stride, es) ||
             !stride_ok(args->out_row_stride, 2) || !stride_ok(args->out_head_stride, 2))) ||
      !stride_ok(args->k_row_stride, es) || !stride_ok(args->k_head_stride, es) ||
      !stride_ok(args->v_row_stride, es) || !stride_ok(args->v_head_stride, es))
    return set_error(GB_ERR_INVALID_ARG,
                     "row and head strides must be non-negative multiples of 16 bytes");
  if (q && ((batch->total_q > 1 && args->out_row_stride < batch->head_dim) ||
            (args->n_heads > 1 && args->out_head_stride < batch->head_dim)))
    return set_error(GB_ERR_INVALID_ARG, "q_out's strides must be at least head_dim");
  if (q && args->q_out_dev == args->q_dev &&
      (in != batch->dtype || args->out_row_stride != args->q_row_stride ||
       args->out_head_stride != args->q_head_stride))
    return set_error(GB_ERR_INVALID_ARG, "q_out may be q only in the same type and strides");
  a.nh = args->n_heads;
  a.hd = batch->head_dim;
  a.rot = args->rot_dim;
  a.units = (int64_t)batch->total_q * (a.nh + 2 * batch->n_kv_heads);
  if (a.units / (kRopeThreads / 32) >= 0x7fffffffll)
    return set_error(GB_ERR_UNSUPPORTED, "too many rows x heads for one call");
  a.q = args->q_dev, a.k = args->k_dev, a.v = args->v_dev;
  a.q_row = args->q_row_stride, a.q_head = args->q_head_stride;
  a.k_row = args->k_row_stride, a.k_head = args->k_head_stride;
  a.v_row = args->v_row_stride, a.v_head = args->v_head_stride;
  a.q_out = args->q_out_dev;
  a.o_row = args->out_row_stride, a.o_head = args->out_head_stride;
  a.q_norm = args->q_norm_dev, a.k_norm = args->k_norm_dev;
  a.cos_t = args->cos_dev, a.sin_t = args->sin_dev;
  a.table_rows = args->table_rows;
  a.k_pool = args->k_pool_dev, a.v_pool = args->v_pool_dev;
  a.eps = args->eps;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = batch->dtype == GB_DTYPE_BF16 ? launch_rope_in<__nv_bfloat16>(a, in, st)
                                                      : launch_rope_in<__half>(a, in, st);
  if (e != cudaSuccess)
    return set_error(GB_ERR_CUDA, "rope_append launch: %s", cudaGetErrorString(e));
  return GB_OK;
}

extern "C" int gb_paged_copy(void* const* pools_dev, int32_t n_pools, int64_t n_pages,
                             int64_t page_bytes, int64_t page_stride, const int32_t* src,
                             const int32_t* dst, int32_t n, void* stream) {
  using namespace gb;
  using namespace gb::paged;
  if (n_pools < 0 || n < 0) return set_error(GB_ERR_INVALID_ARG, "n_pools and n must be >= 0");
  if (n_pages < 1 || n_pages > 0x7fffffffll)
    return set_error(GB_ERR_INVALID_ARG, "n_pages must be in 1..2^31 - 1");
  if (page_bytes < 16 || page_bytes % 16 || page_stride % 16 || page_stride < page_bytes)
    return set_error(GB_ERR_INVALID_ARG,
                     "page_bytes and page_stride must be multiples of 16, page_stride >= page_bytes");
  if (page_bytes > (int64_t)1 << 30) return set_error(GB_ERR_UNSUPPORTED, "pages above 1 GiB");
  if (n_pools == 0 || n == 0) return GB_OK;
  if (!pools_dev || !src || !dst)
    return set_error(GB_ERR_INVALID_ARG, "pools, src and dst must not be null");
  for (int p = 0; p < n_pools; ++p)
    if (!pools_dev[p] || !aligned16(pools_dev[p]))
      return set_error(GB_ERR_INVALID_ARG, "pool %d is null or not 16-byte aligned", p);
  // every dst once, and none of them a src: the copies then commute
  try {
    std::vector<int32_t> d(dst, dst + n);
    std::sort(d.begin(), d.end());
    if (d.front() < 0 || d.back() >= n_pages)
      return set_error(GB_ERR_INVALID_ARG, "a dst page is outside [0, %lld)", (long long)n_pages);
    for (int i = 1; i < n; ++i)
      if (d[i] == d[i - 1])
        return set_error(GB_ERR_INVALID_ARG, "page %d is written twice", d[i]);
    for (int i = 0; i < n; ++i) {
      if (src[i] < 0 || src[i] >= n_pages)
        return set_error(GB_ERR_INVALID_ARG, "src page %d is outside [0, %lld)", src[i],
                         (long long)n_pages);
      if (std::binary_search(d.begin(), d.end(), src[i]))
        return set_error(GB_ERR_INVALID_ARG, "page %d is both read and written", src[i]);
    }
  } catch (const std::bad_alloc&) {
    return set_error(GB_ERR_NO_MEMORY, "host memory for the page check");
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // parameters of 1.1 KB for a fork's few pages, of 18 KB for a compaction
  const cudaError_t e =
      n <= 64 && n_pools <= 64
          ? launch_copy<64, 64>(pools_dev, n_pools, page_bytes, page_stride, src, dst, n, st)
          : launch_copy<256, 2048>(pools_dev, n_pools, page_bytes, page_stride, src, dst, n, st);
  if (e != cudaSuccess) return set_error(GB_ERR_CUDA, "page copy launch: %s", cudaGetErrorString(e));
  return GB_OK;
}
