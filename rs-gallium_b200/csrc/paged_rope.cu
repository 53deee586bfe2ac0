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
// the halves-layout rotation, q to q_out, k and v to their pages.  The work is
// a list of (row, head) units, rows of nh + 2 nkv heads; a group of
// head_dim / 8 lanes takes one unit, 8 elements (16 bytes of a 2-byte type) a
// lane, so a warp's loads and stores are whole 128-byte lines.  The rotation
// pairs element j with j + rot / 2, which another lane of the group holds at a
// fixed lane distance (rot / 16), so one shuffle per element exchanges them.
// Bound by memory: each element is read once and written once.  The rows'
// sequences and slots are looked up by one warp per row (32-way search of
// q_start) while the first loads of q, k and v, which need neither, are in
// flight.

constexpr int kRopeThreads = 256;

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

// U units of each lane group in flight.
template <typename In, typename Out, int HD, int U>
__global__ void __launch_bounds__(kRopeThreads) rope_append_kernel(const __grid_constant__ RopeArgs a) {
  constexpr int L = HD / 8;                // lanes per unit
  constexpr int G = kRopeThreads / L;      // units per pass of the CTA
  constexpr int kMaxRows = G * U;          // rows a CTA's units can touch
  __shared__ RowInfo rows[kMaxRows];
  const int heads = a.nh + 2 * a.b.nkv;
  const int64_t unit0 = (int64_t)blockIdx.x * (G * U);
  const int64_t last = min(unit0 + G * U, a.units) - 1;
  const int row0 = (int)(unit0 / heads), n_rows = (int)(last / heads) - row0 + 1;
  const int grp = threadIdx.x / L, gl = threadIdx.x % L, d = gl * 8;
  Load8<In> x[U];
  int row[U], head[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t unit = unit0 + u * G + grp;
    row[u] = -1;
    head[u] = 0;
    if (unit <= last) {
      row[u] = (int)(unit / heads);
      head[u] = (int)(unit - (int64_t)row[u] * heads);
      const int h = head[u];
      if (h < a.nh)
        x[u].load(a.q, row[u] * a.q_row + h * a.q_head + d);
      else if (h < a.nh + a.b.nkv)
        x[u].load(a.k, row[u] * a.k_row + (h - a.nh) * a.k_head + d);
      else
        x[u].load(a.v, row[u] * a.v_row + (h - a.nh - a.b.nkv) * a.v_head + d);
    }
  }
  for (int i = threadIdx.x >> 5; i < n_rows; i += kRopeThreads / 32) {
    const RowInfo r = find_row(a.b, row0 + i, a.rot ? a.table_rows : INT64_MAX, threadIdx.x & 31);
    if ((threadIdx.x & 31) == 0) rows[i] = r;
  }
  __syncthreads();
  const int half = a.rot / 2;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int h = head[u];
    const bool live = row[u] >= 0;
    const RowInfo info = live ? rows[row[u] - row0] : RowInfo{-1, 0, -1};
    const bool is_q = h < a.nh, is_v = h >= a.nh + a.b.nkv;
    float y[8];
    if (live) {
      x[u].get(y);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = 0.0f;
    }
    const float* w = is_v ? nullptr : is_q ? a.q_norm : a.k_norm;
    if (a.q_norm || a.k_norm) {  // the same on every lane: the shuffles meet
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = __fmaf_rn(y[i], y[i], ss);
#pragma unroll
      for (int o = L / 2; o >= 1; o >>= 1) ss += __shfl_xor_sync(kFullMask, ss, o);
      if (w) {
        const float m = sqrtf(__fadd_rn(__fmul_rn(ss, 1.0f / HD), a.eps));
        const float4 w0 = *reinterpret_cast<const float4*>(w + d);
        const float4 w1 = *reinterpret_cast<const float4*>(w + d + 4);
        const float ws[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = __fmul_rn(__fdiv_rn(y[i], m), ws[i]);
      }
    }
    if (half) {
      const int lane = threadIdx.x & 31, gap = half / 8;  // lanes to the partner
      const bool first = gl < gap;
      const int partner = first ? lane + gap : gl < 2 * gap ? lane - gap : lane;
      float other[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) other[i] = __shfl_sync(kFullMask, y[i], partner);
      if (!is_v && gl < 2 * gap && info.pos >= 0) {
        const int64_t at = (int64_t)info.pos * half + (first ? d : d - half);
        const float4* c4 = reinterpret_cast<const float4*>(a.cos_t + at);
        const float4* s4 = reinterpret_cast<const float4*>(a.sin_t + at);
        const float4 c0 = c4[0], c1 = c4[1], s0 = s4[0], s1 = s4[1];
        const float cs[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
        const float sn[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
        for (int i = 0; i < 8; ++i)
          y[i] = first ? __fsub_rn(__fmul_rn(y[i], cs[i]), __fmul_rn(other[i], sn[i]))
                       : __fadd_rn(__fmul_rn(other[i], sn[i]), __fmul_rn(y[i], cs[i]));
      }
    }
    if (!live || info.pos < 0) continue;
    uint4 o;
    o.x = Elem<Out>::pack(y[0], y[1]);
    o.y = Elem<Out>::pack(y[2], y[3]);
    o.z = Elem<Out>::pack(y[4], y[5]);
    o.w = Elem<Out>::pack(y[6], y[7]);
    if (is_q) {
      *reinterpret_cast<uint4*>(static_cast<Out*>(a.q_out) + row[u] * a.o_row + h * a.o_head + d) = o;
    } else if (info.page >= 0) {
      const int g = is_v ? h - a.nh - a.b.nkv : h - a.nh;
      Out* pool = static_cast<Out*>(is_v ? a.v_pool : a.k_pool);
      *reinterpret_cast<uint4*>(pool + info.page + info.slot * a.b.slot_stride +
                                g * a.b.head_stride + d) = o;
    }
  }
}

template <typename In, typename Out, int HD>
cudaError_t launch_rope(const RopeArgs& a, cudaStream_t st) {
  constexpr int G = kRopeThreads / (HD / 8);
  // Few units: one per lane group, so that they spread over the SMs.
  if (a.units <= (int64_t)G * 148 * 4) {
    rope_append_kernel<In, Out, HD, 1><<<(unsigned)((a.units + G - 1) / G), kRopeThreads, 0, st>>>(a);
  } else {
    rope_append_kernel<In, Out, HD, 4>
        <<<(unsigned)((a.units + 4 * G - 1) / (4 * G)), kRopeThreads, 0, st>>>(a);
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
