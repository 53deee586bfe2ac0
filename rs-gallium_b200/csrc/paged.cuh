// paged.cuh -- the paged KV cache's batch as the kernels see it (gb_paged_batch):
// bounds-checked lengths, page numbers and addresses, and the element types.
#pragma once

#include "common.cuh"
#include "moe_internal.h"

namespace gb {
namespace paged {

struct Batch {
  int n_seqs, total_q, max_q, max_kv;
  int nkv, page_shift, n_pages;
  int64_t page_stride, slot_stride, head_stride;  // elements
  const int32_t* q_start;
  const int32_t* kv_len;
  const int32_t* table;
  int64_t table_stride;
  int* err;
};

// Host: validates the descriptor (no device access) and fills `b`.
int check_batch(const gb_paged_batch* d, Batch* b);

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Strides that keep every vector of 8 elements (16 bytes of a 2-byte type) aligned.
inline bool stride_ok(int64_t s, int64_t elem_bytes) { return s >= 0 && (s * elem_bytes) % 16 == 0; }

__device__ __forceinline__ void flag(const Batch& b, int bit) {
  if (b.err) atomicOr(b.err, bit);
}

// Sequence s's rows and cached positions, clamped to what the arrays hold.
struct Seq {
  int row0, q_len, kv_len;
};
__device__ __forceinline__ Seq load_seq(const Batch& b, int s, bool report) {
  const int a = __ldg(b.q_start + s), e = __ldg(b.q_start + s + 1), kv = __ldg(b.kv_len + s);
  Seq r;
  r.row0 = min(max(a, 0), b.total_q);
  r.q_len = min(max(e, r.row0), b.total_q) - r.row0;
  const int64_t held = b.table_stride << b.page_shift;
  const int cap = held < b.max_kv ? (int)held : b.max_kv;
  r.kv_len = min(max(kv, 0), cap);
  if (report && (a != r.row0 || e != r.row0 + r.q_len || kv != r.kv_len || r.q_len > b.max_q))
    flag(b, GB_PAGED_BAD_LENGTH);
  return r;
}

// 2-byte element types of the pools.
template <typename T>
struct Elem;
template <>
struct Elem<__nv_bfloat16> {
  static constexpr int kType = GB_DTYPE_BF16;
  // log2 of the weight that a softmax gives its maximum: f16 weights of 2^8 keep
  // those down to 2^-22 of the maximum normal; bf16 has f32's range.
  static constexpr float kTop = 0.0f;
  static constexpr uint32_t kExpMask = 0x7f80u;  // all ones: inf or NaN
  __device__ static __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  __device__ static __forceinline__ float2 unpack(uint32_t u) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  }
};
template <>
struct Elem<__half> {
  static constexpr int kType = GB_DTYPE_F16;
  static constexpr float kTop = 8.0f;
  static constexpr uint32_t kExpMask = 0x7c00u;
  __device__ static __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  __device__ static __forceinline__ float2 unpack(uint32_t u) {
    return __half22float2(*reinterpret_cast<const __half2*>(&u));
  }
};

}  // namespace paged
}  // namespace gb
