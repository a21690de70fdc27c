// Shared by the serving operators (qkrope.cu, attn.cu, attn_tc.cu, sample.cu): the paged cache as the kernels take it, the
// row a sequence's tokens stand in, and conversions of the half-precision types.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/clb200.h"
#include "common.cuh"

namespace clb {

constexpr uint32_t T_BF16 = CLB200_T_BF16;

template <typename T>
CLB_DEV float to_f32(T v);
template <>
CLB_DEV float to_f32<float>(float v) { return v; }
template <>
CLB_DEV float to_f32<__half>(__half v) { return __half2float(v); }
template <>
CLB_DEV float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
CLB_DEV T from_f32(float v);
template <>
CLB_DEV float from_f32<float>(float v) { return v; }
template <>
CLB_DEV __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
CLB_DEV __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Two floats rounded to a half-precision type, a in the low half.
template <typename C>
CLB_DEV uint32_t pack2(float a, float b) {
  if constexpr (__is_same(C, __half)) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
  } else if constexpr (__is_same(C, __nv_bfloat16)) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
  } else {
    return 0;   // not reached: floats are not packed
  }
}

// Four floats times f, rounded to O (16 or 8 bytes, aligned).
template <typename O>
CLB_DEV void store4(O *p, float4 v, float f) {
  if constexpr (sizeof(O) == 4) {
    *reinterpret_cast<float4 *>(p) = make_float4(v.x * f, v.y * f, v.z * f, v.w * f);
  } else {
    uint2 w;
    O *h = reinterpret_cast<O *>(&w);
    h[0] = from_f32<O>(v.x * f); h[1] = from_f32<O>(v.y * f); h[2] = from_f32<O>(v.z * f); h[3] = from_f32<O>(v.w * f);
    *reinterpret_cast<uint2 *>(p) = w;
  }
}

// The last s in [0, n_seq) with q_start[s] <= row, by bisection: the sequence whose rows hold `row` when q_start does not
// descend and q_start[0] <= row < q_start[n_seq] (sequences without rows are passed over). Reads inside q_start whatever it
// holds.
CLB_DEV int seq_of_row(const int *q_start, int n_seq, int row) {
  int lo = 0, hi = n_seq - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (q_start[mid] <= row) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// The page that holds position pos of sequence s, or -1 (and the error word set) when the table does not reach it or names
// no page.
CLB_DEV int page_of(const clb200_kv &kv, int s, int pos, int *err) {
  const int i = pos / kv.page_size;
  int page = -1;
  if (pos >= 0 && i < kv.table_width) page = kv.table[static_cast<int64_t>(s) * kv.table_stride + i];
  if (page < 0 || page >= kv.n_pages) {
    set_error(err, ERR_BAD_PAGE);
    return -1;
  }
  return page;
}

constexpr unsigned FULL_MASK = 0xffffffffu;

// Host: 0 when the cache description can be used, 1 with err set (nothing it points to is read).
int check_kv(const clb200_kv *kv, char *err, size_t errlen);

// Host: query heads per key/value head that the attention takes.
constexpr int ATTN_MAX_GROUP = 16;

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Host: whether [a, a + n) and [b, b + m) (bytes) share a byte.
inline bool overlap(const void *a, size_t n, const void *b, size_t m) {
  const auto x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + m && y < x + n;
}

// Host: makes a device current for a call and gives the caller's back afterwards.
struct OnDevice {
  int before = -1;
  explicit OnDevice(int device) {
    if (cudaGetDevice(&before) != cudaSuccess || before == device) before = -1;
    else cudaSetDevice(device);
  }
  ~OnDevice() {
    if (before >= 0) cudaSetDevice(before);
  }
};

}  // namespace clb
