// Device helpers of the paged key/value cache's kernels: a sequence's place in a step, pool rows, and the 4-bit
// format's values.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "kvcache.h"
#include "ptx.cuh"

namespace jc {

// One sequence's new rows and cached length, held to the call's bounds. What lies outside them (start not rising
// within the packed rows, more new tokens than max_new, a length below 0 or above max_length or the table) sets
// the error bit, and the sequence then has no new tokens here: nothing of it is read or written.
struct KvSeq {
  int row0, n, length;
};

__device__ __forceinline__ KvSeq kv_seq(const KvStep& st, int page_size, int s, uint32_t* err) {
  KvSeq q;
  int r1;
  if (st.start) {
    q.row0 = __ldg(st.start + s);
    r1 = __ldg(st.start + s + 1);
  } else {
    q.row0 = s;
    r1 = s + 1;
  }
  q.length = __ldg(st.length + s);
  const bool bad = q.row0 < 0 || r1 < q.row0 || r1 > st.tokens || r1 - q.row0 > st.max_new || q.length < 0 ||
                   q.length > st.max_length || q.length > static_cast<long long>(st.table_pages) * page_size;
  q.n = bad ? 0 : r1 - q.row0;
  if (bad) atomicOr(err, kErrKvStep);
  return q;
}

// First pool row of kv head h of the page that holds index t of sequence s, or −1 (an entry outside the pool).
__device__ __forceinline__ long long kv_page_row(const KvCache& c, const int* table_row, int page, int h) {
  const int id = __ldg(table_row + page);
  if (id < 0 || id >= c.pages) return -1;
  return (static_cast<long long>(id) * c.kv_heads + h) * c.page_size;
}

template <typename T>
__device__ __forceinline__ float kv_float(T x) {
  if constexpr (std::is_same<T, __half>::value)
    return __half2float(x);
  else
    return __bfloat162float(x);
}

// FP16 stores saturate at ±65504 as the library's others do; a NaN stays one.
template <typename T>
__device__ __forceinline__ T kv_round(float x) {
  if constexpr (std::is_same<T, __half>::value)
    return __float2half_rn(x > 65504.0f ? 65504.0f : x < -65504.0f ? -65504.0f : x);
  else
    return __float2bfloat16_rn(x);
}

template <typename T>
__device__ __forceinline__ float2 kv_unpack(uint32_t u) {
  if constexpr (std::is_same<T, __half>::value)
    return __half22float2(*reinterpret_cast<__half2*>(&u));
  else
    return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&u));
}

// Two values as kv_round does one: rounded to infinity past the range, which the two-wide minimum and maximum (keeping
// NaN) bring back to ±65504.
template <typename T>
__device__ __forceinline__ uint32_t kv_pack(float a, float b) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 most = __half2half2(__ushort_as_half(0x7BFF)), least = __half2half2(__ushort_as_half(0xFBFF));
    const __half2 h = __hmax2_nan(__hmin2_nan(__floats2half2_rn(a, b), most), least);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

// 16 bytes of rows that the same kernel may write (a call in place): not the read-only path of __ldg. A thread's loads may
// still move past other rows' stores, which are to other addresses.
__device__ __forceinline__ uint4 kv_load16(const void* p) {
  uint4 v;
  asm("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// The smaller (larger) of two values, NaN if either is one.
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The value that 4-bit code c stands for: fp16(c · scale + min), one rounding (c is exact in FP16).
__device__ __forceinline__ __half kv_code_value(uint32_t c, __half2 sm) {
  return __hfma(__ushort2half_rn(static_cast<unsigned short>(c)), __low2half(sm), __high2half(sm));
}

}  // namespace jc
