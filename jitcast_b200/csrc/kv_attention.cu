// Attention of new tokens over the paged key/value cache: causal, with a sliding window and sinks.
//
// Token t of a sequence sees the keys j ≤ t with j > t − window (window 0: all) or j < sinks;
// out = Σ_j softmax_j(scale · q·k_j) · v_j, zeros where a token sees no key.
#include "kvcache.cuh"

namespace jc {

namespace {

// The keys that index t sees are [0, head) and [first, t + 1).
__device__ __forceinline__ void kv_visible(const KvAttnArgs& a, int t, int& head, int& first) {
  first = a.window > 0 && t + 1 > a.window ? t + 1 - a.window : 0;
  head = a.sinks < first ? a.sinks : first;
}

// One row of the output by one warp, key by key on the CUDA cores in FP32 (lane l holds dims l, l + 32, ..),
// with the running maximum and sum of the softmax. Only visible keys are read, so whatever lies in hidden ones
// (infinities, NaN) stays out.
template <typename T, int BITS, int D>
__device__ void kv_attend_row(const KvAttnArgs& a, int s, int t, int head, const T* q, T* out) {
  constexpr int N = D / 32;
  const int lane = threadIdx.x & 31;
  const int kvh = head / (a.heads / a.c.kv_heads);
  const int* table = a.st.table + s * a.st.ld_table;
  float x[N], o[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    x[i] = kv_float(q[lane + 32 * i]) * a.scale;
    o[i] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  int sink, first;
  kv_visible(a, t, sink, first);
  for (int j = sink > 0 ? 0 : first; j <= t; j = j + 1 == sink ? first : j + 1) {
    const long long page = kv_page_row(a.c, table, j / a.c.page_size, kvh);
    if (page < 0) {
      if (lane == 0) atomicOr(a.err, kErrKvStep);
      continue;
    }
    const long long row = page + j % a.c.page_size;
    float d = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) d = fmaf(x[i], kv_value<T, BITS>(a.c.k, a.c.k_scale, row, D, lane + 32 * i), d);
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) d += __shfl_xor_sync(0xffffffffu, d, w);
    const float mn = fmaxf(m, d);
    const float up = mn == -INFINITY ? 1.0f : __expf(m - mn);  // −inf − −inf would be NaN
    const float p = mn == -INFINITY ? 0.0f : d != d ? d : __expf(d - mn);
    l = l * up + p;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = o[i] * up + p * kv_value<T, BITS>(a.c.v, a.c.v_scale, row, D, lane + 32 * i);
    m = mn;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int i = 0; i < N; ++i) out[lane + 32 * i] = kv_round<T>(o[i] * inv);
}

template <typename T, int BITS, int D>
__global__ void __launch_bounds__(128) kv_attention_rows_kernel(const KvAttnArgs a) {
  const int warp = threadIdx.x >> 5;
  const int s = blockIdx.z, h = blockIdx.x * 4 + warp;
  const KvSeq q = kv_seq(a.st, a.c.page_size, s, a.err);
  if (h >= a.heads) return;
  for (int i = blockIdx.y; i < q.n; i += gridDim.y) {
    const long long row = q.row0 + i;
    const T* x = static_cast<const T*>(a.q.p) + row * a.q.ld + h * a.q.hs;
    T* o = static_cast<T*>(a.out.p) + row * a.out.ld + h * a.out.hs;
    kv_attend_row<T, BITS, D>(a, s, q.length - q.n + i, h, x, o);
  }
}

template <typename T, int BITS, int D>
void attend(const KvAttnArgs& a, cudaStream_t s) {
  const dim3 grid((a.heads + 3) / 4, a.st.max_new < 65535 ? a.st.max_new : 65535, a.st.sequences);
  kv_attention_rows_kernel<T, BITS, D><<<grid, 128, 0, s>>>(a);
}

}  // namespace

long long kv_attention_workspace(const KvAttnArgs&) { return 0; }

cudaError_t launch_kv_attention(const KvAttnArgs& a, cudaStream_t s) {
  if (a.st.sequences == 0 || a.st.max_new == 0) return cudaSuccess;
  if (a.c.bits == 16) {
    if (a.c.dim == 64)
      a.c.f16 ? attend<__half, 16, 64>(a, s) : attend<__nv_bfloat16, 16, 64>(a, s);
    else
      a.c.f16 ? attend<__half, 16, 128>(a, s) : attend<__nv_bfloat16, 16, 128>(a, s);
  } else {
    if (a.c.dim == 64)
      a.c.f16 ? attend<__half, 4, 64>(a, s) : attend<__nv_bfloat16, 4, 64>(a, s);
    else
      a.c.f16 ? attend<__half, 4, 128>(a, s) : attend<__nv_bfloat16, 4, 128>(a, s);
  }
  return cudaGetLastError();
}

}  // namespace jc
