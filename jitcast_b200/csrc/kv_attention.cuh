// What the cache attention's kernels share: which keys a token sees, the ranges of 16-key blocks that a tile of
// query rows reads, and the row-by-row form that recomputes a row whose result is not a number.
#pragma once

#include "kvcache.cuh"

namespace jc {

// The keys that index t sees are [0, sink) and [first, t + 1).
__device__ __forceinline__ int kv_first(const KvAttnArgs& a, int t) {
  return a.window > 0 && t + 1 > a.window ? t + 1 - a.window : 0;
}

// The blocks of 2^shift keys that the tokens t0 .. t1 of one sequence read: blocks 0 .. a − 1 (sinks), then
// b .. b + n − a − 1; n in all, none twice. A page holds a whole number of blocks.
struct KvBlocks {
  int a, b, n;
  __device__ __forceinline__ int at(int x) const { return x < a ? x : x - a + b; }
};

__device__ __forceinline__ KvBlocks kv_blocks(const KvAttnArgs& a, int t0, int t1, int shift) {
  KvBlocks k;
  if (t1 < 0) return KvBlocks{0, 0, 0};
  k.b = kv_first(a, t0 < 0 ? 0 : t0) >> shift;
  const int sink = a.sinks < t1 + 1 ? a.sinks : t1 + 1;
  k.a = (sink >> shift) + ((sink & ((1 << shift) - 1)) != 0 ? 1 : 0);
  if (k.a > k.b) k.a = k.b;
  k.n = k.a + (t1 >> shift) - k.b + 1;
  return k;
}

// Blocks x0 .. x1 − 1 of those.
struct KvSlice {
  int a, b, n, o;
  __device__ __forceinline__ KvSlice(const KvBlocks& k, int x0, int x1)
      : a(k.a > x0 ? k.a - x0 : 0), b(k.a > x0 ? k.b : k.b + x0 - k.a), n(x1 - x0), o(x0) {}
  __device__ __forceinline__ int at(int x) const { return x < a ? x + o : x - a + b; }
};

// The partial results of split s of output row r (token · heads + head): O [splits][rows][D], then (max, sum).
__device__ __forceinline__ float* part_o(const KvAttnArgs& a, int split, long long row, int D) {
  return a.workspace + (split * (static_cast<long long>(a.st.tokens) * a.heads) + row) * D;
}
__device__ __forceinline__ float2* part_ml(const KvAttnArgs& a, int splits, int split, long long row, int D) {
  const long long rows = static_cast<long long>(a.st.tokens) * a.heads;
  return reinterpret_cast<float2*>(a.workspace + splits * rows * D) + split * rows + row;
}

// One row of the output by one warp, key by key on the CUDA cores in FP32 (lane l holds dims l, l + 32, ..),
// with the running maximum and sum of the softmax. It reads visible keys alone. The tiled kernels multiply a hidden
// key's value by a probability of 0, which is NaN for an infinite or undefined value; they hand a row that comes
// out with a NaN to this form, so hidden values stay out of every result and a visible NaN stays in it. So do they with
// a row whose sum is 0: no key of it was there (zeros), or every score is -inf (NaN, as 0 / 0 is).
template <typename T, int BITS, int D>
__device__ __noinline__ void kv_attend_row(const KvAttnArgs& a, int s, int t, int head, const T* q, T* out) {
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
  bool seen = false;
  const int first = kv_first(a, t), sink = a.sinks < first ? a.sinks : first;
  for (int j = sink > 0 ? 0 : first; j <= t; j = j + 1 == sink ? first : j + 1) {
    const long long page = kv_page_row(a.c, table, j / a.c.page_size, kvh);
    if (page < 0) {
      if (lane == 0) atomicOr(a.err, kErrKvStep);
      continue;
    }
    seen = true;
    const long long row = page + j % a.c.page_size;
    float d = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) d = fmaf(x[i], kv_value<T, BITS>(a.c.k, a.c.k_scale, row, D, lane + 32 * i), d);
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) d += __shfl_xor_sync(0xffffffffu, d, w);
    const float mn = fmaxf(m, d);
    const float up = mn == -INFINITY ? 1.0f : __expf(m - mn);  // −inf − −inf would be NaN
    const float p = d != d ? d : mn == -INFINITY ? 0.0f : __expf(d - mn);  // an undefined score stays, whatever came before
    l = l * up + p;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = o[i] * up + p * kv_value<T, BITS>(a.c.v, a.c.v_scale, row, D, lane + 32 * i);
    m = mn;
  }
  const float inv = l != 0.0f ? 1.0f / l : seen ? NAN : 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) out[lane + 32 * i] = kv_round<T>(o[i] * inv);
}

// Codes at bits 0..3 and 16..19 (HIGH: 4..7 and 20..23) of u as FP16: (1024 + c) − 1024, or (1024 + 16 c) / 16 − 64,
// both exact.
template <bool HIGH>
__device__ __forceinline__ __half2 kv_codes(uint32_t u) {
  const uint32_t x = (u & (HIGH ? 0x00F000F0u : 0x000F000Fu)) | 0x64006400u;
  const uint32_t c1 = 0x64006400u, c2 = 0x2C002C00u, c3 = 0xD400D400u;  // 1024; 1/16, −64
  const __half2 h = *reinterpret_cast<const __half2*>(&x);
  if constexpr (HIGH)
    return __hfma2(h, *reinterpret_cast<const __half2*>(&c2), *reinterpret_cast<const __half2*>(&c3));
  else
    return __hsub2(h, *reinterpret_cast<const __half2*>(&c1));
}

// 2^x by the special-function unit: 2 ulp, flushes subnormal results (a probability below 2^-126 is none).
__device__ __forceinline__ float kv_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Probabilities that go into a product as FP16 are taken 2^7 times as large, and their sums with them: one below 2^-25
// rounds to 0 in FP16, and 131,000 keys just under that beside one large one are 1/250 of a row's weight. So the bound is
// 2^-32, 1/30,000 of it. With a maximum that lags by 2^8 at most they stay below 2^15. BF16 has the range as it is.
template <typename M>
constexpr float kProbUp = std::is_same<M, __half>::value ? 7.0f : 0.0f;

// Division of 0 <= u < 2^27 (a 16-key block of a 31-bit length) by a page's blocks, as a product: m = 2^32 / d
// rounded up is off by less than one in d · m, so u · m / 2^32 is exact while u · d < 2^32 (d <= 32, pages of up to 512
// tokens) and larger pages divide.
struct KvDiv {
  unsigned d;
  unsigned long long m;
  __host__ __device__ KvDiv(unsigned by = 1) : d(by), m((1ull << 32) / by + ((1ull << 32) % by ? 1 : 0)) {}
  __device__ __forceinline__ unsigned of(unsigned u) const {
    return d <= 32 ? static_cast<unsigned>((u * m) >> 32) : u / d;
  }
};

// Joins what a kernel's splits left in the workspace: rows in tiles of rows_per_tile, at most `chunk` blocks of 2^shift
// keys a split (a tile with no more than that wrote its rows itself).
cudaError_t launch_kv_join(const KvAttnArgs& a, int shift, int chunk, int splits, int rows_per_tile, cudaStream_t s);

// Splits of the keys that the tiles of this call take, and the workspace of any split.
int kv_tile_splits(const KvAttnArgs& a);
inline long long kv_split_bytes(const KvAttnArgs& a, long long splits) {
  return splits * a.st.tokens * a.heads * (a.c.dim + 2) * 4;
}

}  // namespace jc
