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

// Dims d .. d + 7 (d a multiple of 8) of pool row `row`, loaded, and as FP32: zeros where not `here`, whatever the row holds.
template <typename T, int BITS, int D>
struct KvEight {
  uint4 u;  // 16 bits: the values; 4 bits: x has the codes, y their (scale, min)

  __device__ __forceinline__ void load(const void* pool, const void* scale, int row, int d) {
    if constexpr (BITS == 16) {
      u = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(pool) + row * static_cast<long long>(D) + d));
    } else {
      u.x = __ldg(static_cast<const uint32_t*>(pool) + row * static_cast<long long>(D / 8) + d / 8);
      u.y = __ldg(static_cast<const uint32_t*>(scale) + row * static_cast<long long>(D / kKvGroup) + d / kKvGroup);
    }
  }
  __device__ __forceinline__ void values(bool here, float (&v)[8]) const {
    if constexpr (BITS == 16) {
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = kv_unpack<T>(here ? w[e] : 0u);
        v[2 * e] = f.x, v[2 * e + 1] = f.y;
      }
    } else {
      const uint32_t y = here ? u.y : 0u;
      const __half2 s = __low2half2(*reinterpret_cast<const __half2*>(&y)), m = __high2half2(*reinterpret_cast<const __half2*>(&y));
#pragma unroll
      for (int e = 0; e < 4; ++e) {  // dims e and e + 4
        const uint32_t w = e < 2 ? u.x : u.x >> 8;
        const float2 f = __half22float2(__hfma2(e & 1 ? kv_codes<true>(w) : kv_codes<false>(w), s, m));
        v[e] = f.x, v[e + 4] = f.y;
      }
    }
  }
};

__device__ __forceinline__ float kv_warp_max(float x) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}

// The row-by-row form: groups part, part + parts, .. of 32 of the keys that a row sees, by one warp on the CUDA cores in
// FP32, with the running maximum m and sum l of the softmax (o: dims 8 c .. 8 c + 7 and those 64 further, c = lane % 8, of its
// numerator). It reads visible keys alone. The tiled kernels multiply a hidden key's value by a probability of 0, which is NaN
// for an infinite or undefined value; they hand a row that comes out with a NaN to this form, so hidden values stay out of
// every result and a visible NaN stays in it. So do they with a row whose sum is 0: no key of it was there (zeros), or every
// score is -inf (NaN, as 0 / 0 is).
// Eight lanes take a key's row, so four whole rows a load; in step e the lanes 8 g .. 8 g + 7 have key 8 g + e, and keep its
// score in lane 8 g + e. An undefined score makes the whole row undefined and ends the walk. (A prompt of 4,096 with every
// row worked out again, 4 heads of 64: 4.8 ms, over 4 bits 5.2, where the call takes 0.08: the latencies of a group's chain, 32 rows
// a warp. Key after key it took 58 and 60, with a lane a key's row 6.6.)
template <typename T, int BITS, int D>
__device__ __forceinline__ void kv_attend_keys(const KvAttnArgs& a, int s, int t, int head, const T* q, int part, int parts,
                                               float& m, float& l, float (&o)[D / 64][8], bool& seen) {
  constexpr int N = D / 64;
  constexpr int FLY = BITS == 16 && N == 2 ? 4 : 8;  // rows that a lane has in flight: 32 registers
  const int lane = threadIdx.x & 31, c = lane & 7, g8 = lane & 24;
  const int kvh = head / (a.heads / a.c.kv_heads);
  const int* table = a.st.table + s * a.st.ld_table;
  float x[N][8];
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[i][e] = kv_float(q[64 * i + 8 * c + e]) * a.scale;
      o[i][e] = 0.0f;
    }
  m = -INFINITY, l = 0.0f, seen = false;
  const int first = kv_first(a, t), sink = a.sinks < first ? a.sinks : first;
  const int keys = t < 0 ? 0 : sink + (t - first) + 1;  // [0, sink) and [first, t]
  // the lane's key of the group from k0 in the pool; -1: none. Looked up a group ahead.
  auto row_of = [&](long long k0) -> int {
    if (k0 + lane >= keys) return -1;
    const int k = static_cast<int>(k0) + lane, j = k < sink ? k : k - sink + first;
    const long long page = kv_page_row(a.c, table, j / a.c.page_size, kvh);
    if (page < 0) {
      atomicOr(a.err, kErrKvStep);
      return -1;
    }
    return static_cast<int>(page) + j % a.c.page_size;
  };
  int next = row_of(32ll * part);
  for (long long k0 = 32ll * part; k0 < keys; k0 += 32ll * parts) {
    const int row = next;
    next = row_of(k0 + 32ll * parts);
    const uint32_t there = __ballot_sync(0xffffffffu, row >= 0);
    if (there == 0u) continue;
    seen = true;
    const int other = __shfl_sync(0xffffffffu, row, __ffs(there) - 1), from = row >= 0 ? row : other;
    int rows[8];
    KvEight<T, BITS, D> raw[FLY][N];
    float d = 0.0f, v[8];
#pragma unroll
    for (int e0 = 0; e0 < 8; e0 += FLY) {
#pragma unroll
      for (int e = 0; e < FLY; ++e) {
        rows[e0 + e] = __shfl_sync(0xffffffffu, from, g8 + e0 + e);
#pragma unroll
        for (int i = 0; i < N; ++i) raw[e][i].load(a.c.k, a.c.k_scale, rows[e0 + e], 64 * i + 8 * c);
      }
#pragma unroll
      for (int e = 0; e < FLY; ++e) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          raw[e][i].values(true, v);
#pragma unroll
          for (int k = 0; k < 8; ++k) sum = fmaf(x[i][k], v[k], sum);
          if (e0 + FLY == 8) raw[e][i].load(a.c.v, a.c.v_scale, rows[e], 64 * i + 8 * c);  // in flight under the softmax
        }
#pragma unroll
        for (int w = 1; w < 8; w <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
        if (c == e0 + e) d = sum;
      }
    }
    const float mn = fmaxf(m, kv_warp_max(row >= 0 ? d : -INFINITY));
    const float up = mn == -INFINITY ? 1.0f : __expf(m - mn);  // -inf - -inf would be NaN
    const float p = row < 0 ? 0.0f : d != d ? d : mn == -INFINITY ? 0.0f : __expf(d - mn);  // an undefined score stays
    l = l * up + p;
    m = mn;
    if (__any_sync(0xffffffffu, l != l)) {
      l = NAN;
      return;
    }
#pragma unroll
    for (int e0 = 0; e0 < 8; e0 += FLY)
#pragma unroll
      for (int e = 0; e < FLY; ++e) {
        const float pe = __shfl_sync(0xffffffffu, p, g8 + e0 + e);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          raw[e][i].values((there >> (g8 + e0 + e)) & 1u, v);
          if (e0 + FLY < 8) raw[e][i].load(a.c.v, a.c.v_scale, rows[FLY + e], 64 * i + 8 * c);
#pragma unroll
          for (int k = 0; k < 8; ++k) o[i][k] = e0 + e == 0 ? fmaf(o[i][k], up, pe * v[k]) : fmaf(pe, v[k], o[i][k]);
        }
      }
  }
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) l += __shfl_xor_sync(0xffffffffu, l, w);
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int k = 0; k < 8; ++k)
#pragma unroll
      for (int w = 8; w < 32; w <<= 1) o[i][k] += __shfl_xor_sync(0xffffffffu, o[i][k], w);
}

// What a row's sum divides by.
__device__ __forceinline__ float kv_inverse(float l, bool seen) { return l != 0.0f ? 1.0f / l : seen ? NAN : 0.0f; }

// A row by one warp. (The tiles call it in one place, at their end: what it needs in registers cost them 2 to 6 % where it
// was called in their middle.)
template <typename T, int BITS, int D>
__device__ __noinline__ void kv_attend_row(const KvAttnArgs& a, int s, int t, int head, const T* q, T* out) {
  const int lane = threadIdx.x & 31;
  float m, l, o[D / 64][8];
  bool seen;
  kv_attend_keys<T, BITS, D>(a, s, t, head, q, 0, 1, m, l, o, seen);
  const float inv = kv_inverse(l, seen);
  if (lane < 8)
#pragma unroll
    for (int i = 0; i < D / 64; ++i)
#pragma unroll
      for (int k = 0; k < 8; ++k) out[64 * i + 8 * lane + k] = kv_round<T>(o[i][k] * inv);
}

// A row by a CTA of four warps, which share its keys; `so` [4][D] and `sml` [8] in shared memory, free on entry and on exit.
template <typename T, int BITS, int D>
__device__ __noinline__ void kv_attend_row_cta(const KvAttnArgs& a, int s, int t, int head, const T* q, T* out, float* so,
                                               float* sml) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float m, l, o[D / 64][8];
  bool seen;
  kv_attend_keys<T, BITS, D>(a, s, t, head, q, warp, 4, m, l, o, seen);
  if (lane < 8)
#pragma unroll
    for (int i = 0; i < D / 64; ++i)
#pragma unroll
      for (int k = 0; k < 8; ++k) so[warp * D + 64 * i + 8 * lane + k] = o[i][k];
  if (lane == 0) sml[warp] = m, sml[4 + warp] = l;
  seen = __syncthreads_or(seen) != 0;
  if (warp == 0) {
    const float mm = fmaxf(fmaxf(sml[0], sml[1]), fmaxf(sml[2], sml[3]));
    float sum = 0.0f, y[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) y[i] = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float c = sml[w] == mm ? 1.0f : __expf(sml[w] - mm);  // an undefined sum stays, whatever it is weighed by
      sum = fmaf(sml[4 + w], c, sum);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) y[i] = fmaf(so[w * D + lane + 32 * i], c, y[i]);
    }
    const float inv = kv_inverse(sum, seen);
#pragma unroll
    for (int i = 0; i < D / 32; ++i) out[lane + 32 * i] = kv_round<T>(y[i] * inv);
  }
  __syncthreads();
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
