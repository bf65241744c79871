// Appending to the paged key/value cache, with the position rotation on the way, and reading cached tokens back.
//
// Both move each byte once and compute a few operations on it: HBM bounds them at the largest sizes, the chain
// start → length → page table → store at the smallest. One block per token (its place in the batch is found
// once), one thread per 16 dims of a head: 8 in each half, so a thread holds whole rotation pairs, reads and
// writes 16-byte vectors, and 4 neighbouring threads hold one 32-dim group of a 4-bit row in each half.
#include "kernels.cuh"
#include "kvcache.cuh"

namespace jc {

namespace {

// The sequence of packed row `row`: the last one whose rows start at or before it (empty sequences start there
// too, and are skipped by taking the last). A warp takes 32 bounds at a time, so the loads of a batch do not
// wait for one another.
__device__ __forceinline__ int kv_seq_of(const KvStep& st, int row) {
  if (!st.start) return row;
  const int lane = threadIdx.x & 31;
  int below = 0;
  for (int s0 = 0; s0 < st.sequences; s0 += 32) {
    const int s = s0 + lane;
    below += __popc(__ballot_sync(0xffffffffu, s < st.sequences && __ldg(st.start + s) <= row));
  }
  return below - 1;
}

template <typename T, bool VEC>
__device__ __forceinline__ void load8(const KvRows& r, long long token, int head, int d, float (&x)[8]) {
  const T* p = static_cast<const T*>(r.p) + token * r.ld + head * r.hs + d;
  if constexpr (VEC) {
    const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = kv_unpack<T>(w[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = kv_float(p[i]);
  }
}

template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  return make_uint4(kv_pack<T>(x[0], x[1]), kv_pack<T>(x[2], x[3]), kv_pack<T>(x[4], x[5]), kv_pack<T>(x[6], x[7]));
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(const KvRows& r, long long token, int head, int d, const float (&x)[8]) {
  T* p = static_cast<T*>(r.p) + token * r.ld + head * r.hs + d;
  if constexpr (VEC) {
    *reinterpret_cast<uint4*>(p) = pack8<T>(x);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = kv_round<T>(x[i]);
  }
}

// The larger (smaller) of two values, NaN if either is one: a group with a NaN has no 4-bit form and reads as NaN.
__device__ __forceinline__ float max_nan(float a, float b) { return a != a || a > b ? a : b; }
__device__ __forceinline__ float min_nan(float a, float b) { return a != a || a < b ? a : b; }

// 8 of a group's 32 values, the rest in the 3 lanes beside this one: their codes, and the group's (scale, min).
// scale = fp16((max − min) / 15), min = fp16(min); a code is the nearest of the 16 steps of these rounded two,
// in FP32 with one rounding an operation, so that a value's code does not depend on where it is computed.
// Values beyond ±65504 (and infinities) saturate first, as 16-bit stores do; where the rounded scale would then take
// the top code past FP16's range, a smaller one is used: 15 · scale ≤ max − min − 32, and min is off by at most 16.
__device__ __forceinline__ uint32_t quantise8(float (&x)[8], __half2& sm) {
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = x[i] > 65504.0f ? 65504.0f : x[i] < -65504.0f ? -65504.0f : x[i];
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo = min_nan(x[i], lo);
    hi = max_nan(x[i], hi);
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    lo = min_nan(__shfl_xor_sync(0xffffffffu, lo, o), lo);
    hi = max_nan(__shfl_xor_sync(0xffffffffu, hi, o), hi);
  }
  const float range = __fsub_rn(hi, lo);
  const __half low = __float2half_rn(lo);
  __half scale = __float2half_rn(__fdiv_rn(range, 15.0f));
  if (fmaf(15.0f, __half2float(scale), __half2float(low)) >= 65520.0f)
    scale = __float2half_rd(__fdiv_rd(__fsub_rd(range, 32.0f), 15.0f));
  sm = __halves2half2(scale, low);
  const float s = __half2float(scale), m = __half2float(low);
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float c = s > 0.0f ? rintf(__fdiv_rn(__fsub_rn(x[i], m), s)) : 0.0f;
    w |= static_cast<uint32_t>(fminf(fmaxf(c, 0.0f), 15.0f)) << (4 * i);
  }
  return w;
}

template <typename T, int BITS, int D, bool VEC>
__global__ void __launch_bounds__(256) kv_append_kernel(const __grid_constant__ KvAppendArgs a) {
  constexpr int TPH = D / 16;  // threads per head
  const int row = blockIdx.x;
  const int s = kv_seq_of(a.st, row);
  if (s < 0 || s >= a.st.sequences) {
    if (threadIdx.x == 0) atomicOr(a.err, kErrKvStep);
    return;
  }
  const KvSeq q = kv_seq(a.st, a.c.page_size, s, a.err);
  const int i = row - q.row0;
  if (i < 0 || i >= q.n) return;
  const int t = q.length - q.n + i;  // below 0: more new tokens than the length has, not stored
  const int pos = a.positions ? __ldg(a.positions + row) : t;
  const bool turn = a.rope != nullptr;
  if (turn && t >= 0 && (pos < 0 || pos >= a.rope_rows)) {
    if (threadIdx.x == 0) atomicOr(a.err, kErrKvStep);
    return;
  }
  const int hq = a.q.p ? a.heads : 0, hk = a.c.kv_heads;
  long long page = -1;  // the page's first row for head 0
  if (t >= 0) {
    page = kv_page_row(a.c, a.st.table + s * a.st.ld_table, t / a.c.page_size, 0);
    if (page < 0 && threadIdx.x == 0) atomicOr(a.err, kErrKvStep);
  }
  // a whole number of warps' worth of work each round: the 4-bit groups' shuffles need every lane
  const int work = (hq + 2 * hk) * TPH;
  for (int w0 = blockIdx.y * blockDim.x + threadIdx.x; w0 < ((work + 31) & ~31); w0 += gridDim.y * blockDim.x) {
    const bool on = w0 < work;
    const int w = on ? w0 : work - 1;
    const int slot = w / TPH, e = 8 * (w % TPH);
    const int part = slot < hq ? 0 : slot < hq + hk ? 1 : 2;  // q, k, v
    const int head = part == 0 ? slot : part == 1 ? slot - hq : slot - hq - hk;
    float x[8], y[8];
    const KvRows& src = part == 0 ? a.q : part == 1 ? a.k : a.v;
    load8<T, VEC>(src, row, head, e, x);
    load8<T, VEC>(src, row, head, D / 2 + e, y);
    if (part < 2 && turn && t >= 0 && e < a.pairs) {
      const float* tab = a.rope + static_cast<long long>(pos) * D + e;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (e + j < a.pairs) {  // each product and sum rounded once: the same value in every copy of the token
          const float c = __ldg(tab + j), sn = __ldg(tab + D / 2 + j);
          const float u = __fsub_rn(__fmul_rn(x[j], c), __fmul_rn(y[j], sn));
          y[j] = __fadd_rn(__fmul_rn(y[j], c), __fmul_rn(x[j], sn));
          x[j] = u;
        }
    }
    if (part == 0) {
      if (on) {
        store8<T, VEC>(a.q_out, row, head, e, x);
        store8<T, VEC>(a.q_out, row, head, D / 2 + e, y);
      }
      if (BITS == 16) continue;
    }
    void* pool = part == 1 ? a.c.k : a.c.v;
    const long long r = page + static_cast<long long>(head) * a.c.page_size + (t >= 0 ? t % a.c.page_size : 0);
    const bool put = on && part > 0 && page >= 0;
    if constexpr (BITS == 16) {
      if (put) {
        T* p = static_cast<T*>(pool) + r * D;
        *reinterpret_cast<uint4*>(p + e) = pack8<T>(x);
        *reinterpret_cast<uint4*>(p + D / 2 + e) = pack8<T>(y);
      }
    } else {
      __half2 sx, sy;
      const uint32_t cx = quantise8(x, sx), cy = quantise8(y, sy);
      if (put) {
        uint32_t* p = static_cast<uint32_t*>(pool) + r * (D / 8) + e / 8;
        p[0] = cx;
        p[D / 16] = cy;
        if ((e & 31) == 0) {
          __half2* sc = static_cast<__half2*>(part == 1 ? a.c.k_scale : a.c.v_scale) + r * (D / kKvGroup) + e / kKvGroup;
          sc[0] = sx;
          sc[D / 2 / kKvGroup] = sy;
        }
      }
    }
  }
}

// Cached tokens as packed rows of 16-bit values (a 4-bit cache: FP16, the values its codes stand for).
template <typename T, int BITS, int D, bool VEC>
__global__ void __launch_bounds__(256) kv_read_kernel(const __grid_constant__ KvReadArgs a) {
  constexpr int TPH = D / 8;
  const int row = blockIdx.x;
  const int s = kv_seq_of(a.st, row);
  if (s < 0 || s >= a.st.sequences) {
    if (threadIdx.x == 0) atomicOr(a.err, kErrKvStep);
    return;
  }
  const KvSeq q = kv_seq(a.st, a.c.page_size, s, a.err);
  const int i = row - q.row0;
  if (i < 0 || i >= q.n) return;
  const int t = q.length - q.n + i;
  long long page = -1;
  if (t >= 0) {
    page = kv_page_row(a.c, a.st.table + s * a.st.ld_table, t / a.c.page_size, 0);
    if (page < 0 && threadIdx.x == 0) atomicOr(a.err, kErrKvStep);
  }
  const int hk = a.c.kv_heads;
  for (int w = blockIdx.y * blockDim.x + threadIdx.x; w < 2 * hk * TPH; w += gridDim.y * blockDim.x) {
    const int slot = w / TPH, d = 8 * (w % TPH);
    const bool key = slot < hk;
    const int head = key ? slot : slot - hk;
    const KvRows& dst = key ? a.k : a.v;
    T* out = static_cast<T*>(dst.p) + row * dst.ld + head * dst.hs + d;
    uint4 u = make_uint4(0u, 0u, 0u, 0u);  // a token before the sequence's first, or of no page: zeros
    if (page >= 0) {
      const long long r = page + static_cast<long long>(head) * a.c.page_size + t % a.c.page_size;
      const void* pool = key ? a.c.k : a.c.v;
      if constexpr (BITS == 16) {
        u = *reinterpret_cast<const uint4*>(static_cast<const T*>(pool) + r * D + d);
      } else {
        const uint32_t c = static_cast<const uint32_t*>(pool)[r * (D / 8) + d / 8];
        const __half2 sm = static_cast<const __half2*>(key ? a.c.k_scale : a.c.v_scale)[r * (D / kKvGroup) + d / kKvGroup];
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const __half2 h = __halves2half2(kv_code_value((c >> (8 * j)) & 15u, sm), kv_code_value((c >> (8 * j + 4)) & 15u, sm));
          o[j] = *reinterpret_cast<const uint32_t*>(&h);
        }
        u = make_uint4(o[0], o[1], o[2], o[3]);
      }
    }
    if constexpr (VEC) {
      *reinterpret_cast<uint4*>(out) = u;
    } else {
      const uint32_t o[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint16_t h = static_cast<uint16_t>(o[j >> 1] >> (16 * (j & 1)));
        out[j] = *reinterpret_cast<const T*>(&h);
      }
    }
  }
}

bool vec_rows(const KvRows& r) {
  return r.p == nullptr || ((reinterpret_cast<uintptr_t>(r.p) & 15) == 0 && r.ld % 8 == 0 && r.hs % 8 == 0);
}

// Blocks over one token's work: one, until a token alone has more work than four rounds of its 256 threads.
unsigned splits_of(int work) { return static_cast<unsigned>((work + 1023) / 1024); }

template <typename T, int BITS, int D>
void append(const KvAppendArgs& a, cudaStream_t s) {
  const int work = ((a.q.p ? a.heads : 0) + 2 * a.c.kv_heads) * (D / 16);
  const int threads = work >= 256 ? 256 : (work + 31) & ~31;
  const dim3 grid(static_cast<unsigned>(a.st.tokens), splits_of(work));
  if (vec_rows(a.q) && vec_rows(a.k) && vec_rows(a.v) && vec_rows(a.q_out))
    kv_append_kernel<T, BITS, D, true><<<grid, threads, 0, s>>>(a);
  else
    kv_append_kernel<T, BITS, D, false><<<grid, threads, 0, s>>>(a);
}

template <typename T, int BITS, int D>
void read(const KvReadArgs& a, cudaStream_t s) {
  const int work = 2 * a.c.kv_heads * (D / 8);
  const int threads = work >= 256 ? 256 : (work + 31) & ~31;
  const dim3 grid(static_cast<unsigned>(a.st.tokens), splits_of(work));
  if (vec_rows(a.k) && vec_rows(a.v))
    kv_read_kernel<T, BITS, D, true><<<grid, threads, 0, s>>>(a);
  else
    kv_read_kernel<T, BITS, D, false><<<grid, threads, 0, s>>>(a);
}

}  // namespace

cudaError_t launch_kv_append(const KvAppendArgs& a, cudaStream_t s) {
  if (a.st.tokens == 0) return cudaSuccess;
  if (a.c.bits == 16) {
    if (a.c.dim == 64)
      a.c.f16 ? append<__half, 16, 64>(a, s) : append<__nv_bfloat16, 16, 64>(a, s);
    else
      a.c.f16 ? append<__half, 16, 128>(a, s) : append<__nv_bfloat16, 16, 128>(a, s);
  } else {
    if (a.c.dim == 64)
      a.c.f16 ? append<__half, 4, 64>(a, s) : append<__nv_bfloat16, 4, 64>(a, s);
    else
      a.c.f16 ? append<__half, 4, 128>(a, s) : append<__nv_bfloat16, 4, 128>(a, s);
  }
  return cudaGetLastError();
}

cudaError_t launch_kv_read(const KvReadArgs& a, cudaStream_t s) {
  if (a.st.tokens == 0) return cudaSuccess;
  // 16-bit values are copied as they are, whichever type they have; a 4-bit cache's are FP16
  if (a.c.bits == 16)
    a.c.dim == 64 ? read<__half, 16, 64>(a, s) : read<__half, 16, 128>(a, s);
  else
    a.c.dim == 64 ? read<__half, 4, 64>(a, s) : read<__half, 4, 128>(a, s);
  return cudaGetLastError();
}

}  // namespace jc
