// Appending to the paged key/value cache, with the position rotation on the way, and reading cached tokens back.
//
// Both move each byte once and compute a few operations on it: HBM bounds them at the largest sizes, the chain
// start → length → page table → data at the smallest. A block takes a few tokens where there are many: its warps find
// their places in the batch side by side, then all threads move the data (one token a block left every block waiting
// for that chain: 7 prompts 59 us, now 50; 37 chunks into 4 bits and back 170 us, now 80). A thread takes 16 dims
// of a head: 8 in each half, so it holds whole rotation pairs, reads and writes 16-byte vectors, and 4 neighbouring
// threads hold one 32-dim group of a 4-bit row in each half.
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
    const uint4 u = kv_load16(p);
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

// 8 of a group's 32 values, the rest in the 3 lanes beside this one: their codes, and the group's (scale, min).
// scale = fp16((max − min) / 15), min = fp16(min); a code is the nearest of the 16 steps of these rounded two,
// in FP32. A group with a NaN has no 4-bit form: its scale and minimum are NaN, and it reads as NaN.
// Values beyond ±65504 (and infinities) saturate first, as 16-bit stores do; where the rounded scale would then take
// the top code past FP16's range, a smaller one is used: 15 · scale ≤ max − min − 32, and min is off by at most 16.
__device__ __forceinline__ uint32_t quantise8(float (&x)[8], __half2& sm) {
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = max_nan(min_nan(x[i], 65504.0f), -65504.0f);
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
  // (x − min) / scale to the nearest integer, ties to even. The quotient has to be the rounded one (16-bit inputs give
  // exact ties, of which a product with the reciprocal alone breaks some: 0.04 % of the codes), which fused arithmetic
  // gives from the rounded reciprocal r and q = d r as q + r (d − s q) (Markstein, 1990); a division each took 24 of 72 us.
  // Then clamped, and rounded by adding 2^23, which leaves the integer in the last bits. A scale of 0 gives code 0.
  const float s = __half2float(scale), m = __half2float(low), r = s > 0.0f ? __frcp_rn(s) : 0.0f;
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float d = __fsub_rn(x[i], m), q0 = __fmul_rn(d, r), q = fmaf(fmaf(-q0, s, d), r, q0);
    w |= (__float_as_uint(fminf(fmaxf(q, 0.0f), 15.0f) + 8388608.0f) & 15u) << (4 * i);
  }
  return w;
}

// Where a token's data goes: pool row of its slot for head 0 (−1: nowhere), its index and its row of the rotation table.
struct Place {
  long long row;
  int t, pos;
  bool on;  // false: nothing of the token is read or written
};
constexpr int kTokens = 8;  // most tokens of a block

// The places of a block's tokens row0 .. row0 + n − 1, a warp each.
__device__ __forceinline__ void find_places(const KvCache& c, const KvStep& st, const int* positions, int rope_rows, int row0,
                                            int n, Place* out, uint32_t* err) {
  for (int k = threadIdx.x >> 5; k < n; k += blockDim.x >> 5) {
    const int row = row0 + k, s = kv_seq_of(st, row);
    Place p{-1, 0, 0, false};
    bool bad = s < 0 || s >= st.sequences;
    if (!bad) {
      const KvSeq q = kv_seq(st, c.page_size, s, err);
      const int i = row - q.row0;
      if (i >= 0 && i < q.n) {
        p.t = q.length - q.n + i;  // below 0: more new tokens than the length has, not stored
        p.pos = positions ? __ldg(positions + row) : p.t;
        p.on = true;
        if (p.t >= 0) {
          p.row = kv_page_row(c, st.table + s * st.ld_table, p.t / c.page_size, 0);
          bad = p.row < 0;
          if (p.row >= 0) p.row += p.t % c.page_size;
          if (rope_rows > 0 && (p.pos < 0 || p.pos >= rope_rows)) {
            bad = true;
            p.on = false;
          }
        }
      }
    }
    if ((threadIdx.x & 31) == 0) {
      if (bad) atomicOr(err, kErrKvStep);
      out[k] = p;
    }
  }
  __syncthreads();
}

template <typename T, int BITS, int D, bool VEC>
__global__ void __launch_bounds__(256) kv_append_kernel(const __grid_constant__ KvAppendArgs a, int per_block) {
  constexpr int TPH = D / 16;  // threads per head
  __shared__ Place places[kTokens];
  const int row0 = blockIdx.x * per_block, n = min(per_block, a.st.tokens - row0);
  find_places(a.c, a.st, a.positions, a.rope ? a.rope_rows : 0, row0, n, places, a.err);
  const int hq = a.q.p ? a.heads : 0, hk = a.c.kv_heads;
  // a whole number of warps' worth of work each round: the 4-bit groups' shuffles need every lane
  const int work = (hq + 2 * hk) * TPH;
  for (int w0 = blockIdx.y * blockDim.x + threadIdx.x; w0 < ((work + 31) & ~31); w0 += gridDim.y * blockDim.x) {
    const int w = w0 < work ? w0 : work - 1;
    const int slot = w / TPH, e = 8 * (w % TPH);
    const int part = slot < hq ? 0 : slot < hq + hk ? 1 : 2;  // q, k, v
    const int head = part == 0 ? slot : part == 1 ? slot - hq : slot - hq - hk;
    const KvRows src = part == 0 ? a.q : part == 1 ? a.k : a.v;
    const bool quantise = BITS == 4 && __any_sync(0xffffffffu, part > 0);
#pragma unroll 2
    for (int k = 0; k < n; ++k) {
      const Place p = places[k];
      if (!p.on) continue;
      const int row = row0 + k;
      float x[8], y[8];
      load8<T, VEC>(src, row, head, e, x);
      load8<T, VEC>(src, row, head, D / 2 + e, y);
      if (part < 2 && p.t >= 0 && e < a.pairs) {
        const float* tab = a.rope + static_cast<long long>(p.pos) * D + e;
        float c[8], sn[8];
        if (((reinterpret_cast<uintptr_t>(a.rope)) & 15) == 0) {
#pragma unroll
          for (int j = 0; j < 8; j += 4) {
            const float4 cv = __ldg(reinterpret_cast<const float4*>(tab + j)), sv = __ldg(reinterpret_cast<const float4*>(tab + D / 2 + j));
            c[j] = cv.x, c[j + 1] = cv.y, c[j + 2] = cv.z, c[j + 3] = cv.w;
            sn[j] = sv.x, sn[j + 1] = sv.y, sn[j + 2] = sv.z, sn[j + 3] = sv.w;
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) c[j] = __ldg(tab + j), sn[j] = __ldg(tab + D / 2 + j);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (e + j < a.pairs) {  // each product and sum rounded once: the same value in every copy of the token
            const float u = __fsub_rn(__fmul_rn(x[j], c[j]), __fmul_rn(y[j], sn[j]));
            y[j] = __fadd_rn(__fmul_rn(y[j], c[j]), __fmul_rn(x[j], sn[j]));
            x[j] = u;
          }
      }
      if (part == 0 && w0 < work) {
        store8<T, VEC>(a.q_out, row, head, e, x);
        store8<T, VEC>(a.q_out, row, head, D / 2 + e, y);
      }
      void* pool = part == 1 ? a.c.k : a.c.v;
      const long long r = p.row + static_cast<long long>(head) * a.c.page_size;
      const bool put = w0 < work && part > 0 && p.row >= 0;
      if constexpr (BITS == 16) {
        if (put) {
          T* d = static_cast<T*>(pool) + r * D;
          *reinterpret_cast<uint4*>(d + e) = pack8<T>(x);
          *reinterpret_cast<uint4*>(d + D / 2 + e) = pack8<T>(y);
        }
      } else if (quantise) {
        __half2 sx, sy;
        const uint32_t cx = quantise8(x, sx), cy = quantise8(y, sy);
        if (put) {
          uint32_t* d = static_cast<uint32_t*>(pool) + r * (D / 8) + e / 8;
          d[0] = cx;
          d[D / 16] = cy;
          if ((e & 31) == 0) {
            __half2* sc = static_cast<__half2*>(part == 1 ? a.c.k_scale : a.c.v_scale) + r * (D / kKvGroup) + e / kKvGroup;
            sc[0] = sx;
            sc[D / 2 / kKvGroup] = sy;
          }
        }
      }
    }
  }
}

// Cached tokens as packed rows of 16-bit values (a 4-bit cache: FP16, the values its codes stand for). A thread takes
// 8 dims.
template <typename T, int BITS, int D, bool VEC>
__global__ void __launch_bounds__(256) kv_read_kernel(const __grid_constant__ KvReadArgs a, int per_block) {
  constexpr int TPH = D / 8;
  __shared__ Place places[kTokens];
  const int row0 = blockIdx.x * per_block, n = min(per_block, a.st.tokens - row0);
  find_places(a.c, a.st, nullptr, 0, row0, n, places, a.err);
  const int hk = a.c.kv_heads;
  for (int w = blockIdx.y * blockDim.x + threadIdx.x; w < 2 * hk * TPH; w += gridDim.y * blockDim.x) {
    const int slot = w / TPH, d = 8 * (w % TPH);
    const bool key = slot < hk;
    const int head = key ? slot : slot - hk;
    const KvRows dst = key ? a.k : a.v;
    const void* pool = key ? a.c.k : a.c.v;
    const void* scale = key ? a.c.k_scale : a.c.v_scale;
#pragma unroll 4
    for (int k = 0; k < n; ++k) {
      const Place p = places[k];
      if (!p.on) continue;
      uint4 u = make_uint4(0u, 0u, 0u, 0u);  // a token before the sequence's first, or of no page: zeros
      if (p.row >= 0) {
        const long long r = p.row + static_cast<long long>(head) * a.c.page_size;
        if constexpr (BITS == 16) {
          u = *reinterpret_cast<const uint4*>(static_cast<const T*>(pool) + r * D + d);
        } else {
          const uint32_t c = static_cast<const uint32_t*>(pool)[r * (D / 8) + d / 8];
          const __half2 sm = static_cast<const __half2*>(scale)[r * (D / kKvGroup) + d / kKvGroup];
          uint32_t o[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const __half2 h = __halves2half2(kv_code_value((c >> (8 * j)) & 15u, sm), kv_code_value((c >> (8 * j + 4)) & 15u, sm));
            o[j] = *reinterpret_cast<const uint32_t*>(&h);
          }
          u = make_uint4(o[0], o[1], o[2], o[3]);
        }
      }
      T* out = static_cast<T*>(dst.p) + static_cast<long long>(row0 + k) * dst.ld + head * dst.hs + d;
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
}

bool vec_rows(const KvRows& r) {
  return r.p == nullptr || ((reinterpret_cast<uintptr_t>(r.p) & 15) == 0 && r.ld % 8 == 0 && r.hs % 8 == 0);
}

// Threads for one token's work (up to 256, in rounds of alike size: blocks of 384 leave an SM a third of its threads, 59
// against 48 us at 8016 tokens of 48 heads of 128), blocks over it where a token alone has more than
// four rounds, and tokens a block: one while that leaves an SM fewer than eight blocks, else up to kTokens.
struct Launch {
  dim3 grid;
  int threads, per_block;
  Launch(int tokens, int work) {
    const int rounds = (work + 255) / 256;
    threads = ((work + rounds - 1) / rounds + 31) & ~31;
    per_block = tokens / (148 * 8);
    per_block = per_block < 1 ? 1 : per_block > kTokens ? kTokens : per_block;
    grid = dim3(static_cast<unsigned>((tokens + per_block - 1) / per_block), static_cast<unsigned>((rounds + 3) / 4));
  }
};

template <typename T, int BITS, int D>
void append(const KvAppendArgs& a, cudaStream_t s) {
  const Launch l(a.st.tokens, ((a.q.p ? a.heads : 0) + 2 * a.c.kv_heads) * (D / 16));
  if (vec_rows(a.q) && vec_rows(a.k) && vec_rows(a.v) && vec_rows(a.q_out))
    kv_append_kernel<T, BITS, D, true><<<l.grid, l.threads, 0, s>>>(a, l.per_block);
  else
    kv_append_kernel<T, BITS, D, false><<<l.grid, l.threads, 0, s>>>(a, l.per_block);
}

template <typename T, int BITS, int D>
void read(const KvReadArgs& a, cudaStream_t s) {
  const Launch l(a.st.tokens, 2 * a.c.kv_heads * (D / 8));
  if (vec_rows(a.k) && vec_rows(a.v))
    kv_read_kernel<T, BITS, D, true><<<l.grid, l.threads, 0, s>>>(a, l.per_block);
  else
    kv_read_kernel<T, BITS, D, false><<<l.grid, l.threads, 0, s>>>(a, l.per_block);
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
