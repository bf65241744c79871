// Cache attention of many query rows a key (prompts, prompt chunks) on the 5th-generation tensor cores.
//
// A CTA takes 256 packed rows (token · group + head of the group) of one sequence and kv head as two 128-row tiles,
// and walks the keys that they see 128 at a time (8 of the 16-key blocks: sinks first, then the band):
//
//   S_i = Q_i · Kᵀ    tcgen05.mma kind::f16, Q and K K-major in shared memory, S in TMEM (128 × 128 FP32)
//   O_i += P_i · V    P from TMEM (over S's columns, 16 bits), V MN-major in shared memory, O in TMEM
//
// Four softmax warps a tile (a thread a row: running maximum and sum need no shuffle), one TMA producer
// warp (a lane a 16-key block: pages may lie anywhere) and one MMA issuer. The two tiles alternate: while one tile's
// products run, the other's exponentials do, and both read each K and V tile once from shared memory, which halves
// the bytes from L2. What bounds it: at 64 dims the exponentials (128 · 128 a tile at 16 a clock and SM: 1024 clocks,
// against 512 for the products), at 128 dims both alike.
//
// The running maximum moves only when a score passes it by 2^kLazy (as in the split kernel), so O is rescaled in
// TMEM in few steps. S(j + 1) is issued after P·V(j) of its tile by the same thread, so when a softmax warp sees
// S(j + 1) ready, O holds every P·V up to j and no product is touching it.
#include <algorithm>

#include "gemm.h"
#include "kv_attention.cuh"

namespace jc {

namespace {

constexpr int kRows = 128;   // rows of a tile (TMEM lanes)
constexpr int kKeys = 128;   // keys of a step
constexpr int kTcThreads = 384;
// Registers a thread: 168 at launch (three warps on each SM quarter); the third warpgroup gives some of its to the
// softmax warpgroups, which hold a row of 128 scores. 2 · 224 + 56 = 3 · 168.
constexpr int kTcRegs = 168, kTcRegsSoftmax = 224, kTcRegsIssue = 56;
constexpr float kTcLog2e = 1.4426950408889634f;
constexpr float kTcLazy = 8.0f;

template <int D>
struct TcCfg {
  static constexpr int STAGES = D == 64 ? 4 : 2;
  static constexpr int TILE = kKeys * D * 2;    // bytes of a K, V or Q tile
  static constexpr int Q_OFF = 0;
  static constexpr int K_OFF = 2 * TILE;
  static constexpr int V_OFF = K_OFF + STAGES * TILE;
  static constexpr int BAR_OFF = V_OFF + STAGES * TILE;
  static constexpr int SMEM = BAR_OFF + 512 + 1024;
  static constexpr int ATOM = kKeys * 128;      // bytes of a tile's 64-dim column block (128-byte swizzled rows)
};

struct TcArgs {
  int shift;         // 2^shift keys a block: the largest power of two, up to 64, that a page holds a whole number of
  int supers;        // 256-row tiles of the longest sequence
  int pool_rows;     // rows of the pools: a coordinate outside them
  int vec_q, vec_o;  // 16-byte vectors
  KvDiv page;        // blocks of a page
};

__device__ __forceinline__ uint32_t sw128(int r, int c) {
  return static_cast<uint32_t>(r * 128 + ((((c >> 3) ^ r) & 7) << 4) + ((c & 7) << 1));
}

template <typename T>
__device__ __forceinline__ uint32_t pack_p(float a, float b) {
  if constexpr (std::is_same<T, __half>::value) {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  } else {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
}

// Two FP32 values in one 64-bit register: one instruction adds or multiplies both.
__device__ __forceinline__ uint64_t pack_f32x2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack_f32x2(uint64_t x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
  return r;
}
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Bits lo .. hi − 1 of 16.
__device__ __forceinline__ uint32_t bits16(int lo, int hi) {
  lo = min(max(lo, 0), 16), hi = min(max(hi, 0), 16);
  return hi <= lo ? 0u : (1u << hi) - (1u << lo);
}

// The keys of block b that index t sees, as 16 bits.
__device__ __forceinline__ uint32_t block_bits(int key0, int t, int first, int sinks) {
  const uint32_t past = bits16(0, t + 1 - key0);
  return past & (bits16(first - key0, 16) | bits16(0, sinks - key0 > 16 ? 16 : sinks - key0));
}

// MN-major B descriptor of 16 keys of V: 8-key groups 1024 bytes apart (SBO), 64-dim column blocks an atom apart (LBO).
__device__ __forceinline__ uint64_t sdesc_v(uint32_t saddr, uint32_t atom_bytes) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(atom_bytes >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}

template <typename T, int D>
__global__ void __launch_bounds__(kTcThreads, 1) kv_attention_tc_kernel(const __grid_constant__ CUtensorMap tmK,
                                                                       const __grid_constant__ CUtensorMap tmV,
                                                                       const __grid_constant__ KvAttnArgs a,
                                                                       const __grid_constant__ TcArgs tc) {
  using C = TcCfg<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::BAR_OFF);
  uint64_t* k_full = bars;                    // [STAGES] TMA → MMA
  uint64_t* k_free = k_full + C::STAGES;      // [STAGES] MMA → TMA
  uint64_t* v_full = k_free + C::STAGES;
  uint64_t* v_free = v_full + C::STAGES;
  uint64_t* s_full = v_free + C::STAGES;      // [2] MMA → softmax: S of the tile ready
  uint64_t* p_full = s_full + 2;              // [2] softmax → MMA: P written (128 arrivals)
  uint64_t* o_full = p_full + 2;              // [2] MMA → softmax: every product of the tile done
  uint64_t* q_full = o_full + 2;              // [2] softmax → MMA: Q written (128 arrivals)
  uint64_t* v_raw = q_full + 2;               // [1] TMA → producer: a V tile with hidden rows to clear
  uint64_t* drain = v_raw + 1;                // [1] MMA: products issued before it gave up
  uint32_t* slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile uint32_t* abort_flag = slot + 1;
  uint32_t* bad_page = slot + 2;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int seq = blockIdx.y;
  // later rows see more keys: they start first
  const int super = tc.supers - 1 - static_cast<int>(blockIdx.x) / a.c.kv_heads;
  const int kvh = static_cast<int>(blockIdx.x) % a.c.kv_heads;
  const KvSeq sq = kv_seq(a.st, a.c.page_size, seq, a.err);
  const int group = a.heads / a.c.kv_heads;
  const int r0 = super * 2 * kRows;
  const int rows = min(sq.n * group - r0, 2 * kRows);
  if (rows <= 0) return;
  const int base_t = sq.length - sq.n;
  const int t0 = base_t + r0 / group, t1 = base_t + (r0 + rows - 1) / group;
  const KvBlocks kb = kv_blocks(a, t0, t1, tc.shift);
  const int per = kKeys >> tc.shift;  // blocks of a step
  const int steps = (kb.n + per - 1) >> (7 - tc.shift);
  const int tiles = rows > kRows ? 2 : 1;
  const int* table = a.st.table + seq * a.st.ld_table;

  if (tid == 0) {
    for (int i = 0; i < C::STAGES; ++i) {
      mbar_init(k_full + i, 1);
      mbar_init(k_free + i, 1);
      mbar_init(v_full + i, 1);
      mbar_init(v_free + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full + i, 1);
      mbar_init(p_full + i, kRows);
      mbar_init(o_full + i, 1);
      mbar_init(q_full + i, kRows);
    }
    mbar_init(v_raw, 1);
    mbar_init(drain, 1);
    *abort_flag = 0;
    *bad_page = 0;
    fence_mbar_init();
  }
  if (warp == 9) {
    tmem_alloc(slot, 512);
    tmem_relinquish();
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *slot;
  // every page that the tile reads lies in the pool, or the rows go the row-by-row way, which leaves such pages out
  for (int x = tid; x < kb.n; x += kTcThreads) {
    const int id = __ldg(table + tc.page.of(kb.at(x)));
    if (id < 0 || id >= a.c.pages) *bad_page = 1u;
  }
  __syncthreads();
  const bool good = *bad_page == 0u;

  if (good && warp >= 8) {
   asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kTcRegsIssue));
   if (warp == 8) {
    // ---- producer: lane = block (and 64-dim column block) of a step ----
    const int blk = lane & (per - 1), atom = lane >> (7 - tc.shift);
    const bool mine = atom < D / 64;
    const int size = 1 << tc.shift, first = kv_first(a, t0 < 0 ? 0 : t0);
    const uint32_t off = atom * C::ATOM + blk * (size * 128);
    bool ok = true;
    uint32_t raw_phase = 0;
    // the pool row of the lane's block in step j; past the last block: outside the pool, which loads zeros
    auto row_of = [&](int j) -> int {
      const int x = j * per + blk;
      if (!mine || x >= kb.n) return tc.pool_rows;
      const int b = kb.at(x);
      const unsigned pg = tc.page.of(b);
      return (__ldg(table + pg) * a.c.kv_heads + kvh) * a.c.page_size + ((b - static_cast<int>(pg * tc.page.d)) << tc.shift);
    };
    int row = row_of(0);
    for (int j = 0; j < steps && ok; ++j) {
      const int st = j % C::STAGES;
      const uint32_t ph = (j / C::STAGES) & 1;
      const int next = row_of(j + 1);  // in flight during this step's waits
      if (!mbar_wait(k_free + st, ph ^ 1) || *abort_flag) ok = false;
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (lane == 0) mbar_arrive_expect_tx(k_full + st, C::TILE);
      __syncwarp();
      if (mine) tma_load_2d(smem + C::K_OFF + st * C::TILE + off, &tmK, k_full + st, 64 * atom, row);
      if (!mbar_wait(v_free + st, ph ^ 1) || *abort_flag) ok = false;
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      // keys of the step that no row of the CTA sees: their values, whatever they are, become zeros
      const int x = j * per + blk, key0 = kb.at(x) << tc.shift;
      const bool part = mine && x < kb.n && (key0 + size - 1 > t1 || (key0 < first && key0 + size > a.sinks));
      const bool clear = __any_sync(0xffffffffu, part);
      uint8_t* vt = smem + C::V_OFF + st * C::TILE + off;
      uint64_t* bar = clear ? v_raw : v_full + st;
      if (lane == 0) mbar_arrive_expect_tx(bar, C::TILE);
      __syncwarp();
      if (mine) tma_load_2d(vt, &tmV, bar, 64 * atom, row);
      if (clear) {
        ok = mbar_wait(v_raw, raw_phase);
        raw_phase ^= 1;
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        for (uint32_t left = __ballot_sync(0xffffffffu, part); left; left &= left - 1) {
          const int from = __ffs(left) - 1;  // the whole warp clears that lane's block
          const int k0 = __shfl_sync(0xffffffffu, key0, from);
          uint8_t* p = smem + C::V_OFF + st * C::TILE + __shfl_sync(0xffffffffu, off, from);
          for (int w = lane; w < size * 8; w += 32) {
            const int key = k0 + (w >> 3);
            if (key > t1 || (key < first && key >= a.sinks)) *reinterpret_cast<uint4*>(p + 16 * w) = make_uint4(0u, 0u, 0u, 0u);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(v_full + st);
      }
      row = next;
    }
    if (!ok) {
      if (lane == 0) {
        *abort_flag = 1;
        atomicOr(a.err, kErrAttnWait);
      }
      // the copies in flight land before the CTA's shared memory can go
      __syncwarp();
      for (int i = 0; i < C::STAGES; ++i) {
        mbar_wait(k_full + i, 0, 1000000);
        mbar_wait(v_full + i, 0, 1000000);
      }
    }
   } else if (warp == 9) {
    // ---- MMA issuer ----
    if (lane == 0 && steps > 0) {
      constexpr uint32_t fmt = std::is_same<T, __half>::value ? 0u : 1u;
      constexpr uint32_t is = idesc_f32acc(fmt, kRows, kKeys);
      constexpr uint32_t io = idesc_f32acc(fmt, kRows, D) | (1u << 16);  // B (V) MN-major
      const uint32_t qa = smem_u32(smem + C::Q_OFF), ka = smem_u32(smem + C::K_OFF), va = smem_u32(smem + C::V_OFF);
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t ph) {
        if (ok && (!mbar_wait(bar, ph) || *abort_flag)) ok = false;
        return ok;
      };
      auto scores = [&](int i, int j) {  // S_i of step j
        const uint32_t q = qa + i * C::TILE, k = ka + (j % C::STAGES) * C::TILE;
#pragma unroll
        for (int d = 0; d < D / 16; ++d)
          umma_bf16(tmem + i * kKeys, sdesc_k_sw128(q + (d >> 2) * C::ATOM + 32 * (d & 3)),
                    sdesc_k_sw128(k + (d >> 2) * C::ATOM + 32 * (d & 3)), is, d > 0);
        umma_commit(s_full + i);
      };
      wait(k_full, 0);
      for (int i = 0; i < tiles && ok; ++i) {
        if (!wait(q_full + i, 0)) break;
        tc_fence_after();
        scores(i, 0);
      }
      if (ok) umma_commit(k_free);
      for (int j = 0; j < steps && ok; ++j) {
        const int jn = j + 1;
        if (jn < steps) wait(k_full + jn % C::STAGES, (jn / C::STAGES) & 1);
        wait(v_full + j % C::STAGES, (j / C::STAGES) & 1);
        for (int i = 0; i < tiles && ok; ++i) {
          if (!wait(p_full + i, j & 1)) break;
          tc_fence_after();
          const uint32_t v = va + (j % C::STAGES) * C::TILE;
#pragma unroll
          for (int k = 0; k < kKeys / 16; ++k)
            umma_f16_ts(tmem + 2 * kKeys + i * D, tmem + i * kKeys + 8 * k, sdesc_v(v + 2048 * k, C::ATOM), io,
                        j > 0 || k > 0);
          if (jn < steps)
            scores(i, jn);
          else
            umma_commit(o_full + i);
        }
        if (ok) {
          umma_commit(v_free + j % C::STAGES);
          if (jn < steps) umma_commit(k_free + jn % C::STAGES);
        }
      }
      if (!ok) {
        *abort_flag = 1;
        atomicOr(a.err, kErrAttnWait);
        umma_commit(drain);  // every product issued has completed once this flips
        mbar_wait(drain, 0, 1000000);
      }
    }
    __syncwarp();
   }
  } else if (good) {
    // ---- softmax: tile i, a thread a row ----
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kTcRegsSoftmax));
    const int i = warp >> 2, row = (warp & 3) * 32 + lane;
    if (i < tiles) {
      const int r = r0 + i * kRows + row;
      const bool mine = r < r0 + rows;
      const bool any = r0 + i * kRows + (warp & 3) * 32 < r0 + rows;  // the warp has a row
      const int rr = mine ? r : r0 + rows - 1;
      const int tok = rr / group, head = kvh * group + rr % group;
      const int t = base_t + tok, first = kv_first(a, t < 0 ? 0 : t);
      const long long grow = static_cast<long long>(sq.row0) + tok;
      const T* qp = static_cast<const T*>(a.q.p) + grow * a.q.ld + head * a.q.hs;
      uint8_t* qs = smem + C::Q_OFF + i * C::TILE;
#pragma unroll
      for (int c = 0; c < D / 8; ++c) {
        uint4 u = make_uint4(0u, 0u, 0u, 0u);
        if (mine) {
          if (tc.vec_q) {
            u = __ldg(reinterpret_cast<const uint4*>(qp) + c);
          } else {
            const uint16_t* h = reinterpret_cast<const uint16_t*>(qp) + 8 * c;
            u.x = h[0] | static_cast<uint32_t>(h[1]) << 16, u.y = h[2] | static_cast<uint32_t>(h[3]) << 16;
            u.z = h[4] | static_cast<uint32_t>(h[5]) << 16, u.w = h[6] | static_cast<uint32_t>(h[7]) << 16;
          }
        }
        *reinterpret_cast<uint4*>(qs + (c >> 3) * C::ATOM + sw128(row, 8 * (c & 7))) = u;
      }
      fence_proxy_async_smem();
      mbar_arrive(q_full + i);

      // the warp's tokens
      const int rw0 = r0 + i * kRows + (warp & 3) * 32, rw1 = min(rw0 + 31, r0 + rows - 1);
      const int tw0 = base_t + rw0 / group, tw1 = base_t + rw1 / group;
      const int fw0 = kv_first(a, tw0 < 0 ? 0 : tw0), fw1 = kv_first(a, tw1 < 0 ? 0 : tw1);
      const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
      const uint32_t s_col = lanes + i * kKeys, o_col = lanes + 2 * kKeys + i * D;
      const float sl2 = a.scale * kTcLog2e;
      float m = -INFINITY, l = 0.0f;
      bool ok = true;
      for (int j = 0; j < steps; ++j) {
        const bool got = mbar_wait(s_full + i, j & 1) && !*abort_flag;
        ok = __all_sync(0xffffffffu, got);
        if (!ok) break;
        tc_fence_after();
        if (any) {
          float s[4][32];
          uint32_t shut = 0u;  // 32-key chunks that no row of the warp sees
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(s_col + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(s[c]));
          tmem_ld_wait();
          // Hide what a row does not see. A step of the band that every row of the warp sees whole skips this.
          const int key0 = kb.at(j * per) << tc.shift;
          if (!(j * per >= kb.a && key0 + kKeys - 1 <= tw0 && key0 >= fw1)) {
            const int sub = tc.shift - 4;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const int ha = 8 * j + 2 * c, hc = ha + 1;  // the chunk's two 16-key halves
              const int ka = (kb.at(ha >> sub) << tc.shift) + ((ha & ((1 << sub) - 1)) << 4);
              const int kc = (kb.at(hc >> sub) << tc.shift) + ((hc & ((1 << sub) - 1)) << 4);
              if ((ka > tw1 || (ka + 15 < fw0 && ka >= a.sinks)) && (kc > tw1 || (kc + 15 < fw0 && kc >= a.sinks))) shut |= 1u << c;
              const uint32_t bits = block_bits(ka, t, first, a.sinks) | block_bits(kc, t, first, a.sinks) << 16;
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!((bits >> e) & 1u)) s[c][e] = -INFINITY;
            }
          }
          float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // four chains
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 32; e += 2) mx4[(e >> 1) & 3] = fmax3(mx4[(e >> 1) & 3], s[c][e], s[c][e + 1]);
          const float top = fmax3(mx4[0], mx4[1], fmaxf(mx4[2], mx4[3])) * sl2;
          if (__any_sync(0xffffffffu, top > m + kTcLazy)) {
            const float mn = fmaxf(m, top);
            const float up = mn == -INFINITY ? 1.0f : kv_ex2(m - mn);
            m = mn;
            l *= up;
            if (j > 0) {
#pragma unroll
              for (int c = 0; c < D / 32; ++c) {
                uint32_t o[32];
                tmem_ld_32x32b_x32(o_col + 32 * c, o);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * up);
                tmem_st_32x32b_x32(o_col + 32 * c, o);
              }
            }
          }
          const float base = m == -INFINITY ? 0.0f : m;
          uint64_t l2[4] = {0ull, 0ull, 0ull, 0ull};  // pairs of partial row sums
          const uint64_t sc2 = pack_f32x2(sl2, sl2), base2 = pack_f32x2(-base, -base);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t pk[16];
            if ((shut >> c) & 1u) {
#pragma unroll
              for (int e = 0; e < 16; ++e) pk[e] = 0u;
            } else {
#pragma unroll
              for (int e = 0; e < 32; e += 2) {
                const float2 x = unpack_f32x2(fma_f32x2(pack_f32x2(s[c][e], s[c][e + 1]), sc2, base2));
                const float p0 = kv_ex2(x.x), p1 = kv_ex2(x.y);
                l2[(e >> 1) & 3] = add_f32x2(l2[(e >> 1) & 3], pack_f32x2(p0, p1));
                pk[e >> 1] = pack_p<T>(p0, p1);
              }
            }
            tmem_st_32x32b_x16(s_col + 16 * c, pk);
          }
          const float2 la = unpack_f32x2(add_f32x2(add_f32x2(l2[0], l2[1]), add_f32x2(l2[2], l2[3])));
          l += la.x + la.y;
          tmem_st_wait();
        }
        tc_fence_before();
        mbar_arrive(p_full + i);
      }
      if (ok) {
        const bool got = steps == 0 || (mbar_wait(o_full + i, 0) && !*abort_flag);
        ok = __all_sync(0xffffffffu, got);
      }
      if (!ok) {
        *abort_flag = 1;
        if (lane == 0) atomicOr(a.err, kErrAttnWait);
      } else if (any) {
        tc_fence_after();
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        T* op = static_cast<T*>(a.out.p) + grow * a.out.ld + head * a.out.hs;
        bool nan = l != l;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          if (steps > 0) {
            tmem_ld_32x32b_x32(o_col + 32 * c, o);
            tmem_ld_wait();
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = 0u;
          }
          if (mine) {
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              const float v0 = __uint_as_float(o[e]) * inv, v1 = __uint_as_float(o[e + 1]) * inv;
              nan |= v0 != v0 || v1 != v1;
              pk[e >> 1] = kv_pack<T>(v0, v1);
            }
            if (tc.vec_o) {
              uint4* dst = reinterpret_cast<uint4*>(op + 32 * c);
#pragma unroll
              for (int u = 0; u < 4; ++u) dst[u] = make_uint4(pk[4 * u], pk[4 * u + 1], pk[4 * u + 2], pk[4 * u + 3]);
            } else {
              uint16_t* dst = reinterpret_cast<uint16_t*>(op + 32 * c);
#pragma unroll
              for (int u = 0; u < 16; ++u) dst[2 * u] = pk[u] & 0xFFFFu, dst[2 * u + 1] = pk[u] >> 16;
            }
          }
        }
        uint32_t redo = __ballot_sync(0xffffffffu, mine && nan);
        __syncwarp();
        while (redo) {
          const int w = __ffs(redo) - 1;
          redo &= redo - 1;
          const int xr = rw0 + w, xt = xr / group, xh = kvh * group + xr % group;
          const long long xg = static_cast<long long>(sq.row0) + xt;
          kv_attend_row<T, 16, D>(a, seq, base_t + xt, xh, static_cast<const T*>(a.q.p) + xg * a.q.ld + xh * a.q.hs,
                                  static_cast<T*>(a.out.p) + xg * a.out.ld + xh * a.out.hs);
        }
      }
    }
  } else {
    for (int r = warp; r < rows; r += kTcThreads / 32) {
      const int xr = r0 + r, xt = xr / group, xh = kvh * group + xr % group;
      const long long xg = static_cast<long long>(sq.row0) + xt;
      kv_attend_row<T, 16, D>(a, seq, base_t + xt, xh, static_cast<const T*>(a.q.p) + xg * a.q.ld + xh * a.q.hs,
                              static_cast<T*>(a.out.p) + xg * a.out.ld + xh * a.out.hs);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <typename T, int D>
cudaError_t launch_tc(const KvAttnArgs& a, cudaStream_t s) {
  using C = TcCfg<D>;
  const long long group = a.heads / a.c.kv_heads;
  TcArgs tc{};
  tc.supers = static_cast<int>((a.st.max_new * group + 2 * kRows - 1) / (2 * kRows));
  tc.pool_rows = a.c.pages * a.c.kv_heads * a.c.page_size;
  auto fits = [](const KvRows& r) {
    return (reinterpret_cast<uintptr_t>(r.p) & 15) == 0 && r.ld % 8 == 0 && r.hs % 8 == 0;
  };
  tc.vec_q = fits(a.q);
  tc.vec_o = fits(a.out);
  tc.shift = a.c.page_size % 64 == 0 ? 6 : a.c.page_size % 32 == 0 ? 5 : 4;
  tc.page = KvDiv(static_cast<unsigned>(a.c.page_size >> tc.shift));
  CUtensorMap mk, mv;
  const int op = std::is_same<T, __half>::value ? kOpF16 : kOpBF16;
  if (!make_operand_map(&mk, a.c.k, op, tc.pool_rows, D, D, 1 << tc.shift) ||
      !make_operand_map(&mv, a.c.v, op, tc.pool_rows, D, D, 1 << tc.shift))
    return cudaErrorInvalidValue;
  cudaError_t e = cudaFuncSetAttribute(kv_attention_tc_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
  if (e != cudaSuccess) return e;
  // the warpgroups' shares add up to the launch's registers only if it has this many
  cudaFuncAttributes at{};
  if ((e = cudaFuncGetAttributes(&at, kv_attention_tc_kernel<T, D>)) != cudaSuccess) return e;
  if (at.numRegs != kTcRegs) return cudaErrorInvalidConfiguration;
  const dim3 grid(static_cast<unsigned>(tc.supers) * a.c.kv_heads, a.st.sequences);
  kv_attention_tc_kernel<T, D><<<grid, kTcThreads, C::SMEM, s>>>(mk, mv, a, tc);
  return cudaGetLastError();
}

}  // namespace

// Rows from which the tensor-core tiles are used: a 128-row tile costs the same for one row as for all.
bool kv_attention_tc_ok(const KvAttnArgs& a) {
  return a.c.bits == 16 && static_cast<long long>(a.st.max_new) * (a.heads / a.c.kv_heads) > 32;
}

cudaError_t launch_kv_attention_tc(const KvAttnArgs& a, cudaStream_t s) {
  if (a.c.dim == 64) return a.c.f16 ? launch_tc<__half, 64>(a, s) : launch_tc<__nv_bfloat16, 64>(a, s);
  return a.c.f16 ? launch_tc<__half, 128>(a, s) : launch_tc<__nv_bfloat16, 128>(a, s);
}

}  // namespace jc
