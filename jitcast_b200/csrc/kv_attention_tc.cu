// Cache attention of many query rows a key (prompts, prompt chunks) on the 5th-generation tensor cores.
//
// A CTA takes 256 packed rows (token · group + head of the group) of one sequence and kv head as two 128-row tiles,
// and walks the keys that they see 128 at a time (8 of the 16-key blocks: sinks first, then the band):
//
//   S_i = Q_i · Kᵀ    tcgen05.mma kind::f16, Q and K K-major in shared memory, S in TMEM (128 × 128 FP32)
//   O_i += P_i · V    P from TMEM (over S's columns, 16 bits), V MN-major in shared memory, O in TMEM
//
// Four softmax warps a tile (a thread a row: running maximum and sum need no shuffle), one TMA producer warp (a lane
// a block of keys: pages may lie anywhere) and one MMA issuer. The two tiles alternate: while one tile's products run,
// the other's exponentials do, and both read each K and V tile once from shared memory, which halves the bytes from L2.
// What bounds it: at 64 dims the exponentials (128 · 128 a tile at 16 a clock and SM: 1024 clocks, against 512 for the
// products); at 128 dims the products' rate would take 1024 too, but S, both of whose operands come from shared memory, was
// measured at 632 clocks a tile for 512 by rate. A step takes 1.5 to 1.9 times that, the latencies of the chain product →
// TMEM load → exponentials → TMEM store → product that the other tile (or CTA) does not cover. Taking some exponentials on the FMA
// units by a polynomial made it slower (issue slots), P in TMEM columns of its own too (one more handshake a step).
//
// S(j + 1) is issued after P·V(j) of its tile by the same thread, so when a softmax warp sees S(j + 1) ready, O holds
// every P·V up to j and no product is touching it: the rare rescaling of O (where the running maximum moves by much)
// needs no barrier of its own.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "copies.h"
#include "gemm.h"
#include "kv_attention.cuh"

namespace jc {

namespace {

constexpr int kRows = 128;   // rows of a tile (TMEM lanes)
constexpr float kTcLog2e = 1.4426950408889634f;
constexpr float kTcLazy = 8.0f;
constexpr int kUnpack = 7;   // warps that unpack a 4-bit cache's tiles (8 and 10 to 15)

// LONG 0 (64 dims): 64 keys a step, so that S and O of both tiles take 256 TMEM columns and two CTAs fit on an SM: a
// CTA's start and end run under the other's steps.
// LONG 1: 128 keys a step and one CTA an SM; its softmax warps hold their rows' 128 scores, for which the other
// warpgroups give up registers: of 168 a thread at launch, 2 · 208 + 88 = 3 · 168; over a 4-bit cache, with a fourth
// warpgroup for the unpacking, of 128, 2 · 184 + 2 · 72 = 4 · 128.
template <int BITS, int D, int LONG>
struct TcCfg {
  static_assert(LONG || D == 64, "the short form is for 64 dims");
  static constexpr int KEYS = LONG ? 128 : 64;     // keys of a step
  static constexpr int LOG_KEYS = LONG ? 7 : 6;
  static constexpr int CTAS = LONG ? 1 : 2;        // on an SM
  static constexpr int THREADS = BITS == 4 ? 512 : LONG ? 384 : 320;
  static constexpr bool SPLIT_REGS = LONG, HOLD = LONG;
  static constexpr int REGS = BITS == 4 ? 128 : 168, REGS_SOFTMAX = BITS == 4 ? 184 : 208, REGS_ISSUE = BITS == 4 ? 72 : 88;
  static constexpr int STAGES = LONG && D == 128 ? 2 : 4;
  static constexpr int Q_TILE = kRows * D * 2;     // bytes of a Q (and at the end an output) tile
  static constexpr int TILE = KEYS * D * 2;        // bytes of a K or V tile
  static constexpr int ATOM = KEYS * 128;          // of its 64-dim column blocks (128-byte swizzled rows)
  static constexpr int Q_ATOM = kRows * 128;
  static constexpr int Q_OFF = 0;
  static constexpr int K_OFF = 2 * Q_TILE;
  static constexpr int V_OFF = K_OFF + STAGES * TILE;
  static constexpr int BAR_OFF = V_OFF + STAGES * TILE;
  static constexpr int MUL_OFF = BAR_OFF + 512;    // 4 bits: what each row's q was divided by
  static constexpr int SMEM = MUL_OFF + 2 * kRows * 4 + 1024;
  static constexpr int O_COL = 2 * KEYS;           // TMEM columns: S (and P over it) of both tiles, O of both
  static constexpr int TMEM = LONG ? 512 : 256;
};

struct TcArgs {
  int shift;         // 2^shift keys a block: the largest power of two, up to 64, that a page holds a whole number of
  int supers;        // 256-row tiles of the longest sequence
  int chunk, splits; // blocks that a CTA takes at most (whole steps), CTAs along the longest sequence's keys
  int pool_rows;     // rows of the pools: a coordinate outside them
  int vec_q, vec_o;  // 16-byte vectors
  KvDiv page;        // blocks of a page
};

// Waits for a barrier's phase: true when it completes, false once another role has given up or the limit has passed.
// The clock is read only after some tries: reading %globaltimer takes longer than most waits here.
__device__ __forceinline__ bool bar_wait(uint64_t* bar, uint32_t parity, const volatile uint32_t* abort_flag) {
#pragma unroll 1
  for (int i = 0; i < 32; ++i)
    if (mbar_try_wait_long(bar, parity)) return true;
  const uint64_t t0 = globaltimer();
  while (!mbar_try_wait_long(bar, parity))
    if (*abort_flag || globaltimer() - t0 > kWaitLimitNs) return false;
  return true;
}

// Waits for a phase of what is in flight at the end, some 100 ms at most.
__device__ __forceinline__ void last_wait(uint64_t* bar, uint32_t parity) {
#pragma unroll 1
  for (int i = 0; i < 100; ++i)
    if (mbar_try_wait_long(bar, parity)) return;
}

__device__ __forceinline__ bool elect_one() {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(ok));
  return ok != 0;
}

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

// Two FP32 fused multiply-adds (additions) in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, c, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
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

// The producers over a 4-bit cache: kUnpack warps load a step's codes and scales, and write the FP16 values that they
// stand for as the swizzled K and V tiles. A lane takes 32 dims (one group) of a key: 16 bytes of codes, one (scale, min),
// four 16-byte stores. While a K tile is unpacked the V tile's codes are in flight, and the next K's under the V tile.
// Within each 8 dims the values lie in the order 0, 4, 1, 5, 2, 6, 3, 7, as they come out of a word of codes: Q is written
// in that order too, and the output's columns are put back at the end. Keys that no row sees become zeros.
template <int D, typename C>
__device__ __forceinline__ void unpack_tiles(const KvAttnArgs& a, const TcArgs& tc, const KvSlice& kb, const int* table,
                                             int kvh, int steps, int t0, int t1, uint8_t* smem, uint64_t* k_full,
                                             uint64_t* k_free, uint64_t* v_full, uint64_t* v_free,
                                             volatile uint32_t* abort_flag, int part, int lane) {
  constexpr int TASKS = C::KEYS * (D / 32), ROUNDS = (TASKS + 32 * kUnpack - 1) / (32 * kUnpack);
  struct Codes {
    uint4 c[ROUNDS];
    uint32_t sm[ROUNDS];  // 0: a key that no row sees
  };
  const int size = 1 << tc.shift, per = C::KEYS >> tc.shift, first = kv_first(a, t0);
  // pool row of the lane's block of step j (lanes 0 .. per − 1), fetched a step ahead of its codes
  auto row_of = [&](int j) -> int {
    const int b = j * per + lane;
    if (lane >= per || b >= kb.n) return 0;
    const int kblk = kb.at(b);
    const unsigned pg = tc.page.of(kblk);
    return (__ldg(table + pg) * a.c.kv_heads + kvh) * a.c.page_size + ((kblk - static_cast<int>(pg * tc.page.d)) << tc.shift);
  };
  auto load = [&](int j, int rows, const void* pool, const void* scale, Codes& x) {
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
      const int task = (r * kUnpack + part) * 32 + lane, key = task / (D / 32), grp = task % (D / 32);
      const int b = j * per + (key >> tc.shift), in = key & (size - 1), idx = (kb.at(b) << tc.shift) + in;
      const long long row = __shfl_sync(0xffffffffu, rows, (key >> tc.shift) & 31) + in;
      const bool on = task < TASKS && b < kb.n && idx <= t1 && (idx >= first || idx < a.sinks);
      x.c[r] = on ? __ldg(static_cast<const uint4*>(pool) + row * (D / 32) + grp) : make_uint4(0u, 0u, 0u, 0u);
      x.sm[r] = on ? __ldg(static_cast<const uint32_t*>(scale) + row * (D / 32) + grp) : 0u;
    }
  };
  auto unpack = [&](const Codes& x, uint8_t* tile) {
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
      const int task = (r * kUnpack + part) * 32 + lane, key = task / (D / 32), grp = task % (D / 32);
      if (task >= TASKS) continue;
      const __half2 s = __low2half2(*reinterpret_cast<const __half2*>(&x.sm[r])), m = __high2half2(*reinterpret_cast<const __half2*>(&x.sm[r]));
      // groups 2 and 3 (the other column block, same banks) store their words in the order 2, 3, 0, 1
      const bool turn = (grp & 2) != 0;
      const uint32_t w[4] = {turn ? x.c[r].z : x.c[r].x, turn ? x.c[r].w : x.c[r].y, turn ? x.c[r].x : x.c[r].z,
                             turn ? x.c[r].y : x.c[r].w};
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int ch = 4 * grp + (q ^ (grp & 2));
        const __half2 h[4] = {__hfma2(kv_codes<false>(w[q]), s, m), __hfma2(kv_codes<true>(w[q]), s, m),
                              __hfma2(kv_codes<false>(w[q] >> 8), s, m), __hfma2(kv_codes<true>(w[q] >> 8), s, m)};
        *reinterpret_cast<uint4*>(tile + (ch >> 3) * C::ATOM + sw128(key, 8 * (ch & 7))) = *reinterpret_cast<const uint4*>(h);
      }
    }
    fence_proxy_async_smem();
    __syncwarp();
  };
  Codes k, v;
  bool ok = true;
  int rows = row_of(0), rows_n = row_of(1);
  load(0, rows, a.c.k, a.c.k_scale, k);
  for (int j = 0; j < steps; ++j) {
    const int st = j % C::STAGES;
    const uint32_t ph = ((j / C::STAGES) & 1) ^ 1;
    load(j, rows, a.c.v, a.c.v_scale, v);
    rows = rows_n;
    rows_n = row_of(j + 2);
    ok = __all_sync(0xffffffffu, bar_wait(k_free + st, ph, abort_flag));
    if (!ok) break;
    unpack(k, smem + C::K_OFF + st * C::TILE);
    if (lane == 0) mbar_arrive(k_full + st);
    load(j + 1, rows, a.c.k, a.c.k_scale, k);  // past the last step: nothing is seen, nothing read
    ok = __all_sync(0xffffffffu, bar_wait(v_free + st, ph, abort_flag));
    if (!ok) break;
    unpack(v, smem + C::V_OFF + st * C::TILE);
    if (lane == 0) mbar_arrive(v_full + st);
  }
  if (!ok && lane == 0) {
    *abort_flag = 1;
    atomicOr(a.err, kErrAttnWait);
  }
}

template <typename T, int BITS, int D, int LONG>
__global__ void __launch_bounds__((TcCfg<BITS, D, LONG>::THREADS), (TcCfg<BITS, D, LONG>::CTAS))
    kv_attention_tc_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                           const __grid_constant__ KvAttnArgs a, const __grid_constant__ TcArgs tc) {
  using C = TcCfg<BITS, D, LONG>;
  using M = std::conditional_t<BITS == 4, __half, T>;  // the products' type
  static_assert(BITS == 16 || LONG, "a 4-bit cache takes the long form");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::BAR_OFF);
  uint64_t* k_full = bars;                    // [STAGES] TMA → MMA
  uint64_t* k_free = k_full + C::STAGES;      // [STAGES] MMA → TMA
  uint64_t* v_full = k_free + C::STAGES;
  uint64_t* v_free = v_full + C::STAGES;
  uint64_t* s_full = v_free + C::STAGES;      // [2] MMA → softmax: S of the tile ready
  uint64_t* p_full = s_full + 2;              // [2] softmax → MMA: P written (4 warps)
  uint64_t* o_full = p_full + 2;              // [2] MMA → softmax: every product of the tile done
  uint64_t* q_full = o_full + 2;              // [2] softmax → MMA: Q written (4 warps)
  uint64_t* v_raw = q_full + 2;               // [1] TMA → producer: a V tile with hidden rows to clear
  uint64_t* drain = v_raw + 1;                // [1] MMA: every product that it issued has completed
  uint32_t* slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile uint32_t* abort_flag = slot + 1;

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
  const KvBlocks all = kv_blocks(a, t0, t1, tc.shift);
  const int split = blockIdx.z, x0 = split * tc.chunk;
  if (split > 0 && x0 >= all.n) return;
  const bool whole = all.n <= tc.chunk;  // no other CTA has keys of this tile
  const KvSlice kb(all, x0, min(all.n, x0 + tc.chunk));
  const int per = C::KEYS >> tc.shift;  // blocks of a step
  const int steps = (kb.n + per - 1) >> (C::LOG_KEYS - tc.shift);
  const int tiles = rows > kRows ? 2 : 1;
  const int* table = a.st.table + seq * a.st.ld_table;

  if (tid == 0) {
    for (int i = 0; i < C::STAGES; ++i) {
      mbar_init(k_full + i, BITS == 4 ? kUnpack : 1);
      mbar_init(k_free + i, 1);
      mbar_init(v_full + i, BITS == 4 ? kUnpack : 1);
      mbar_init(v_free + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full + i, 1);
      mbar_init(p_full + i, 4);
      mbar_init(o_full + i, 1);
      mbar_init(q_full + i, 4);
    }
    mbar_init(v_raw, 1);
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 9) {
    tmem_alloc(slot, C::TMEM);
    tmem_relinquish();
    tc_fence_before();
  }
  // the warp's 32 rows of Q, 16 bytes a lane and neighbouring lanes in one row
  constexpr int CH = D / 8, RPI = 32 / CH;  // 16-byte chunks of a row, rows of one round
  const int wrow = (warp & 3) * 32;               // the warp's first row of its tile
  const int w0 = r0 + (warp >> 2) * kRows + wrow;  // and its packed row
  const int ch = lane % CH;
  // the lane's rows w0 + lane / CH, + RPI, ..: token and head of the group, without a division each
  struct RowWalk {
    int tok, rem, dt, dr, group;
    __device__ __forceinline__ RowWalk(int r, int step, int g) : tok(r / g), rem(r % g), dt(step / g), dr(step % g), group(g) {}
    __device__ __forceinline__ void next() {
      tok += dt;
      rem += dr;
      if (rem >= group) rem -= group, ++tok;
    }
  };
  uint4 qv[CH];
  if (warp < 8) {
    RowWalk at(w0 + lane / CH, RPI, group);
    const T* base = static_cast<const T*>(a.q.p) + sq.row0 * a.q.ld + kvh * group * a.q.hs + 8 * ch;
    if (tc.vec_q) {
#pragma unroll
      for (int c = 0; c < CH; ++c, at.next()) {
        const bool on = w0 + c * RPI + lane / CH < r0 + rows;  // a row past the last reads the first one, and is zeroed
        const uint4 u = kv_load16(base + (on ? at.tok * a.q.ld + at.rem * a.q.hs : 0));
        qv[c] = make_uint4(on ? u.x : 0u, on ? u.y : 0u, on ? u.z : 0u, on ? u.w : 0u);
      }
    } else {
#pragma unroll
      for (int c = 0; c < CH; ++c, at.next()) {
        qv[c] = make_uint4(0u, 0u, 0u, 0u);
        if (w0 + c * RPI + lane / CH < r0 + rows) {
          const uint16_t* h = reinterpret_cast<const uint16_t*>(base + at.tok * a.q.ld + at.rem * a.q.hs);
          qv[c].x = h[0] | static_cast<uint32_t>(h[1]) << 16, qv[c].y = h[2] | static_cast<uint32_t>(h[3]) << 16;
          qv[c].z = h[4] | static_cast<uint32_t>(h[5]) << 16, qv[c].w = h[6] | static_cast<uint32_t>(h[7]) << 16;
        }
      }
    }
  }
  // every page that the tile reads lies in the pool, or the rows go the row-by-row way, which leaves such pages out
  int bad = 0;
  for (int x = tid; x < kb.n; x += C::THREADS) {
    const int id = __ldg(table + tc.page.of(kb.at(x)));
    bad |= id < 0 || id >= a.c.pages;
  }
  // the producer's blocks of the first step, looked up under the barrier
  const int pblk = lane & (per - 1), patom = lane >> (C::LOG_KEYS - tc.shift);
  auto row_of = [&](int j) -> int {  // pool row of the lane's block in step j; past the last: outside the pool, zeros
    const int x = j * per + pblk;
    if (patom >= D / 64 || x >= kb.n) return tc.pool_rows;
    const int b = kb.at(x);
    const unsigned pg = tc.page.of(b);
    return (__ldg(table + pg) * a.c.kv_heads + kvh) * a.c.page_size + ((b - static_cast<int>(pg * tc.page.d)) << tc.shift);
  };
  const int row_first = BITS == 16 && warp == 8 ? row_of(0) : 0;
  const bool good = __syncthreads_or(bad) == 0;
  tc_fence_after();
  const uint32_t tmem = *slot;
  uint32_t redo = 0u;  // rows of the warp to be worked out again, key by key

  if (good && warp >= 8) {
    if constexpr (C::SPLIT_REGS) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REGS_ISSUE));
    if (BITS == 4 && warp != 9) {
      if constexpr (BITS == 4) {
        unpack_tiles<D, C>(a, tc, kb, table, kvh, steps, t0 < 0 ? 0 : t0, t1, smem, k_full, k_free, v_full, v_free, abort_flag,
                           warp == 8 ? 0 : warp - 9, lane);
      }
    } else if (BITS == 16 && warp == 8) {
      // ---- producer: lane = block (and 64-dim column block) of a step ----
      const int blk = pblk, atom = patom;
      const bool mine = atom < D / 64;
      const int size = 1 << tc.shift, first = kv_first(a, t0 < 0 ? 0 : t0);
      const uint32_t off = atom * C::ATOM + blk * (size * 128);
      bool ok = true;
      uint32_t raw_phase = 0;
      int k_sent = 0, v_sent = 0;  // steps whose copies complete on k_full, v_full
      bool raw_sent = false;       // a V tile is on its way to v_raw
      int row = row_first;
      for (int j = 0; j < steps && ok; ++j) {
        const int st = j % C::STAGES;
        const uint32_t ph = (j / C::STAGES) & 1;
        const int next = row_of(j + 1);  // in flight during this step's waits
        ok = bar_wait(k_free + st, ph ^ 1, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(k_full + st, C::TILE);
        __syncwarp();
        if (mine) tma_load_2d(smem + C::K_OFF + st * C::TILE + off, &tmK, k_full + st, 64 * atom, row);
        k_sent = j + 1;
        ok = bar_wait(v_free + st, ph ^ 1, abort_flag);
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
          raw_sent = true;
          ok = __all_sync(0xffffffffu, bar_wait(v_raw, raw_phase, abort_flag));
          if (!ok) break;
          raw_phase ^= 1;
          raw_sent = false;
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
        v_sent = j + 1;
        row = next;
      }
      if (lane == 0) {
        if (!ok) {
          *abort_flag = 1;
          atomicOr(a.err, kErrAttnWait);
        }
        // No copy is in flight when the CTA's shared memory can go, whichever role gave up
        for_last_copies(k_sent, C::STAGES, [&](int i, uint32_t parity) { last_wait(k_full + i, parity); });
        for_last_copies(v_sent, C::STAGES, [&](int i, uint32_t parity) { last_wait(v_full + i, parity); });
        if (raw_sent) last_wait(v_raw, raw_phase);
      }
      __syncwarp();
    } else if (warp == 9) {
      // ---- MMA issuer ----
      // The whole warp runs it, one elected lane issues: what the instructions take stays in uniform registers (with one
      // lane in a branch of its own, an MMA took 80 clocks to issue).
      if (steps > 0) {
        const bool leader = elect_one();
        constexpr uint32_t fmt = std::is_same<M, __half>::value ? 0u : 1u;
        constexpr uint32_t is = idesc_f32acc(fmt, kRows, C::KEYS);
        constexpr uint32_t io = idesc_f32acc(fmt, kRows, D) | (1u << 16);  // B (V) MN-major
        const uint32_t qa = smem_u32(smem + C::Q_OFF), ka = smem_u32(smem + C::K_OFF), va = smem_u32(smem + C::V_OFF);
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t ph) {
          ok = ok && __all_sync(0xffffffffu, bar_wait(bar, ph, abort_flag));
          return ok;
        };
        auto scores = [&](int i, int j) {  // S_i of step j
          if (!leader) return;
          const uint32_t q = qa + i * C::Q_TILE, k = ka + (j % C::STAGES) * C::TILE;
#pragma unroll
          for (int d = 0; d < D / 16; ++d)
            umma_bf16(tmem + i * C::KEYS, sdesc_k_sw128(q + (d >> 2) * C::Q_ATOM + 32 * (d & 3)),
                      sdesc_k_sw128(k + (d >> 2) * C::ATOM + 32 * (d & 3)), is, d > 0);
          umma_commit(s_full + i);
        };
        auto commit = [&](uint64_t* bar) {
          if (leader) umma_commit(bar);
        };
        auto values = [&](int i, int j) {  // O_i of step j
          if (!leader) return;
          const uint32_t v = va + (j % C::STAGES) * C::TILE;
#pragma unroll
          for (int k = 0; k < C::KEYS / 16; ++k)
            umma_f16_ts(tmem + C::O_COL + i * D, tmem + i * C::KEYS + 8 * k, sdesc_v(v + 2048 * k, C::ATOM), io,
                        j > 0 || k > 0);
        };
        wait(k_full, 0);
        for (int i = 0; i < tiles && ok; ++i) {
          // long walks: tile 1 starts when tile 0 has its first P, and the offset stays: one tile's exponentials run
          // under the other's products (20,000 keys, 64 dims: 288 -> 256 us)
          if (!wait(q_full + i, 0) || (C::KEYS == 128 && i == 1 && steps > 24 && !wait(p_full, 0))) break;
          tc_fence_after();
          scores(i, 0);
        }
        if (ok) commit(k_free);
        for (int j = 0; j < steps && ok; ++j) {
          const int jn = j + 1;
          if (jn < steps) wait(k_full + jn % C::STAGES, (jn / C::STAGES) & 1);
          wait(v_full + j % C::STAGES, (j / C::STAGES) & 1);
          for (int i = 0; i < tiles && ok; ++i) {
            if (!wait(p_full + i, j & 1)) break;
            tc_fence_after();
            values(i, j);
            if (jn < steps)
              scores(i, jn);
            else
              commit(o_full + i);
          }
          if (ok) {
            commit(v_free + j % C::STAGES);
            if (jn < steps) commit(k_free + jn % C::STAGES);
          }
        }
        if (leader) {
          if (!ok) {
            *abort_flag = 1;
            atomicOr(a.err, kErrAttnWait);
          }
          umma_commit(drain);  // every product issued has completed once this flips, whichever role gave up
          last_wait(drain, 0);
        }
      }
      __syncwarp();
    }
  } else if (good) {
    // ---- softmax: tile i, a thread a row ----
    if constexpr (C::SPLIT_REGS) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::REGS_SOFTMAX));
    const int i = warp >> 2;
    if (i < tiles) {
      uint8_t* qs = smem + C::Q_OFF + i * C::Q_TILE;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int row = wrow + c * RPI + lane / CH;
        uint4 u = qv[c];
        if constexpr (BITS == 4) {
          // FP16, divided by the power of two of the row's largest element (BF16's range does not matter then), in the
          // order of dims that the unpacked keys have: (0, 4), (1, 5), (2, 6), (3, 7) of each 8
          const float2 f0 = kv_unpack<T>(u.x), f1 = kv_unpack<T>(u.y), f2 = kv_unpack<T>(u.z), f3 = kv_unpack<T>(u.w);
          float most = fmaxf(fmaxf(fmaxf(fabsf(f0.x), fabsf(f0.y)), fmaxf(fabsf(f1.x), fabsf(f1.y))),
                             fmaxf(fmaxf(fabsf(f2.x), fabsf(f2.y)), fmaxf(fabsf(f3.x), fabsf(f3.y))));
#pragma unroll
          for (int w = 1; w < CH; w <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, w));
          const uint32_t eb = __float_as_uint(most) & 0x7F800000u;
          const float mul = eb != 0u && eb != 0x7F800000u ? __uint_as_float(eb) : 1.0f, inv = 1.0f / mul;
          u = make_uint4(pack_p<__half>(f0.x * inv, f2.x * inv), pack_p<__half>(f0.y * inv, f2.y * inv),
                         pack_p<__half>(f1.x * inv, f3.x * inv), pack_p<__half>(f1.y * inv, f3.y * inv));
          if (ch == 0) reinterpret_cast<float*>(smem + C::MUL_OFF)[i * kRows + row] = mul;
        }
        *reinterpret_cast<uint4*>(qs + (ch >> 3) * C::Q_ATOM + sw128(row, 8 * (ch & 7))) = u;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full + i);

      const bool any = w0 < r0 + rows;  // the warp has a row
      const bool mine = w0 + lane < r0 + rows;
      // the thread's token and the warp's
      const int w1 = min(w0 + 31, r0 + rows - 1);
      const int t = base_t + min(w0 + lane, w1) / group, first = kv_first(a, t < 0 ? 0 : t);
      const int tw0 = base_t + w0 / group, tw1 = base_t + w1 / group;
      const int fw0 = kv_first(a, tw0 < 0 ? 0 : tw0), fw1 = kv_first(a, tw1 < 0 ? 0 : tw1);
      const uint32_t lanes = tmem + (static_cast<uint32_t>(wrow) << 16);
      const uint32_t s_col = lanes + i * C::KEYS, o_col = lanes + C::O_COL + i * D;
      const float sl2 = a.scale * kTcLog2e * (BITS == 4 ? reinterpret_cast<const float*>(smem + C::MUL_OFF)[i * kRows + wrow + lane] : 1.0f);
      // steps open0 .. open1 − 1 lie in the band, and every row of the warp sees every key of them
      const int to_band = kb.a - kb.b;  // block x of the band is key block x − to_band
      const int open0 = (max(kb.a, to_band + ((fw1 + (1 << tc.shift) - 1) >> tc.shift)) + per - 1) / per;
      const int last_open = tw0 + 1 < C::KEYS ? -1 : to_band + ((tw0 + 1 - C::KEYS) >> tc.shift);  // a step's first block
      const int open1 = last_open < 0 ? 0 : last_open / per + 1;
      float m = -INFINITY, l = 0.0f;
      bool ok = true;
      for (int j = 0; j < steps; ++j) {
        const bool got = bar_wait(s_full + i, j & 1, abort_flag);
        ok = __all_sync(0xffffffffu, got);
        if (!ok) break;
        tc_fence_after();
        if (any) {
          constexpr int NC = C::KEYS / 32;
          auto load = [&](int c, float (&x)[32]) { tmem_ld_32x32b_x32(s_col + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(x)); };
          // raises the running maximum to `top` and takes l and O along
          auto raise = [&](float top) {
            const float mn = fmaxf(m, top);
            const float up = mn == -INFINITY ? 1.0f : kv_ex2(m - mn);
            m = mn;
            l *= up;
            if (j > 0) {
#pragma unroll 1
              for (int c = 0; c < D / 32; ++c) {
                uint32_t o[32];
                tmem_ld_32x32b_x32(o_col + 32 * c, o);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * up);
                tmem_st_32x32b_x32(o_col + 32 * c, o);
              }
            }
          };
          float2 ls[2];  // the step's row sum, in four chains
          // P of a chunk: 2^(x · sl2 − base), its sums in FP32 before the rounding to 16 bits
          auto probabilities = [&](const float (&x)[32], float base, uint32_t (&pk)[16]) {
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              const float2 y = fma2(make_float2(x[e], x[e + 1]), make_float2(sl2, sl2), make_float2(-base, -base));
              const float2 p = make_float2(kv_ex2(y.x), kv_ex2(y.y));
              ls[(e >> 1) & 1] = add2(ls[(e >> 1) & 1], p);
              pk[e >> 1] = pack_p<M>(p.x, p.y);
            }
          };
          auto row_sum = [&] { return (ls[0].x + ls[0].y) + (ls[1].x + ls[1].y); };
          // A step that every row of the warp sees whole, once there is a maximum to take the exponentials against: the
          // scores stay in registers. Only where a row's sum then shows that a score had passed the running maximum by
          // much, the step's own is taken and the exponentials once more. P is no larger than its row's sum: what
          // kMost lets through fits FP16.
          if (C::HOLD && j >= open0 && j < open1 && !__any_sync(0xffffffffu, m == -INFINITY)) {
            constexpr float kMost = std::is_same<M, __half>::value ? 65504.0f : 16384.0f;
            float s[NC][32];
#pragma unroll
            for (int c = 0; c < NC; ++c) load(c, s[c]);
            tmem_ld_wait();
            for (bool again = false;;) {
              ls[0] = ls[1] = make_float2(0.0f, 0.0f);
#pragma unroll
              for (int c = 0; c < NC; ++c) {
                uint32_t pk[16];
                probabilities(s[c], m - kProbUp<M>, pk);
                tmem_st_32x32b_x16(s_col + 16 * c, pk);
              }
              if (again || !__any_sync(0xffffffffu, !(row_sum() <= kMost))) break;
              again = true;
              tmem_st_wait();  // the same columns are written once more
              float mx = s[0][0];
#pragma unroll
              for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int e = 0; e < 32; ++e) mx = fmaxf(mx, s[c][e]);
              raise(mx * sl2);
            }
            l += row_sum();
          } else {
            // Any other step, by 32 keys read twice: for the maximum (raised where a score passes it by 2^kLazy), then
            // for P, with what a row does not see hidden and what no row of the warp sees skipped.
            const int sub = tc.shift - 4;
            auto chunk_keys = [&](int c, int& ka, int& kc) {  // first keys of the chunk's two 16-key halves
              const int ha = 2 * NC * j + 2 * c, hc = ha + 1;
              ka = (kb.at(ha >> sub) << tc.shift) + ((ha & ((1 << sub) - 1)) << 4);
              kc = (kb.at(hc >> sub) << tc.shift) + ((hc & ((1 << sub) - 1)) << 4);
            };
            auto closed = [&](int k) { return k > tw1 || (k + 15 < fw0 && k >= a.sinks); };
            auto hide = [&](int ka, int kc, float (&x)[32]) {
              if (ka + 31 <= tw0 && ka >= fw1 && kc == ka + 16) return;
              const uint32_t bits = block_bits(ka, t, first, a.sinks) | block_bits(kc, t, first, a.sinks) << 16;
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!((bits >> e) & 1u)) x[e] = -INFINITY;
            };
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
            for (int c = 0; c < NC; ++c) {
              int ka, kc;
              chunk_keys(c, ka, kc);
              if (closed(ka) && closed(kc)) continue;
              float x[32];
              load(c, x);
              tmem_ld_wait();
              hide(ka, kc, x);
#pragma unroll
              for (int e = 0; e < 32; e += 2) mx[(e >> 1) & 3] = fmax3(mx[(e >> 1) & 3], x[e], x[e + 1]);
            }
            const float top = fmax3(mx[0], mx[1], fmaxf(mx[2], mx[3])) * sl2;
            if (__any_sync(0xffffffffu, top > m + kTcLazy)) raise(top);
            const float base = (m == -INFINITY ? 0.0f : m) - kProbUp<M>;
            ls[0] = ls[1] = make_float2(0.0f, 0.0f);
#pragma unroll 1
            for (int c = 0; c < NC; ++c) {
              // P over S: chunk c goes over S's columns 16 c .. 16 c + 15, whose chunk (c / 2) has been read by now
              uint32_t pk[16];
              int ka, kc;
              chunk_keys(c, ka, kc);
              if (closed(ka) && closed(kc)) {
#pragma unroll
                for (int e = 0; e < 16; ++e) pk[e] = 0u;
              } else {
                float x[32];
                load(c, x);
                tmem_ld_wait();
                hide(ka, kc, x);
                probabilities(x, base, pk);
              }
              tmem_st_32x32b_x16(s_col + 16 * c, pk);
            }
            l += row_sum();
          }
          tmem_st_wait();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + i);
      }
      if (ok) {
        const bool got = steps == 0 || bar_wait(o_full + i, 0, abort_flag);
        ok = __all_sync(0xffffffffu, got);
      }
      if (!ok) {
        *abort_flag = 1;
        if (lane == 0) atomicOr(a.err, kErrAttnWait);
      } else if (any) {
        tc_fence_after();
        if (!whole) {  // O as it stands, and the row's maximum and sum
          const int r = w0 + lane, tok = r / group, head = kvh * group + r - tok * group;
          const long long row = (static_cast<long long>(sq.row0) + tok) * a.heads + head;
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            tmem_ld_32x32b_x32(o_col + 32 * c, o);
            tmem_ld_wait();
            if (!mine) continue;
            float4* dst = reinterpret_cast<float4*>(part_o(a, split, row, D) + 32 * c);
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              const int c0 = BITS == 16 ? e : (e & ~7) + (e & 4 ? 1 : 0), st = BITS == 16 ? 1 : 2;  // as below
              dst[e >> 2] = make_float4(__uint_as_float(o[c0]), __uint_as_float(o[c0 + st]),
                                        __uint_as_float(o[c0 + (BITS == 16 ? 2 : 4)]), __uint_as_float(o[c0 + (BITS == 16 ? 3 : 6)]));
            }
          }
          if (mine) *part_ml(a, tc.splits, split, row, D) = make_float2(m, l);
        } else {
          const float inv = m == -INFINITY || l == 0.0f ? 0.0f : 1.0f / l;  // no maximum: no key seen
          bool nan = l != l || (inv == 0.0f && t >= 0);  // undefined, or a token of an index that has seen no key
          // the row's values through the tile's (consumed) Q into whole-row stores
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
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              // the columns of dims e, e + 1 (4 bits: unpacked values lie in the order 0, 4, 1, 5, 2, 6, 3, 7)
              const int c0 = BITS == 16 ? e : (e & ~7) + (e & 4 ? 1 : 0) + (e & 2 ? 4 : 0), c1 = BITS == 16 ? e + 1 : c0 + 2;
              const float v0 = __uint_as_float(o[c0]) * inv, v1 = __uint_as_float(o[c1]) * inv;
              nan |= v0 != v0 || v1 != v1;
              // FP16 saturates; a row with a NaN is computed again below
              if constexpr (std::is_same<T, __half>::value)
                pk[e >> 1] = pack_p<T>(fminf(fmaxf(v0, -65504.0f), 65504.0f), fminf(fmaxf(v1, -65504.0f), 65504.0f));
              else
                pk[e >> 1] = pack_p<T>(v0, v1);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u)
              *reinterpret_cast<uint4*>(qs + (c >> 1) * C::Q_ATOM + sw128(wrow + lane, 8 * (4 * (c & 1) + u))) =
                  make_uint4(pk[4 * u], pk[4 * u + 1], pk[4 * u + 2], pk[4 * u + 3]);
          }
          // rows to be worked out again are not stored: their q may lie where their output goes
          redo = __ballot_sync(0xffffffffu, mine && nan);
          __syncwarp();
          {
            RowWalk at(w0 + lane / CH, RPI, group);
            T* base = static_cast<T*>(a.out.p) + sq.row0 * a.out.ld + kvh * group * a.out.hs + 8 * ch;
#pragma unroll
            for (int c = 0; c < CH; ++c, at.next()) {
              const int row = c * RPI + lane / CH;
              const uint4 v = *reinterpret_cast<const uint4*>(qs + (ch >> 3) * C::Q_ATOM + sw128(wrow + row, 8 * (ch & 7)));
              T* op = base + at.tok * a.out.ld + at.rem * a.out.hs;
              if (w0 + row > w1 || ((redo >> row) & 1u)) continue;
              if (tc.vec_o) {
                *reinterpret_cast<uint4*>(op) = v;
              } else {
                uint16_t* h = reinterpret_cast<uint16_t*>(op);
                h[0] = v.x & 0xFFFFu, h[1] = v.x >> 16, h[2] = v.y & 0xFFFFu, h[3] = v.y >> 16;
                h[4] = v.z & 0xFFFFu, h[5] = v.z >> 16, h[6] = v.w & 0xFFFFu, h[7] = v.w >> 16;
              }
            }
          }
        }
      }
    }
  } else if (warp < 8) {
    const int r = w0 + lane;
    if (whole)
      redo = __ballot_sync(0xffffffffu, r < r0 + rows);
    else if (r < r0 + rows)  // the join works a row out again whose sum is not a number
      *part_ml(a, tc.splits, split, (static_cast<long long>(sq.row0) + r / group) * a.heads + kvh * group + r % group, D) =
          make_float2(0.0f, NAN);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, C::TMEM);
  }
  for (; redo; redo &= redo - 1) {
    const int r = w0 + __ffs(redo) - 1, tok = r / group, head = kvh * group + r % group;
    const long long row = static_cast<long long>(sq.row0) + tok;
    kv_attend_row<T, BITS, D>(a, seq, base_t + tok, head, static_cast<const T*>(a.q.p) + row * a.q.ld + head * a.q.hs,
                              static_cast<T*>(a.out.p) + row * a.out.ld + head * a.out.hs);
  }
}

// The most blocks of 2^shift keys that a 256-row tile reads.
long long most_blocks(const KvAttnArgs& a, int shift) {
  const long long group = a.heads / a.c.kv_heads, tokens = (2 * kRows + group - 2) / group + 1, size = 1ll << shift;
  const long long reach = a.sinks + static_cast<long long>(a.window) + tokens + 2 * (size - 1);
  const long long keys = a.window > 0 && reach < a.st.max_length ? reach : a.st.max_length;
  return (keys + size - 1) / size;
}

template <typename T, int BITS, int D, int LONG>
cudaError_t launch_tc(const KvAttnArgs& a, cudaStream_t s) {
  using C = TcCfg<BITS, D, LONG>;
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
  CUtensorMap mk{}, mv{};
  const int op = std::is_same<T, __half>::value ? kOpF16 : kOpBF16;
  if (BITS == 16 && (!make_operand_map(&mk, a.c.k, op, tc.pool_rows, D, D, 1 << tc.shift) ||
                     !make_operand_map(&mv, a.c.v, op, tc.pool_rows, D, D, 1 << tc.shift)))
    return cudaErrorInvalidValue;
  // once a device: its shared memory, and that the warpgroups' shares add up to the registers of the launch
  static std::atomic<uint64_t> ready{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (!(ready.load(std::memory_order_relaxed) & bit)) {
    e = cudaFuncSetAttribute(kv_attention_tc_kernel<T, BITS, D, LONG>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e != cudaSuccess) return e;
    if (C::SPLIT_REGS) {
      cudaFuncAttributes at{};
      if ((e = cudaFuncGetAttributes(&at, kv_attention_tc_kernel<T, BITS, D, LONG>)) != cudaSuccess) return e;
      if (at.numRegs != C::REGS) return cudaErrorInvalidConfiguration;
    }
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  const int per = C::KEYS >> tc.shift;
  tc.splits = kv_tile_splits(a);
  const long long blocks = most_blocks(a, tc.shift);
  tc.chunk = static_cast<int>(((blocks + tc.splits - 1) / tc.splits + per - 1) / per * per);
  if (tc.chunk < per) tc.chunk = per;
  const dim3 grid(static_cast<unsigned>(tc.supers) * a.c.kv_heads, a.st.sequences, tc.splits);
  kv_attention_tc_kernel<T, BITS, D, LONG><<<grid, C::THREADS, C::SMEM, s>>>(mk, mv, a, tc);
  if (tc.splits > 1) return launch_kv_join(a, tc.shift, tc.chunk, tc.splits, 2 * kRows, s);
  return cudaGetLastError();
}

}  // namespace

// The most keys that a row sees.
static long long most_keys(const KvAttnArgs& a) {
  return a.window > 0 ? std::min<long long>(a.st.max_length, static_cast<long long>(a.window) + a.sinks) : a.st.max_length;
}

static long long tile_ctas(const KvAttnArgs& a) {
  const long long rows = static_cast<long long>(a.st.max_new) * (a.heads / a.c.kv_heads);
  return (rows + 2 * kRows - 1) / (2 * kRows) * a.c.kv_heads * a.st.sequences;
}

// Two CTAs an SM where there are that many, or where a walk is a few steps (64 sequences of 130 tokens: 47 against
// 78 us; 64 of 1000: 394 against 530 us; 36 of 256 new tokens over 4096: alike); one with longer steps where there are
// not (9 of 256 over 20,000, 144 CTAs: 256 against 454 us).
static bool short_tiles(const KvAttnArgs& a) {
  return a.c.bits == 16 && a.c.dim == 64 && (tile_ctas(a) >= 2 * 148 || most_keys(a) <= 512);
}

// The tiles' estimated time in microseconds with their keys in `splits` parts: 128 keys a wave of CTAs in 1.55 (64 dims),
// 1.85 (128 dims), 2.6 (64 dims, two CTAs an SM), over 4 bits 2.5 and 3.5; 10 for the call, and for the join 8 and the parts'
// results written and read at 2 TB/s (2 x 1000 new tokens of 32 heads in 4 parts: 352 us, in one 185).
static double tile_time(const KvAttnArgs& a, int splits) {
  const bool twice = short_tiles(a), wide = a.c.dim == 128;
  const long long slots = twice ? 2 * 148 : 148, waves = (tile_ctas(a) * splits + slots - 1) / slots;
  const double step = a.c.bits == 4 ? (wide ? 3.5 : 2.5) : wide ? 1.85 : twice ? 2.6 : 1.55;
  const double join = splits > 1 ? 8.0 + 2e-6 / 2.0 * static_cast<double>(kv_split_bytes(a, splits)) : 0.0;
  return 10.0 + static_cast<double>(waves) * std::ceil(static_cast<double>(most_keys(a)) / 128.0 / splits) * step + join;
}

// Parts of the keys: the fewest that the estimate likes best, each of 1024 keys at least.
int kv_tile_splits(const KvAttnArgs& a) {
  int best = 1;
  if (short_tiles(a)) return best;
  for (int s = 2; s <= 16 && most_keys(a) / s >= 1024; ++s)
    if (tile_time(a, s) < 0.95 * tile_time(a, best)) best = s;
  return best;
}

// Tiles or splits. A tile walks its keys for 256 rows, however few it has; splits read the keys once every 16 rows. Up to
// 32 rows go to the splits; above, the smaller of two estimates, from calls of 40 to 1024 rows, 500 to 20,000 keys and 1 to
// 1024 kv heads x sequences; splits take 3 ps (128 dims: 5) a row and key and 13 us. 8 kv heads, 20,000 keys, tiles in one
// part: 40 rows 231 us by tiles and 31 by splits (64 dims), 256 rows 297 and 209, 1024 rows 298 and 650 (128 dims);
// 64 x 8 kv heads, 40 rows, 4000 keys: 252 and 461.
bool kv_attention_tc_ok(const KvAttnArgs& a) {
  const long long rows = static_cast<long long>(a.st.max_new) * (a.heads / a.c.kv_heads);
  if (rows <= 32) return false;
  const double keys = static_cast<double>(most_keys(a)), heads = static_cast<double>(a.c.kv_heads) * a.st.sequences;
  const double splits = 13.0 + static_cast<double>((rows + 15) / 16 * 16) * keys * heads * (a.c.dim == 128 ? 5e-6 : 3e-6);
  return tile_time(a, kv_tile_splits(a)) <= splits;
}

cudaError_t launch_kv_attention_tc(const KvAttnArgs& a, cudaStream_t s) {
  if (a.c.bits == 4) {
    if (a.c.dim == 128) return a.c.f16 ? launch_tc<__half, 4, 128, 1>(a, s) : launch_tc<__nv_bfloat16, 4, 128, 1>(a, s);
    return a.c.f16 ? launch_tc<__half, 4, 64, 1>(a, s) : launch_tc<__nv_bfloat16, 4, 64, 1>(a, s);
  }
  if (a.c.dim == 128) return a.c.f16 ? launch_tc<__half, 16, 128, 1>(a, s) : launch_tc<__nv_bfloat16, 16, 128, 1>(a, s);
  if (short_tiles(a)) return a.c.f16 ? launch_tc<__half, 16, 64, 0>(a, s) : launch_tc<__nv_bfloat16, 16, 64, 0>(a, s);
  return a.c.f16 ? launch_tc<__half, 16, 64, 1>(a, s) : launch_tc<__nv_bfloat16, 16, 64, 1>(a, s);
}

}  // namespace jc
