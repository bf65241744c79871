// Attention of new tokens over the paged key/value cache: causal, with a sliding window and sinks.
//
// Token t of a sequence sees the keys j ≤ t with j > t − window (window 0: all) or j < sinks;
// out = Σ_j softmax_j(scale · q·k_j) · v_j, zeros where a token sees no key.
//
// kv_attention_split_kernel: few query rows a key (single tokens, and the heads that share a kv head). HBM bounds
// it: every cached key and value in reach is read once, and 4·D operations a row and key are too few to matter. So
// the keys go from global memory straight into tensor-core fragments, with no shared memory and no barrier in the
// loop: with A = 16 keys × 16 dims and B = 16 dims × 8 query rows,
//
//   Sᵀ = K · Qᵀ    and    Oᵀ = Vᵀ · Pᵀ      (mma.sync m16n8k16, FP32 accumulation)
//
// any order of the dims will do as long as K and Q share it, and any order of O's dims as long as the store undoes
// it: a lane loads 16 contiguous bytes of a key's row and calls them its fragments. V needs pairs of keys in a
// register, which a byte permute of two keys' rows gives; Pᵀ needs Sᵀ's 8 × 8 blocks transposed, which movmatrix does.
// A warp walks its own 16-key blocks with a running maximum and sum and joins the others at the end; a sequence's
// keys are split over blocks of four warps where rows alone would leave SMs idle, and kv_combine_kernel joins those.
//
// 4-bit codes become FP16 in registers: a code under the exponent of 1024 (0x6400) is 1024 + c; subtracting 1024 is
// exact, and one FMA with the pair (scale, min) gives the value, rounded once. Queries go to FP16 divided by a power
// of two that takes their largest element to [1, 2), so that BF16's range does not matter.
#include <cstring>
#include <type_traits>

#include "kv_attention.cuh"
#include "mma_sync.cuh"

namespace jc {

namespace {

constexpr int kWarps = 4;
// CTAs that a call is split into where its rows alone are fewer: one wave of equal ones for one sequence (131,000 keys
// over 4 bits, 64 dims in pages of 64: 52 us, 56 with two waves, 66 with four), many small ones for sequences of any lengths (48 of 5000 to 32,500
// keys: 330 us, 367 with two waves).
constexpr int kCtasOne = 148 * 4, kCtasMany = 148 * 16, kMaxSplits = kCtasMany;
constexpr float kLog2e = 1.4426950408889634f;
// A row's running maximum moves only when a score passes it by this much (as a power of two): probabilities then
// reach 2^8 (FP16: 2^15, see kProbUp), which costs no precision in any of the types, and most blocks rescale nothing.
constexpr float kLazy = 8.0f;

__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ uint32_t lo16(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x5410); }
__device__ __forceinline__ uint32_t hi16(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x7632); }

__device__ __forceinline__ uint32_t h2u(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 u2h(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }

// The registers of SUB 16-key blocks: lane (g, t) = (lane / 4, lane % 4) has keys g and g + 8 of K (a quarter of the
// dims each) and keys 2t, 2t + 1, 2t + 8, 2t + 9 of V (an eighth of the dims each).
template <int BITS, int D, int SUB>
struct Frag;

template <int D>
struct Frag<16, D, 1> {
  uint4 k[2][D / 32];
  uint4 v[4][D / 64];

  __device__ __forceinline__ void load_k(const KvCache& c, long long row, int, int g, int t) {
    const uint4* p = static_cast<const uint4*>(c.k) + (row + g) * (D / 8) + t;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < D / 32; ++i) k[h][i] = __ldg(p + 8 * h * (D / 8) + 4 * i);
  }
  __device__ __forceinline__ void load_v(const KvCache& c, long long row, int, int g, int t) {
    const uint4* p = static_cast<const uint4*>(c.v) + (row + 2 * t) * (D / 8) + g;
#pragma unroll
    for (int h = 0; h < 4; ++h)
#pragma unroll
      for (int i = 0; i < D / 64; ++i) v[h][i] = __ldg(p + ((h & 1) + 8 * (h >> 1)) * (D / 8) + 8 * i);
  }
  __device__ __forceinline__ void hide_v(int, int h) {
#pragma unroll
    for (int i = 0; i < D / 64; ++i) v[h][i] = make_uint4(0u, 0u, 0u, 0u);
  }
  // K's A fragments of dim step j: (key g, key g + 8) × (first, second) pair of the lane's dims
  __device__ __forceinline__ void k_frags(int, uint32_t (&f)[D / 16][4]) const {
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      f[2 * i][0] = k[0][i].x, f[2 * i][1] = k[1][i].x, f[2 * i][2] = k[0][i].y, f[2 * i][3] = k[1][i].y;
      f[2 * i + 1][0] = k[0][i].z, f[2 * i + 1][1] = k[1][i].z, f[2 * i + 1][2] = k[0][i].w,
                 f[2 * i + 1][3] = k[1][i].w;
    }
  }
  // Vᵀ's A fragments of dim tile j: rows g and g + 8 are dims v_dim(j, g) and v_dim(j, g) + v_step
  __device__ __forceinline__ void v_frags(int, uint32_t (&f)[D / 16][4]) const {
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      const uint32_t a[4][4] = {{v[0][i].x, v[0][i].y, v[0][i].z, v[0][i].w},
                                {v[1][i].x, v[1][i].y, v[1][i].z, v[1][i].w},
                                {v[2][i].x, v[2][i].y, v[2][i].z, v[2][i].w},
                                {v[3][i].x, v[3][i].y, v[3][i].z, v[3][i].w}};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        f[4 * i + w][0] = lo16(a[0][w], a[1][w]);
        f[4 * i + w][1] = hi16(a[0][w], a[1][w]);
        f[4 * i + w][2] = lo16(a[2][w], a[3][w]);
        f[4 * i + w][3] = hi16(a[2][w], a[3][w]);
      }
    }
  }
  static __device__ __forceinline__ int v_dim(int j, int g) { return (j >> 2) * 64 + 8 * g + 2 * (j & 3); }
  static constexpr int v_step = 1;
};

template <int D, int SUB>
struct Frag<4, D, SUB> {
  uint32_t k[SUB][2][D / 32];                  // codes of 32 (D = 64: 16) dims from dim t · D / 4
  uint32_t ks[SUB][2];                         // their group's (scale, min)
  uint32_t v[SUB][4][D / 64];                  // codes of 16 (8) dims from dim g · D / 8
  uint32_t vs[SUB][4];

  __device__ __forceinline__ void load_k(const KvCache& c, long long row, int u, int g, int t) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const long long r = row + g + 8 * h;
      if constexpr (D == 128) {
        const uint4 x = __ldg(static_cast<const uint4*>(c.k) + r * 4 + t);
        k[u][h][0] = x.x, k[u][h][1] = x.y, k[u][h][2] = x.z, k[u][h][3] = x.w;
        ks[u][h] = __ldg(static_cast<const uint32_t*>(c.k_scale) + r * 4 + t);
      } else {
        const uint2 x = __ldg(static_cast<const uint2*>(c.k) + r * 4 + t);
        k[u][h][0] = x.x, k[u][h][1] = x.y;
        ks[u][h] = __ldg(static_cast<const uint32_t*>(c.k_scale) + r * 2 + (t >> 1));
      }
    }
  }
  __device__ __forceinline__ void load_v(const KvCache& c, long long row, int u, int g, int t) {
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const long long r = row + 2 * t + (h & 1) + 8 * (h >> 1);
      if constexpr (D == 128) {
        const uint2 x = __ldg(static_cast<const uint2*>(c.v) + r * 8 + g);
        v[u][h][0] = x.x, v[u][h][1] = x.y;
        vs[u][h] = __ldg(static_cast<const uint32_t*>(c.v_scale) + r * 4 + (g >> 1));
      } else {
        v[u][h][0] = __ldg(static_cast<const uint32_t*>(c.v) + r * 8 + g);
        vs[u][h] = __ldg(static_cast<const uint32_t*>(c.v_scale) + r * 2 + (g >> 2));
      }
    }
  }
  __device__ __forceinline__ void hide_v(int u, int h) { vs[u][h] = 0u; }  // scale and minimum 0: values 0
  // as the 16-bit form; the dims of one word are taken in the order (0, 4), (1, 5), (2, 6), (3, 7), which q_order gives Q
  __device__ __forceinline__ void k_frags(int u, uint32_t (&f)[D / 16][4]) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const __half2 s = __low2half2(u2h(ks[u][h])), m = __high2half2(u2h(ks[u][h]));
#pragma unroll
      for (int w = 0; w < D / 32; ++w) {
        const uint32_t x = k[u][h][w], y = x >> 8;
        f[2 * w][h] = h2u(__hfma2(kv_codes<false>(x), s, m));
        f[2 * w][h + 2] = h2u(__hfma2(kv_codes<true>(x), s, m));
        f[2 * w + 1][h] = h2u(__hfma2(kv_codes<false>(y), s, m));
        f[2 * w + 1][h + 2] = h2u(__hfma2(kv_codes<true>(y), s, m));
      }
    }
  }
  __device__ __forceinline__ void v_frags(int u, uint32_t (&f)[D / 16][4]) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // key pairs 2t, 2t + 1 and 2t + 8, 2t + 9
      const __half2 s = u2h(lo16(vs[u][2 * h], vs[u][2 * h + 1])), m = u2h(hi16(vs[u][2 * h], vs[u][2 * h + 1]));
#pragma unroll
      for (int w = 0; w < D / 64; ++w) {
        const uint32_t a = v[u][2 * h][w], b = v[u][2 * h + 1][w];
#pragma unroll
        for (int e = 0; e < 2; ++e) {  // dims 0..3, then 4..7 of the word
          const uint32_t x = e ? hi16(a, b) : lo16(a, b), y = x >> 8;
          f[4 * w][2 * h + e] = h2u(__hfma2(kv_codes<false>(x), s, m));
          f[4 * w + 1][2 * h + e] = h2u(__hfma2(kv_codes<true>(x), s, m));
          f[4 * w + 2][2 * h + e] = h2u(__hfma2(kv_codes<false>(y), s, m));
          f[4 * w + 3][2 * h + e] = h2u(__hfma2(kv_codes<true>(y), s, m));
        }
      }
    }
  }
  static __device__ __forceinline__ int v_dim(int j, int g) { return g * (D / 8) + 8 * (j >> 2) + (j & 3); }
  static constexpr int v_step = 4;
};

struct SplitShape {
  int tiles;        // row tiles of a kv head
  int shift;        // 2^shift keys a block
  int chunk;        // blocks that a CTA takes at most
  int splits;       // CTAs along the longest sequence's keys
  int vec_q, vec_o; // 16-byte vectors of q, 8-byte (4-element) vectors of out
  KvDiv page;       // blocks of a page
};

// The tile's tokens, and where its keys lie.
struct Tile {
  int rows;     // query rows in it
  int t0, t1;   // indexes of its first and last token
  KvBlocks kb;
};

__device__ __forceinline__ Tile tile_of(const KvAttnArgs& a, const KvSeq& q, int group, int r0, int most, int shift) {
  Tile x;
  x.rows = min(q.n * group - r0, most);
  x.t0 = q.length - q.n + r0 / group;
  x.t1 = q.length - q.n + (r0 + x.rows - 1) / group;
  x.kb = x.rows > 0 ? kv_blocks(a, x.t0, x.t1, shift) : KvBlocks{0, 0, 0};
  return x;
}

template <typename T>
__device__ __forceinline__ void store4(T* p, float4 v, bool vec) {
  if (vec) {
    *reinterpret_cast<uint2*>(p) = make_uint2(kv_pack<T>(v.x, v.y), kv_pack<T>(v.z, v.w));
  } else {
    p[0] = kv_round<T>(v.x), p[1] = kv_round<T>(v.y), p[2] = kv_round<T>(v.z), p[3] = kv_round<T>(v.w);
  }
}

template <typename T, int BITS, int D, int NT, int SUB, bool WHOLE>
__global__ void __launch_bounds__(32 * kWarps, NT == 2 ? 2 : BITS == 4 ? 4 : 3) kv_attention_split_kernel(const __grid_constant__ KvAttnArgs a,
                                                                      const __grid_constant__ SplitShape sh) {
  using F = Frag<BITS, D, SUB>;
  using M = std::conditional_t<BITS == 4, __half, T>;  // the products' type
  constexpr int ROWS = 8 * NT, PITCH = D + 4;
  // A step takes SUB 16-key sub-blocks: one block in one page (WHOLE), or SUB blocks that may lie in pages of their own
  constexpr int PAGES = WHOLE ? 1 : SUB, PER = SUB / PAGES, KEYS = 16 * PER;  // KEYS: of a block
  constexpr int SHIFT = PER == 1 ? 4 : PER == 2 ? 5 : 6, STEP = kWarps * PAGES;
  __shared__ float s_o[kWarps][ROWS][PITCH];
  __shared__ float s_m[kWarps][ROWS], s_l[kWarps][ROWS];
  __shared__ uint32_t s_nan;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int seq = blockIdx.z, split = blockIdx.y;
  const int kvh = blockIdx.x / sh.tiles, tile = blockIdx.x - kvh * sh.tiles;
  const KvSeq sq = kv_seq(a.st, a.c.page_size, seq, a.err);
  const int group = a.heads / a.c.kv_heads;
  const int r0 = tile * ROWS;
  const Tile tl = tile_of(a, sq, group, r0, ROWS, SHIFT);
  if (tl.rows <= 0) return;
  const int x1 = min(tl.kb.n, (split + 1) * sh.chunk), x0 = split * sh.chunk;
  if (x0 >= x1 && split > 0) return;

  // Q's fragments (row g + 8 i), in K's order of dims, and what takes each row's products to scaled powers of two
  uint32_t qf[NT][D / 16][2];
  float sl2[NT][2];
  int tq[NT][2];  // index of the lane's rows 2t, 2t + 1 of each 8; −1: no row
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const int r = g + 8 * i, rr = r0 + r;
    const bool on = r < tl.rows;
    const T* p = static_cast<const T*>(a.q.p) + (sq.row0 + (on ? rr / group : 0)) * a.q.ld +
                 (kvh * group + (on ? rr % group : 0)) * a.q.hs;
    uint32_t w[D / 32][4];
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      const int d = BITS == 16 ? 32 * c + 8 * t : t * (D / 4) + 8 * c;
      if (!on) {
        w[c][0] = w[c][1] = w[c][2] = w[c][3] = 0u;
      } else if (sh.vec_q) {
        const uint4 u = kv_load16(p + d);
        w[c][0] = u.x, w[c][1] = u.y, w[c][2] = u.z, w[c][3] = u.w;
      } else {
        const uint16_t* h = reinterpret_cast<const uint16_t*>(p + d);
#pragma unroll
        for (int e = 0; e < 4; ++e) w[c][e] = h[2 * e] | static_cast<uint32_t>(h[2 * e + 1]) << 16;
      }
    }
    float mul = 1.0f;
    if constexpr (BITS == 16) {
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        qf[i][2 * c][0] = w[c][0], qf[i][2 * c][1] = w[c][1];
        qf[i][2 * c + 1][0] = w[c][2], qf[i][2 * c + 1][1] = w[c][3];
      }
    } else {
      float most = 0.0f;
#pragma unroll
      for (int c = 0; c < D / 32; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = kv_unpack<T>(w[c][e]);
          most = fmaxf(most, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
      // 2^e of the largest element, its exponent bits alone (a normal number; 1 for zeros, subnormals, infinities)
      const uint32_t eb = __float_as_uint(most) & 0x7F800000u;
      if (eb != 0u && eb != 0x7F800000u) mul = __uint_as_float(eb);
      const float inv = 1.0f / mul;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        const float2 f0 = kv_unpack<T>(w[c][0]), f1 = kv_unpack<T>(w[c][1]), f2 = kv_unpack<T>(w[c][2]),
                     f3 = kv_unpack<T>(w[c][3]);
        qf[i][2 * c][0] = MmaT<__half>::pack(f0.x * inv, f2.x * inv);
        qf[i][2 * c][1] = MmaT<__half>::pack(f0.y * inv, f2.y * inv);
        qf[i][2 * c + 1][0] = MmaT<__half>::pack(f1.x * inv, f3.x * inv);
        qf[i][2 * c + 1][1] = MmaT<__half>::pack(f1.y * inv, f3.y * inv);
      }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {  // of row 2t + e, whose q the lanes 4 (2t + e) .. hold
      sl2[i][e] = a.scale * kLog2e * __shfl_sync(0xffffffffu, mul, 4 * (2 * t + e));
      const int rq = 2 * t + e + 8 * i;
      tq[i][e] = rq < tl.rows ? sq.length - sq.n + (r0 + rq) / group : -1;
    }
  }

  const int* table = a.st.table + seq * a.st.ld_table;
  // the page of block x; −1: no such block, or an entry outside the pool
  auto page_id = [&](int x) -> int { return x < x1 ? __ldg(table + sh.page.of(tl.kb.at(x))) : -1; };
  // the pool row of block x's first key in that page
  auto pool_row = [&](int x, int id) -> long long {
    if (id < 0 || id >= a.c.pages) {
      if (x < x1 && lane == 0) atomicOr(a.err, kErrKvStep);
      return -1;
    }
    const int b = tl.kb.at(x);
    const int slot = (b - static_cast<int>(sh.page.of(b)) * static_cast<int>(sh.page.d)) << SHIFT;
    return (static_cast<long long>(id) * a.c.kv_heads + kvh) * a.c.page_size + slot;
  };

  F f;
  float o[NT][D / 16][4], m[NT][2], l[NT][2];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
#pragma unroll
    for (int j = 0; j < D / 16; ++j) o[i][j][0] = o[i][j][1] = o[i][j][2] = o[i][j][3] = 0.0f;
    m[i][0] = m[i][1] = -INFINITY;
    l[i][0] = l[i][1] = 0.0f;
  }
  // blocks that every row of the tile sees whole need no mask: those from open0 of the band, up to open_t
  const int open0 = kv_first(a, tl.t1), open_t = tl.t0 - (KEYS - 1);
  // The warp's steps, kWarps apart. A step's K is in flight while the one before it goes through the softmax and P·V,
  // its V from there to its own P·V, and its page ids one step further ahead. A block without a page is hidden as a
  // whole: its registers then hold whatever they held.
  int x = x0 + warp * PAGES;
  long long row[PAGES];
  int idn[PAGES];
#pragma unroll
  for (int p = 0; p < PAGES; ++p) {
    row[p] = pool_row(x + p, page_id(x + p));
    if (row[p] >= 0) {
#pragma unroll
      for (int u = 0; u < PER; ++u) {
        f.load_k(a.c, row[p] + 16 * u, p * PER + u, g, t);
        f.load_v(a.c, row[p] + 16 * u, p * PER + u, g, t);
      }
    }
    idn[p] = page_id(x + STEP + p);
  }
  for (; x < x1; x += STEP) {
    uint32_t on = 0u;
#pragma unroll
    for (int p = 0; p < PAGES; ++p) {
      on |= row[p] >= 0 ? 1u << p : 0u;
      row[p] = pool_row(x + STEP + p, idn[p]);
      idn[p] = page_id(x + 2 * STEP + p);
    }
    float s[SUB][NT][4];
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
      uint32_t kf[D / 16][4];
      f.k_frags(u, kf);
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        s[u][i][0] = s[u][i][1] = s[u][i][2] = s[u][i][3] = 0.0f;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) MmaT<M>::mma(s[u][i], kf[j], qf[i][j][0], qf[i][j][1]);
      }
    }
#pragma unroll
    for (int p = 0; p < PAGES; ++p)
      if (row[p] >= 0) {
#pragma unroll
        for (int u = 0; u < PER; ++u) f.load_k(a.c, row[p] + 16 * u, p * PER + u, g, t);
      }
    // hide what a row does not see
#pragma unroll
    for (int p = 0; p < PAGES; ++p) {
      const int key0 = tl.kb.at(x + p) << SHIFT;
      const bool here = (on >> p) & 1u;
      if (here && key0 <= open_t && (key0 >= open0 || key0 + KEYS <= a.sinks)) continue;
#pragma unroll
      for (int w = 0; w < PER; ++w) {
        const int u = p * PER + w, k0 = key0 + 16 * w;
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int j = k0 + g + 8 * (e >> 1), tt = tq[i][e & 1];
            if (!here || j > tt || (j < kv_first(a, tt) && j >= a.sinks)) s[u][i][e] = -INFINITY;
          }
        // and values that no row sees (slots past the length hold anything)
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const int j = k0 + 2 * t + (h & 1) + 8 * (h >> 1);
          if (!here || j > tl.t1 || (j < kv_first(a, tl.t0) && j >= a.sinks)) f.hide_v(u, h);
        }
      }
    }
    // the running maximum, moved only where a score passes it by 2^kLazy
    float mx[NT][2];
    bool move = false;
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float v = fmaxf(s[0][i][e], s[0][i][e + 2]);
#pragma unroll
        for (int u = 1; u < SUB; ++u) v = fmax3(v, s[u][i][e], s[u][i][e + 2]);
        mx[i][e] = v * sl2[i][e];
        move |= mx[i][e] > m[i][e] + kLazy;
      }
    if (__any_sync(0xffffffffu, move)) {
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float v = mx[i][e];
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, w));
          v = fmaxf(v, m[i][e]);
          const float up = v == -INFINITY ? 1.0f : kv_ex2(m[i][e] - v);
          m[i][e] = v;
          l[i][e] *= up;
#pragma unroll
          for (int j = 0; j < D / 16; ++j) {
            o[i][j][e] *= up;
            o[i][j][e + 2] *= up;
          }
        }
    }
    // P, its sums in FP32 before the rounding to 16 bits, and O
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
      uint32_t pf[NT][2];
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float base = (m[i][e & 1] == -INFINITY ? 0.0f : m[i][e & 1]) - kProbUp<M>;
          p[e] = kv_ex2(fmaf(s[u][i][e], sl2[i][e & 1], -base));
          l[i][e & 1] += p[e];
        }
        pf[i][0] = movmatrix(MmaT<M>::pack(p[0], p[1]));
        pf[i][1] = movmatrix(MmaT<M>::pack(p[2], p[3]));
      }
      uint32_t vf[D / 16][4];
      f.v_frags(u, vf);
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < D / 16; ++j) MmaT<M>::mma(o[i][j], vf[j], pf[i][0], pf[i][1]);
    }
#pragma unroll
    for (int p = 0; p < PAGES; ++p)
      if (row[p] >= 0) {
#pragma unroll
        for (int u = 0; u < PER; ++u) f.load_v(a.c, row[p] + 16 * u, p * PER + u, g, t);
      }
  }

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // join the warps
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = 2 * t + e + 8 * i;
#pragma unroll
      for (int w = 4; w < 32; w <<= 1) l[i][e] += __shfl_xor_sync(0xffffffffu, l[i][e], w);
      if (g == 0) {
        s_m[warp][r] = m[i][e];
        s_l[warp][r] = l[i][e];
      }
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        s_o[warp][r][F::v_dim(j, g)] = o[i][j][e];
        s_o[warp][r][F::v_dim(j, g) + F::v_step] = o[i][j][e + 2];
      }
    }
  if (tid == 0) s_nan = 0u;
  __syncthreads();
  const bool whole = tl.kb.n <= sh.chunk;  // no other CTA has keys of this tile
  for (int w1 = 32 * warp; w1 < tl.rows * (D / 4); w1 += 32 * kWarps) {
    const int w = w1 + lane;
    const bool on = w < tl.rows * (D / 4);
    const int r = on ? w / (D / 4) : 0, d = 4 * (w % (D / 4));
    float mm = s_m[0][r];
#pragma unroll
    for (int k = 1; k < kWarps; ++k) mm = fmaxf(mm, s_m[k][r]);
    const float base = mm == -INFINITY ? 0.0f : mm;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) {
      const float c = kv_ex2(s_m[k][r] - base);
      const float4 v = *reinterpret_cast<const float4*>(&s_o[k][r][d]);
      acc.x = fmaf(v.x, c, acc.x), acc.y = fmaf(v.y, c, acc.y), acc.z = fmaf(v.z, c, acc.z), acc.w = fmaf(v.w, c, acc.w);
      sum = fmaf(s_l[k][r], c, sum);
    }
    const int rr = r0 + r, head = kvh * group + rr % group;
    const long long row = sq.row0 + rr / group;
    if (whole) {
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      acc.x *= inv, acc.y *= inv, acc.z *= inv, acc.w *= inv;
      const bool none = sum == 0.0f && sq.length - sq.n + rr / group >= 0;  // a token of an index sees its own key at least
      // A row to be worked out again is not stored, its q may lie where its output goes; a row's lanes are neighbours
      const bool nan = none || acc.x != acc.x || acc.y != acc.y || acc.z != acc.z || acc.w != acc.w;
      const uint32_t bad = __ballot_sync(0xffffffffu, on && nan) & (D == 128 ? ~0u : 0xFFFFu << (lane & 16));
      if (on && bad == 0u)
        store4(static_cast<T*>(a.out.p) + row * a.out.ld + head * a.out.hs + d, acc, sh.vec_o);
      else if (on && d == 0)
        atomicOr(&s_nan, 1u << r);
    } else if (on) {
      *reinterpret_cast<float4*>(part_o(a, split, row * a.heads + head, D) + d) = acc;
      if (d == 0) *part_ml(a, sh.splits, split, row * a.heads + head, D) = make_float2(mm, sum);
    }
  }
  if (!whole) return;
  __syncthreads();
  for (uint32_t left = s_nan; left; left &= left - 1) {  // the same for every thread
    const int rr = r0 + __ffs(left) - 1, i = rr / group, head = kvh * group + rr % group;
    const long long row = sq.row0 + i;
    kv_attend_row_cta<T, BITS, D>(a, seq, sq.length - sq.n + i, head, static_cast<const T*>(a.q.p) + row * a.q.ld + head * a.q.hs,
                                  static_cast<T*>(a.out.p) + row * a.out.ld + head * a.out.hs, &s_o[0][0][0], &s_m[0][0]);
  }
}

// Joins the splits of an output row: a block a row, D / 4 threads a split at a time, the splits' weights first and
// their sums in a fixed order. It reads what the splits wrote once. Launched under the splits' end (programmatic
// dependent launch), it waits for them on the device. Twelve blocks an SM: with the registers that a row worked out again
// could use (168) there are three (48 sequences, window of 4,096: 141 us against 134).
template <typename T, int BITS, int D>
__global__ void __launch_bounds__(128, 12) kv_combine_kernel(const __grid_constant__ KvAttnArgs a,
                                                         const __grid_constant__ SplitShape sh, int rows_per_tile) {
  constexpr int LANES = D / 4, WAYS = 128 / LANES;
  __shared__ float s_c[kMaxSplits], s_red[8];
  __shared__ float4 s_acc[WAYS][LANES];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const KvSeq sq = kv_seq(a.st, a.c.page_size, blockIdx.y, a.err);
  const int group = a.heads / a.c.kv_heads;
  const int i = blockIdx.x / a.heads, head = blockIdx.x - i * a.heads;
  const int r = i * group + head % group;  // its row of the kv head
  const Tile tl = tile_of(a, sq, group, r / rows_per_tile * rows_per_tile, rows_per_tile, sh.shift);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (i >= sq.n || tl.kb.n <= sh.chunk) return;  // one split wrote the row itself
  const int splits = (tl.kb.n + sh.chunk - 1) / sh.chunk;
  const long long row = (static_cast<long long>(sq.row0) + i) * a.heads + head;
  float mm = -INFINITY;
  for (int k = tid; k < splits; k += 128) mm = fmaxf(mm, part_ml(a, sh.splits, k, row, D)->x);
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, w));
  if (lane == 0) s_red[warp] = mm;
  __syncthreads();
  mm = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
  const float base = mm == -INFINITY ? 0.0f : mm;
  float sum = 0.0f;
  for (int k = tid; k < splits; k += 128) {
    const float2 ml = *part_ml(a, sh.splits, k, row, D);
    const float c = kv_ex2(ml.x - base);
    s_c[k] = c;
    sum = fmaf(ml.y, c, sum);
  }
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
  if (lane == 0) s_red[4 + warp] = sum;
  __syncthreads();
  sum = (s_red[4] + s_red[5]) + (s_red[6] + s_red[7]);
  const int way = tid / LANES, d = tid % LANES;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
  for (int k = way; k < splits; k += WAYS) {
    const float4 v = *reinterpret_cast<const float4*>(part_o(a, k, row, D) + 4 * d);
    const float c = s_c[k];
    acc.x = fmaf(v.x, c, acc.x), acc.y = fmaf(v.y, c, acc.y), acc.z = fmaf(v.z, c, acc.z), acc.w = fmaf(v.w, c, acc.w);
  }
  s_acc[way][d] = acc;
  __syncthreads();
  bool bad = false;
  if (tid < LANES) {
#pragma unroll
    for (int w = 1; w < WAYS; ++w) {
      const float4 v = s_acc[w][d];
      acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    acc.x *= inv, acc.y *= inv, acc.z *= inv, acc.w *= inv;
    bad = (sum == 0.0f && sq.length - sq.n + i >= 0) || acc.x != acc.x || acc.y != acc.y || acc.z != acc.z || acc.w != acc.w;
  }
  const long long g = static_cast<long long>(sq.row0) + i;
  T* out = static_cast<T*>(a.out.p) + g * a.out.ld + head * a.out.hs;
  if (!__syncthreads_or(bad)) {
    if (tid < LANES) store4(out + 4 * d, acc, sh.vec_o);
  } else {  // q is still there where the output goes to its place
    kv_attend_row_cta<T, BITS, D>(a, blockIdx.y, sq.length - sq.n + i, head,
                                  static_cast<const T*>(a.q.p) + g * a.q.ld + head * a.q.hs, out, &s_acc[0][0].x, s_red);
  }
}

int rows_per_tile(const KvAttnArgs& a) {
  const long long rows = static_cast<long long>(a.st.max_new) * (a.heads / a.c.kv_heads);
  return rows <= 8 ? 8 : 16;
}

// 16-key sub-blocks of a step: a 4-bit cache takes 32 keys (64 at 64 dims) at a time, 5 KB of codes and scales in
// flight a warp; one page lookup for all of them where a page holds whole steps, else one each.
template <int BITS, int D>
constexpr int kSubs = BITS == 16 ? 1 : D == 64 ? 4 : 2;

int subs_of(const KvAttnArgs& a) { return a.c.bits == 16 ? 1 : a.c.dim == 64 ? 4 : 2; }
bool whole_steps(const KvAttnArgs& a) { return a.c.page_size % (16 * subs_of(a)) == 0; }

// The most blocks that a tile reads, and how they are split: enough CTAs for every SM to hold some twice over, of at
// least 128 keys a warp (a shorter loop is all latency; a call a little above that pays a second launch: 3 sequences of 350
// to 611 keys over 4 bits take 14 us, as a whole call of 16 bits 10), each split's partial result being a few rows of D
// floats against chunk blocks of cache.
SplitShape shape_of(const KvAttnArgs& a) {
  const long long group = a.heads / a.c.kv_heads, rpt = rows_per_tile(a);
  SplitShape sh{};
  sh.tiles = static_cast<int>((a.st.max_new * group + rpt - 1) / rpt);
  const int subs = whole_steps(a) ? subs_of(a) : 1, size = 16 * subs;  // of a block
  sh.shift = subs == 1 ? 4 : subs == 2 ? 5 : 6;
  const long long tokens = (rpt + group - 2) / group + 1;  // most tokens of a tile
  long long keys = a.st.max_length;
  // the sinks' last block, and the band's first and last, may be partial
  const long long reach = a.sinks + static_cast<long long>(a.window) + tokens + 2 * (size - 1);
  if (a.window > 0 && reach < keys) keys = reach;
  const long long blocks = (keys + size - 1) / size;
  const long long items = static_cast<long long>(sh.tiles) * a.c.kv_heads * a.st.sequences;
  const long long want = ((a.st.sequences == 1 ? kCtasOne : kCtasMany) + items - 1) / items;  // at most kMaxSplits
  long long chunk = (blocks + want - 1) / want;
  const long long least = 128 * kWarps / size;
  if (chunk < least) chunk = least;
  if (blocks <= chunk) chunk = blocks > 0 ? blocks : 1;
  sh.chunk = static_cast<int>(chunk);
  sh.splits = static_cast<int>((blocks + chunk - 1) / chunk);
  if (sh.splits < 1) sh.splits = 1;
  auto fits = [](const KvRows& r, int bytes) {
    return (reinterpret_cast<uintptr_t>(r.p) & (bytes - 1)) == 0 && r.ld * 2 % bytes == 0 && r.hs * 2 % bytes == 0;
  };
  sh.vec_q = fits(a.q, 16);
  sh.vec_o = fits(a.out, 8);
  sh.page = KvDiv(static_cast<unsigned>(a.c.page_size / size));
  return sh;
}

template <typename T, int BITS, int D, bool WHOLE>
void split(const KvAttnArgs& a, const SplitShape& sh, int rpt, dim3 grid, cudaStream_t s) {
  // (131,000 keys over 4 bits, 64 dims, pages of 16: 66 us by 32 keys, 85 by 64)
  constexpr int SUB = WHOLE ? kSubs<BITS, D> : 2;
  if (rpt == 8)
    kv_attention_split_kernel<T, BITS, D, 1, SUB, WHOLE><<<grid, 32 * kWarps, 0, s>>>(a, sh);
  else
    kv_attention_split_kernel<T, BITS, D, 2, SUB, WHOLE><<<grid, 32 * kWarps, 0, s>>>(a, sh);
}

template <typename T, int BITS, int D>
cudaError_t join(const KvAttnArgs& a, const SplitShape& sh, int rows_per_tile, cudaStream_t s) {
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(a.st.max_new) * a.heads, a.st.sequences);  // at most 2^30: checked at the entry
  cfg.blockDim = dim3(128);
  cfg.stream = s;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kv_combine_kernel<T, BITS, D>, a, sh, rows_per_tile);
}

template <typename T, int BITS, int D>
cudaError_t attend(const KvAttnArgs& a, cudaStream_t s) {
  const SplitShape sh = shape_of(a);
  const int rpt = rows_per_tile(a);
  const dim3 grid(sh.tiles * a.c.kv_heads, sh.splits, a.st.sequences);
  if (BITS == 16 || whole_steps(a))
    split<T, BITS, D, true>(a, sh, rpt, grid, s);
  else
    split<T, BITS, D, BITS == 16>(a, sh, rpt, grid, s);
  if (sh.splits > 1) return join<T, BITS, D>(a, sh, rpt, s);
  return cudaGetLastError();
}

}  // namespace

long long kv_attention_workspace(const KvAttnArgs& a) {
  if (a.st.sequences == 0 || a.st.max_new == 0) return 0;
  const long long splits = kv_attention_tc_ok(a) ? kv_tile_splits(a) : shape_of(a).splits;
  return splits > 1 ? kv_split_bytes(a, splits) : 0;
}

cudaError_t launch_kv_join(const KvAttnArgs& a, int shift, int chunk, int splits, int rows_per_tile, cudaStream_t s) {
  SplitShape sh = shape_of(a);
  sh.shift = shift;
  sh.chunk = chunk;
  sh.splits = splits;
  if (a.c.bits == 16) {
    if (a.c.dim == 64)
      return a.c.f16 ? join<__half, 16, 64>(a, sh, rows_per_tile, s) : join<__nv_bfloat16, 16, 64>(a, sh, rows_per_tile, s);
    return a.c.f16 ? join<__half, 16, 128>(a, sh, rows_per_tile, s) : join<__nv_bfloat16, 16, 128>(a, sh, rows_per_tile, s);
  }
  if (a.c.dim == 64)
    return a.c.f16 ? join<__half, 4, 64>(a, sh, rows_per_tile, s) : join<__nv_bfloat16, 4, 64>(a, sh, rows_per_tile, s);
  return a.c.f16 ? join<__half, 4, 128>(a, sh, rows_per_tile, s) : join<__nv_bfloat16, 4, 128>(a, sh, rows_per_tile, s);
}

cudaError_t launch_kv_attention(const KvAttnArgs& a, cudaStream_t s) {
  if (a.st.sequences == 0 || a.st.max_new == 0) return cudaSuccess;
  if (kv_attention_tc_ok(a)) return launch_kv_attention_tc(a, s);
  if (a.c.bits == 16) {
    if (a.c.dim == 64)
      return a.c.f16 ? attend<__half, 16, 64>(a, s) : attend<__nv_bfloat16, 16, 64>(a, s);
    return a.c.f16 ? attend<__half, 16, 128>(a, s) : attend<__nv_bfloat16, 16, 128>(a, s);
  }
  if (a.c.dim == 64) return a.c.f16 ? attend<__half, 4, 64>(a, s) : attend<__nv_bfloat16, 4, 64>(a, s);
  return a.c.f16 ? attend<__half, 4, 128>(a, s) : attend<__nv_bfloat16, 4, 128>(a, s);
}

}  // namespace jc
