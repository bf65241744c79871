// C-ABI entry points of the paged key/value cache: append (with the position rotation), attention of new tokens
// over it, and reading cached tokens back. Every argument that the host can see is checked before a launch; what
// only the GPU can see (starts, lengths, page ids, positions) is held to the call's bounds by the kernels. No C++ exception
// (an allocation of a message or a device's first use may throw) leaves an entry point.
#include <cmath>
#include <string>

#include "kvcache.h"
#include "runtime.h"

using namespace jc;

namespace {

// Sets the device of a call and puts the caller's back.
struct DeviceScope {
  int prev = -1;
  bool ok;
  explicit DeviceScope(int device) {
    if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
    ok = prev == device || cudaSetDevice(device) == cudaSuccess;
    if (prev == device) prev = -1;
  }
  ~DeviceScope() {
    if (prev >= 0) cudaSetDevice(prev);
  }
};

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

jc_status check_cache(jc_precision precision, const jc_kv_cache* c, KvCache* out) {
  if (!c) return fail(JC_ERR_INVALID_ARG, "null cache");
  if (precision != JC_BF16 && precision != JC_FP16)
    return fail(JC_ERR_INVALID_ARG, "a key/value cache takes JC_BF16 or JC_FP16");
  if (c->bits != 16 && c->bits != 4) return fail(JC_ERR_INVALID_ARG, "cache bits must be 16 or 4");
  if (c->pages < 1 || c->kv_heads < 1) return fail(JC_ERR_INVALID_ARG, "cache pages and kv_heads must be >= 1");
  if (c->head_dim != 64 && c->head_dim != 128)
    return fail(JC_ERR_UNSUPPORTED_SHAPE, "cache head_dim must be 64 or 128");
  if (c->page_size < 16 || c->page_size % 16 != 0)
    return fail(JC_ERR_UNSUPPORTED_SHAPE, "cache page_size must be a multiple of 16");
  const long long rows = static_cast<long long>(c->pages) * c->kv_heads;
  if (rows > 2147483647LL / c->page_size) return fail(JC_ERR_UNSUPPORTED_SHAPE, "cache above 2^31 - 1 pool rows");
  if (!c->k || !c->v) return fail(JC_ERR_INVALID_ARG, "null cache pool");
  if (!aligned(c->k, 16) || !aligned(c->v, 16)) return fail(JC_ERR_INVALID_ARG, "cache pools not 16-byte aligned");
  if (c->bits == 4) {
    if (!c->k_scale || !c->v_scale) return fail(JC_ERR_INVALID_ARG, "a 4-bit cache needs scale pools");
    if (!aligned(c->k_scale, 16) || !aligned(c->v_scale, 16))
      return fail(JC_ERR_INVALID_ARG, "cache scale pools not 16-byte aligned");
  }
  *out = KvCache{c->bits,     precision == JC_FP16 ? 1 : 0, c->pages, c->page_size, c->kv_heads, c->head_dim, c->k, c->v,
                 c->k_scale, c->v_scale};
  return JC_OK;
}

jc_status check_step(const jc_kv_step* s, KvStep* out) {
  if (!s) return fail(JC_ERR_INVALID_ARG, "null step");
  if (s->sequences < 0 || s->tokens < 0 || s->max_new < 0 || s->max_length < 0 || s->table_pages < 0)
    return fail(JC_ERR_INVALID_ARG, "negative step size");
  if (s->sequences > 65535) return fail(JC_ERR_UNSUPPORTED_SHAPE, "at most 65535 sequences in a step");
  if (s->ld_table < s->table_pages) return fail(JC_ERR_INVALID_ARG, "page table pitch below its pages");
  if (!s->start && s->sequences > 0 && (s->tokens != s->sequences || s->max_new != 1))
    return fail(JC_ERR_INVALID_ARG, "a step without starts has one new token per sequence");
  if (s->sequences > 0 && (!s->length || (s->table_pages > 0 && !s->page_table)))
    return fail(JC_ERR_INVALID_ARG, "null length or page table");
  // no sequence has more new tokens than there are rows: a looser bound shapes no launch and sizes no workspace
  const int max_new = s->max_new < s->tokens ? s->max_new : s->tokens;
  *out = KvStep{s->sequences, s->tokens, max_new, s->max_length, s->start, s->length, s->page_table, s->table_pages,
                s->ld_table};
  return JC_OK;
}

jc_status check_rows(const jc_kv_rows* r, const char* name, int dim, int heads, KvRows* out) {
  const std::string n = name;
  if (!r || !r->data) return fail(JC_ERR_INVALID_ARG, "null " + n);
  if (!aligned(r->data, 2)) return fail(JC_ERR_INVALID_ARG, n + " not 2-byte aligned");
  if ((heads > 1 && r->head_stride < dim) || r->ld < 0) return fail(JC_ERR_INVALID_ARG, n + " strides overlap its heads");
  *out = KvRows{r->data, r->ld, r->head_stride};
  return JC_OK;
}

// Rows that a call writes: no two tokens or heads may share an element. Either a token's heads lie within its pitch, or a
// head's tokens do (heads before tokens).
jc_status check_out(const jc_kv_rows* r, const char* name, int dim, int heads, int tokens, KvRows* out) {
  if (jc_status st = check_rows(r, name, dim, heads, out)) return st;
  if (tokens < 2) return JC_OK;
  // n rows of `dim` elements, `inner` apart, fit into `pitch`
  auto within = [dim](long long pitch, int n, long long inner) {
    return pitch >= dim && (n < 2 || inner <= (pitch - dim) / (n - 1));
  };
  if (within(r->ld, heads, r->head_stride) || (r->ld >= dim && within(r->head_stride, tokens, r->ld))) return JC_OK;
  return fail(JC_ERR_INVALID_ARG, std::string(name) + " rows overlap");
}

jc_status check_attention(jc_precision precision, const jc_kv_cache* cache, const jc_kv_step* step, int heads,
                          int window, int sinks, KvAttnArgs* a) {
  if (jc_status st = check_cache(precision, cache, &a->c)) return st;
  if (jc_status st = check_step(step, &a->st)) return st;
  if (heads < 1 || heads % a->c.kv_heads != 0) return fail(JC_ERR_INVALID_ARG, "heads must be a multiple of kv_heads");
  if (heads > 65535) return fail(JC_ERR_UNSUPPORTED_SHAPE, "at most 65535 heads");
  if (static_cast<long long>(a->st.max_new) * heads > (1 << 30))
    return fail(JC_ERR_UNSUPPORTED_SHAPE, "above 2^30 query rows of a sequence");
  if (window < 0 || sinks < 0) return fail(JC_ERR_INVALID_ARG, "window and sinks must be >= 0");
  a->heads = heads;
  a->window = window;
  a->sinks = sinks;
  return JC_OK;
}

}  // namespace

extern "C" {

jc_status jc_kv_append_device(int device, jc_precision precision, const jc_kv_cache* cache, const jc_kv_step* step,
                              const jc_kv_rows* k, const jc_kv_rows* v, const jc_kv_rows* q, int heads,
                              const jc_kv_rows* q_out, const int32_t* positions, const float* rope_table,
                              int rope_rows, int rope_pairs, void* stream) try {
  clear_error();
  KvAppendArgs a{};
  if (jc_status st = check_cache(precision, cache, &a.c)) return st;
  if (jc_status st = check_step(step, &a.st)) return st;
  if (a.st.tokens > 0) {
    if (jc_status st = check_rows(k, "k", a.c.dim, a.c.kv_heads, &a.k)) return st;
    if (jc_status st = check_rows(v, "v", a.c.dim, a.c.kv_heads, &a.v)) return st;
    if (q) {
      if (heads < 1) return fail(JC_ERR_INVALID_ARG, "heads must be >= 1 with q");
      if (jc_status st = check_rows(q, "q", a.c.dim, heads, &a.q)) return st;
      if (jc_status st = check_out(q_out, "q_out", a.c.dim, heads, a.st.tokens, &a.q_out)) return st;
      a.heads = heads;
    }
  }
  if (rope_table) {
    if (rope_pairs < 0 || rope_pairs > a.c.dim / 2)
      return fail(JC_ERR_INVALID_ARG, "rope_pairs must be in [0, head_dim / 2]");
    if (rope_rows < 1) return fail(JC_ERR_INVALID_ARG, "rope_rows must be >= 1");
  }
  a.positions = positions;
  a.rope = rope_table;
  a.rope_rows = rope_rows;
  a.pairs = rope_table ? rope_pairs : 0;
  std::string why;
  DeviceRt* rt = device_rt(device, &why);
  if (!rt) return fail(JC_ERR_NO_DEVICE, why);
  DeviceScope dev(device);
  if (!dev.ok) return fail(JC_ERR_CUDA, "cannot select the device");
  a.err = rt->kv_err;
  const cudaError_t e = launch_kv_append(a, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? JC_OK : fail_cuda(e, "cache append launch");
} catch (...) {
  return JC_ERR_INTERNAL;
}

jc_status jc_kv_attention_workspace(jc_precision precision, const jc_kv_cache* cache, const jc_kv_step* step,
                                    int heads, int window, int sinks, long long* bytes) try {
  clear_error();
  if (!bytes) return fail(JC_ERR_INVALID_ARG, "null bytes");
  KvAttnArgs a{};
  if (jc_status st = check_attention(precision, cache, step, heads, window, sinks, &a)) return st;
  *bytes = kv_attention_workspace(a);
  return JC_OK;
} catch (...) {
  return JC_ERR_INTERNAL;
}

jc_status jc_kv_attention_device(int device, jc_precision precision, const jc_kv_cache* cache, const jc_kv_step* step,
                                 const jc_kv_rows* q, int heads, const jc_kv_rows* out, int window, int sinks,
                                 float scale, void* workspace, long long workspace_bytes, void* stream) try {
  clear_error();
  KvAttnArgs a{};
  if (jc_status st = check_attention(precision, cache, step, heads, window, sinks, &a)) return st;
  if (!(scale > 0.0f) || !std::isfinite(scale)) return fail(JC_ERR_INVALID_ARG, "scale must be positive and finite");
  if (a.st.tokens > 0) {
    if (jc_status st = check_rows(q, "q", a.c.dim, heads, &a.q)) return st;
    if (jc_status st = check_out(out, "out", a.c.dim, heads, a.st.tokens, &a.out)) return st;
  }
  const long long need = kv_attention_workspace(a);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(JC_ERR_INVALID_ARG, "workspace of " + std::to_string(workspace ? workspace_bytes : 0) +
                                        " bytes, the call needs " + std::to_string(need));
  if (need > 0 && !aligned(workspace, 16)) return fail(JC_ERR_INVALID_ARG, "workspace not 16-byte aligned");
  a.scale = scale;
  a.workspace = static_cast<float*>(workspace);
  std::string why;
  DeviceRt* rt = device_rt(device, &why);
  if (!rt) return fail(JC_ERR_NO_DEVICE, why);
  DeviceScope dev(device);
  if (!dev.ok) return fail(JC_ERR_CUDA, "cannot select the device");
  a.err = rt->kv_err;
  const cudaError_t e = launch_kv_attention(a, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? JC_OK : fail_cuda(e, "cache attention launch");
} catch (...) {
  return JC_ERR_INTERNAL;
}

jc_status jc_kv_read_device(int device, jc_precision precision, const jc_kv_cache* cache, const jc_kv_step* step,
                            const jc_kv_rows* k, const jc_kv_rows* v, void* stream) try {
  clear_error();
  KvReadArgs a{};
  if (jc_status st = check_cache(precision, cache, &a.c)) return st;
  if (jc_status st = check_step(step, &a.st)) return st;
  if (a.st.tokens > 0) {
    if (jc_status st = check_out(k, "k", a.c.dim, a.c.kv_heads, a.st.tokens, &a.k)) return st;
    if (jc_status st = check_out(v, "v", a.c.dim, a.c.kv_heads, a.st.tokens, &a.v)) return st;
  }
  std::string why;
  DeviceRt* rt = device_rt(device, &why);
  if (!rt) return fail(JC_ERR_NO_DEVICE, why);
  DeviceScope dev(device);
  if (!dev.ok) return fail(JC_ERR_CUDA, "cannot select the device");
  a.err = rt->kv_err;
  const cudaError_t e = launch_kv_read(a, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? JC_OK : fail_cuda(e, "cache read launch");
} catch (...) {
  return JC_ERR_INTERNAL;
}

}  // extern "C"
