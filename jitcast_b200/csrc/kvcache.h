// The paged key/value cache: what its kernels know of a cache, a step of a batch and the tensors around them.
//
// A pool row is one token's key (or value) of one kv head: pool row (page · kv_heads + head) · page_size + slot.
// 16 bits: D elements of the cache's type. 4 bits: D / 2 bytes (byte j: dim 2j low, 2j + 1 high) and D / 32
// half2 (scale, min) in a second pool; a code c stands for fp16(c · scale + min).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace jc {

constexpr int kKvGroup = 32;  // consecutive dims of a 4-bit row that share one (scale, min)

struct KvCache {
  int bits;       // 16 or 4
  int f16;        // 1: the tensors around the cache (and a 16-bit cache) are FP16, 0: BF16
  int pages, page_size, kv_heads, dim;
  void* k;
  void* v;
  void* k_scale;  // 4 bits: half2 [pool rows, dim / 32]
  void* v_scale;
};

// The sequences of one call. New token i of a sequence with n new tokens has index length − n + i in it.
struct KvStep {
  int sequences;
  int tokens;      // packed rows of the new tokens' tensors
  int max_new;     // most new tokens of a sequence
  int max_length;  // most cached tokens of a sequence
  const int* start;   // [sequences + 1] bounds of each sequence's rows, or null: sequence s has row s alone
  const int* length;  // [sequences]
  const int* table;   // [sequences, ld_table]: the sequence's pages in order
  int table_pages;    // columns of the table that may be read
  long long ld_table;
};

// Rows of heads: element (token, head, dim) at token · ld + head · hs + dim.
struct KvRows {
  void* p;
  long long ld, hs;
};

struct KvAppendArgs {
  KvCache c;
  KvStep st;
  KvRows q, k, v, q_out;  // q.p null: keys and values only
  int heads;              // q heads
  const int* positions;   // [tokens] rows of the rotation table, or null: the token's index
  const float* rope;      // [rope_rows, dim]: cos of pair e at e, its sin at dim / 2 + e; null: no rotation
  int rope_rows, pairs;   // pairs (e, e + dim / 2), e < pairs, rotate
  uint32_t* err;
};

struct KvReadArgs {
  KvCache c;
  KvStep st;
  KvRows k, v;
  uint32_t* err;
};

struct KvAttnArgs {
  KvCache c;
  KvStep st;
  KvRows q, out;
  int heads;
  int window;  // keys of the sliding window, the token's own included; 0: every key
  int sinks;   // first keys of a sequence that stay visible
  float scale;
  float* workspace;  // partial results of split key ranges (kv_attention_workspace bytes)
  uint32_t* err;
};

cudaError_t launch_kv_append(const KvAppendArgs& a, cudaStream_t s);
cudaError_t launch_kv_read(const KvReadArgs& a, cudaStream_t s);
cudaError_t launch_kv_attention(const KvAttnArgs& a, cudaStream_t s);

// The form on 128-row tcgen05 tiles (kv_attention_tc.cu), for the calls that take it.
bool kv_attention_tc_ok(const KvAttnArgs& a);
cudaError_t launch_kv_attention_tc(const KvAttnArgs& a, cudaStream_t s);

// Bytes of workspace that launch_kv_attention needs for this call (0: none); reads no pointer.
long long kv_attention_workspace(const KvAttnArgs& a);

}  // namespace jc
