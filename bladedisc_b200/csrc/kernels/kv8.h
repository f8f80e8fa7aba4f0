// Paged key / value cache held in 8 bits: block tables and slot maps, the append
// (rotary embedding + quantization), reading blocks back, and attention over it.
//
// One layer of the cache is four tensors:
//   k, v               int8  [num_blocks, kv_heads, block_size, dim]   levels
//   k_scale, v_scale   float [num_blocks, kv_heads]                     value = level * scale
// Token p of request r lives in block table[r][p / block_size] at offset p % block_size;
// its slot is block * block_size + offset.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace disc_b200 {

enum KvElemType : int { kKvF16 = 1, kKvBF16 = 2 };  // DISC_B200_F16 / DISC_B200_BF16

constexpr int kKv8DirectKeys = 512;   // caches up to this long take one CTA per item and no workspace
constexpr int kKvMaxRequests = 8192;  // per-request bookkeeping of the table kernels lives in shared memory

struct KvBlocksParams {
  const int32_t* tokens;  // [requests] extend: new tokens asked for; trim: tokens to keep
  int32_t* lens;          // [requests] cached tokens, updated
  int32_t* table;         // [requests, table_width], updated
  int32_t* free_list;     // [num_blocks] stack of free blocks
  int32_t* free_count;    // [1], updated
  int32_t requests, table_width, num_blocks, block_size;
  // extend only
  int32_t max_tokens;     // entries of slots and positions
  int32_t* slots;
  int32_t* positions;
  int32_t* q_start;       // [requests + 1]
  int32_t* q_lens;        // [requests]
  int32_t* kv_lens;       // [requests]
};
cudaError_t kv_blocks_extend_launch(const KvBlocksParams& p, cudaStream_t stream, const char** err);
cudaError_t kv_blocks_trim_launch(const KvBlocksParams& p, cudaStream_t stream, const char** err);

struct Kv8Cache {
  int8_t* k;
  int8_t* v;
  float* k_scale;
  float* v_scale;
  int32_t num_blocks, kv_heads, block_size, dim;
};

struct Kv8AppendParams {
  const void* qkv;         // [tokens, (q_heads + 2 * kv_heads) * dim], row stride ld_qkv
  int64_t tokens, ld_qkv;
  int32_t q_heads;         // may be 0
  void* q_out;             // [tokens, q_heads, dim] rotated, dense; only with cos
  const int32_t* slots;    // [tokens], -1 = not stored
  const int32_t* positions;  // [tokens]; only with cos
  const float* cos_table;  // [positions, dim / 2] or null: no rotation
  const float* sin_table;
  int32_t table_rows;      // rows of cos / sin
  int32_t type;
  Kv8Cache cache;
};
cudaError_t kv8_append_launch(const Kv8AppendParams& p, cudaStream_t stream, const char** err);

struct Kv8ReadParams {
  Kv8Cache cache;
  const int32_t* blocks;   // [count]
  int32_t count;
  void* k_out;             // [count, kv_heads, block_size, dim]
  void* v_out;
  int32_t type;
};
cudaError_t kv8_read_launch(const Kv8ReadParams& p, cudaStream_t stream, const char** err);

struct Kv8AttentionParams {
  const void* q;           // [tokens, q_heads, dim], token stride ld_q, heads dense
  void* out;               // the same shape, token stride ld_out
  int64_t tokens, ld_q, ld_out;
  int32_t q_heads;
  Kv8Cache cache;
  const int32_t* table;    // [requests, table_width]
  const int32_t* q_start;  // [requests] first token row of each request
  const int32_t* q_lens;   // [requests]
  const int32_t* kv_lens;  // [requests]
  int32_t requests, table_width;
  int32_t max_q, max_kv;   // the host's bounds on q_lens and kv_lens
  float scale;
  int32_t type;
  void* workspace;         // kv8_attention_workspace_bytes, 16-byte aligned
  int64_t workspace_bytes;
};
// Device memory that a call on the current device needs, from its sizes alone; none for short caches.
int64_t kv8_attention_workspace_bytes(const Kv8AttentionParams& p);
cudaError_t kv8_attention_launch(const Kv8AttentionParams& p, cudaStream_t stream, const char** err);
int kv8_status_fetch_and_clear();

// Host-side check of one layer's cache description; null when it is fine.
const char* kv8_cache_problem(const Kv8Cache& c);

}  // namespace disc_b200
