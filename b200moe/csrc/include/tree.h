// Host interface of the draft-tree operators: attention of a tree's nodes over the
// paged pool (kernels/tree_attn.cu) and the commit of its accepted path
// (kernels/tree_commit.cu).
#pragma once
#include <cuda_runtime.h>
#include <cstdint>

#include "attention.h"

namespace b200 {

constexpr int kTreeMaxNodes = 256;   // nodes of one tree

#ifdef __CUDACC__
// Whether a sequence's nodes [q0, q1) lie in the rows and its keys hold them.  Compared, not subtracted,
// until the offsets are known to be in range: a difference of two of them may wrap to a small number.
__device__ __forceinline__ bool tree_fits(int q0, int q1, int rows, int max_q_len, int len) {
  return q0 >= 0 && q0 <= q1 && q1 <= rows && q1 - q0 <= max_q_len && (q0 == q1 || len >= q1 - q0);
}
#endif

struct TreeAttnArgs {
  const void* q;             // [rows, q_heads, D] bf16
  const void* k_cache;       // layer base of the pool, [blocks, kv_heads, block_size, D]
  const void* v_cache;
  const float* k_scale;      // kv_int8 == 1: [blocks, kv_heads, block_size] (strided over blocks)
  const float* v_scale;
  int kv_int8;               // 0 bf16, 1 int8 per-token scales, 2 int8 channel mode (ch)
  KvChannel ch;
  const int* cu_seqlens_q;   // [batch + 1] first node of each sequence
  const int* seq_lens;       // [batch] keys: committed prefix + nodes
  const int* block_tables;   // [batch, max_blocks], rows table_stride apart
  int64_t table_stride;
  const int* parents;        // [rows] place of a node's parent in its tree, -1: none
  int batch;
  int rows;
  int max_q_len;             // no tree has more nodes (<= kTreeMaxNodes)
  int max_blocks;
  int num_blocks;
  int block_size;
  int64_t block_stride;      // elements between consecutive blocks of one layer
  int64_t scale_block_stride;
  int num_kv_heads;
  int group;                 // q heads per kv head
  int head_dim;
  float scale;
  void* out;                 // [rows, q_heads, D] bf16
  int* status;               // device status word
};
// The forms return the number of kernels that they launched.
int tree_attn(const TreeAttnArgs& a, cudaStream_t s);

// Tensor-core form (kernels/tree_attn_tc.cu): head_dim 64 or 128, blocks that hold whole
// tiles of 64 keys or divide one in multiples of 8 rows.
constexpr int kTreeTcBatch = 1024;   // sequences of one launch
struct TreeAttnTcPlan {
  int sub_rows;              // key rows of one TMA box
  int part_rows;             // rows of one partial result
  int grid;
  int64_t workspace_bytes;
  void* workspace;           // 16-byte aligned
  const float* key_scales;   // staged int8 values: [batch][kv_heads][k | v][key_stride], else null
  int key_stride;            // a multiple of 64
};
// False where the shape is not the tensor-core kernel's.
bool tree_attn_tc_plan(const TreeAttnArgs& a, int max_q_len, TreeAttnTcPlan* p);
int tree_attn_tc(const TreeAttnArgs& a, const TreeAttnTcPlan& p, cudaStream_t s);

// int8 pools (kernels/tree_stage.cu): the keys and values of up to `seqs` sequences at a time go
// to a bf16 stage that the tensor-core form reads.
int64_t tree_stage_bytes(const TreeAttnArgs& a, int seqs);
int tree_attn_staged(const TreeAttnArgs& a, const TreeAttnTcPlan& p, int seqs, void* stage, cudaStream_t s);

// One kind of rows the commit moves: [blocks, planes, block_size, row_bytes], contiguous.
struct TreeRows {
  uint8_t* base;
  int row_bytes;
};
struct TreeCommitArgs {
  TreeRows rows[3];          // payload, int8 scales, channel-mode side values
  int kinds;
  int planes;                // layers * 2 * kv_heads
  int block_size;
  int num_blocks;
  const int* cu_seqlens_q;   // [batch + 1]
  const int* seq_lens;       // [batch] committed prefix + nodes
  const int* block_tables;   // [batch, max_blocks], rows table_stride apart
  int64_t table_stride;
  const int* parents;        // [nodes]
  const int* draft;          // [nodes] drafted token of each node
  const int* target;         // [nodes] token the model picks behind each node
  int batch;
  int nodes;                 // entries of parents / draft / target
  int max_blocks;
  int max_q_len;             // row length of path / tokens
  int* accepted;             // [batch]
  int* path;                 // [batch, max_q_len], -1 behind the path
  int* tokens;               // [batch, max_q_len], -1 behind the path
  int* status;
};
// Returns the number of kernels that it launched.
int tree_commit(const TreeCommitArgs& a, cudaStream_t s);

}  // namespace b200
