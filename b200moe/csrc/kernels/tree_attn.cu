// Attention of the nodes of drafted trees over the paged pool.
//
//   o_i = sum_j p_ij v_j,   p_ij = softmax_j(scale * q_i . k_j)
//
// where j runs over the committed prefix [0, P) of node i's sequence and over node i
// and its ancestors, whose keys sit at positions P + node.
//
// The general form, for what the tensor-core form (tree_attn_tc.cu) does not take, block sizes
// other than 8, 16, 32 and multiples of 64 and more than 128 query heads on a KV head: one warp per (node, query head), a lane scores one key of 32, the warp keeps the
// running maximum and sum in fp32, and each lane accumulates D / 32 columns of o.  It is bound
// by instructions (16 trees of 16 nodes at 1152 context: 4.9 ms with blocks of 48 or 96, 25 us with 64).
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <stdexcept>
#include <string>

#include "pdl.cuh"
#include "sm100.cuh"
#include "tree.h"

namespace b200 {
namespace {

using bf16 = __nv_bfloat16;

constexpr int kWarps = 4;

// Element d of a stored row as the float it stands for.
template <int MODE>
__device__ __forceinline__ float kv_value(const TreeAttnArgs& a, const void* pool, const void* side, int kv, int64_t blk,
                                          int h, int y, int d, float row_scale) {
  const int64_t at = blk * a.block_stride + ((int64_t)h * a.block_size + y) * a.head_dim + d;
  if (MODE == 0) return __bfloat162float(static_cast<const bf16*>(pool)[at]);
  const float q = (float)static_cast<const int8_t*>(pool)[at];
  if (MODE == 1) return q * row_scale;
  const int n_out = a.ch.n_out[h];
  for (int o = 0; o < n_out; ++o)
    if (a.ch.out_idx[h * kKvNoutMax + o] == d)
      return __bfloat162float(static_cast<const bf16*>(side)[blk * a.ch.side_block_stride +
                                                             ((int64_t)h * a.block_size + y) * kKvNoutMax + o]);
  // the channel mode's values are bf16 by definition, as its other readers round them
  return __bfloat162float(__float2bfloat16(q * a.ch.dscale[((int64_t)kv * a.num_kv_heads + h) * a.head_dim + d]));
}

__device__ __forceinline__ bool usable(const TreeAttnArgs& a, int b) {
  const int q0 = a.cu_seqlens_q[b], q1 = a.cu_seqlens_q[b + 1], len = a.seq_lens[b];
  return tree_fits(q0, q1, a.rows, a.max_q_len, len) && (q0 == q1 || len <= (int64_t)a.max_blocks * a.block_size);
}

// Whether row is a node of sequence b.
__device__ __forceinline__ bool holds(const TreeAttnArgs& a, int b, int row) {
  return a.cu_seqlens_q[b] <= row && row < a.cu_seqlens_q[b + 1] && usable(a, b);
}

template <int D, int MODE>
__global__ void __launch_bounds__(kWarps * 32) tree_attn_kernel(const TreeAttnArgs a) {
  pdl_enter();
  __shared__ int s_par[kTreeMaxNodes];
  __shared__ float s_q[kWarps][D];
  __shared__ int s_found;
  const int row = blockIdx.x, h = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (row == 0 && h == 0)      // report the trees that do not fit
    for (int i = threadIdx.x; i < a.batch; i += kWarps * 32)
      if (!usable(a, i)) record_status(a.status, kStatusBadShape);
  // the sequence that holds this row: last b with cu[b] <= row
  int b = 0, hi = a.batch;
  while (hi - b > 1) {
    const int mid = (b + hi) >> 1;
    if (a.cu_seqlens_q[mid] <= row) b = mid; else hi = mid;
  }
  if (!holds(a, b, row)) {     // none, or offsets of a bad tree led the search astray
    if (threadIdx.x == 0) s_found = a.batch;
    __syncthreads();
    for (int i = threadIdx.x; i < a.batch; i += kWarps * 32)
      if (holds(a, i, row)) atomicMin(&s_found, i);
    __syncthreads();
    b = s_found;
    if (b == a.batch) return;  // rows of bad trees and behind the last sequence
  }
  const int q0 = a.cu_seqlens_q[b], q1 = a.cu_seqlens_q[b + 1], len = a.seq_lens[b];
  const int n = q1 - q0, node = row - q0, prefix = len - n;
  for (int i = threadIdx.x; i < n; i += kWarps * 32) s_par[i] = a.parents[q0 + i];
  __syncthreads();
  const int* tab = a.block_tables + b * a.table_stride;
  const float sl2 = a.scale * 1.4426950408889634f;
  bool bad = false;
  for (int g = warp; g < a.group; g += kWarps) {
    const int64_t qrow = ((int64_t)row * a.num_kv_heads * a.group + h * a.group + g) * D;
    for (int d = lane; d < D; d += 32) s_q[warp][d] = __bfloat162float(static_cast<const bf16*>(a.q)[qrow + d]);
    __syncwarp();
    float m = -INFINITY, l = 0.f, o[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) o[i] = 0.f;
    bool any = false;    // a key has been read
    for (int k0 = 0; k0 < len; k0 += 32) {
      const int key = k0 + lane;
      bool see = key < prefix;
      if (!see && key < len) {
        for (int at = node; at >= 0;) {  // this node's ancestors; a parent behind its child ends the walk
          if (at == key - prefix) { see = true; break; }
          const int up = s_par[at];
          at = up < at ? up : -1;
        }
      }
      int64_t blk = 0;
      const int bi = key / a.block_size, y = key % a.block_size;
      if (see) {
        blk = tab[bi];
        if (blk < 0 || blk >= a.num_blocks) { bad = true; see = false; blk = 0; }
      }
      float ks = 1.f, vs = 1.f;
      if (MODE == 1 && see) {
        const int64_t at = blk * a.scale_block_stride + (int64_t)h * a.block_size + y;
        ks = a.k_scale[at];
        vs = a.v_scale[at];
      }
      float s = -INFINITY;
      if (see) {
        s = 0.f;
        for (int d = 0; d < D; ++d)
          s = fmaf(s_q[warp][d], kv_value<MODE>(a, a.k_cache, a.ch.side_k, 0, blk, h, y, d, ks), s);
        s *= sl2;
      }
      if (!__any_sync(0xffffffffu, see)) continue;
      any = true;
      // The maximum passes over NaN.  While no score is above -inf, 0 stands for it: a -inf weighs
      // nothing, a NaN makes the sum NaN.
      const float mn = fmaxf(m, warp_max(s));
      const float base = mn == -INFINITY ? 0.f : mn;
      const float alpha = exp2f(m - base);  // m = -inf: 0
      const float p = see ? exp2f(s - base) : 0.f;
      m = mn;
      l = l * alpha + warp_sum(p);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) o[i] *= alpha;
      for (int j = 0; j < 32; ++j) {
        const float pj = __shfl_sync(0xffffffffu, p, j);
        const bool sj = __shfl_sync(0xffffffffu, see, j);
        const int64_t bj = __shfl_sync(0xffffffffu, blk, j);
        const float vj = __shfl_sync(0xffffffffu, vs, j);
        if (!sj) continue;
        const int yj = (k0 + j) % a.block_size;
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
          o[i] = fmaf(pj, kv_value<MODE>(a, a.v_cache, a.ch.side_v, 1, bj, h, yj, i * 32 + lane, vj), o[i]);
      }
    }
    // every score -inf: no softmax, NaN; every block id outside the pool: zeros
    const float inv = any ? 1.f / l : 0.f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
      static_cast<bf16*>(a.out)[qrow + i * 32 + lane] = __float2bfloat16(o[i] * inv);
    __syncwarp();
  }
  if (bad) record_status(a.status, kStatusBadShape);
  pdl_trigger();
}

template <int D>
void launch(const TreeAttnArgs& a, cudaStream_t s) {
  const dim3 grid(a.rows, a.num_kv_heads);
  if (a.kv_int8 == 0) pdl_launch(tree_attn_kernel<D, 0>, grid, kWarps * 32, 0, s, a);
  else if (a.kv_int8 == 1) pdl_launch(tree_attn_kernel<D, 1>, grid, kWarps * 32, 0, s, a);
  else pdl_launch(tree_attn_kernel<D, 2>, grid, kWarps * 32, 0, s, a);
}

}  // namespace

int tree_attn(const TreeAttnArgs& a, cudaStream_t s) {
  if (a.rows == 0 || a.batch == 0) return 0;
  if (a.head_dim == 128) launch<128>(a, s);
  else launch<64>(a, s);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) throw std::runtime_error(std::string("tree_attn: ") + cudaGetErrorString(e));
  return 1;
}

}  // namespace b200
