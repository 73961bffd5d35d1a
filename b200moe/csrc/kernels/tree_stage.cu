// int8 pools for the tensor-core tree attention: one launch brings the blocks of a slice of
// sequences to a bf16 stage that the tensor-core kernel reads by the stage's own block table.
//
// Token mode (k = s_k q8, one factor per key and head): the stage holds the int8 values, which
// bf16 holds exactly, and the factors apply in fp32 to the scores and to P, so no value is
// rounded that the pool does not round.  Channel mode: the stage holds bf16(q8 * dscale), or
// the side value at an outlier dimension, which is what that mode's values are.
//
// Bound by memory: 1 byte read and 2 written per value.  16 sequences of 8208 keys (134 MB of int8) take
// about 100 us, and the attention of the stage 70 us; at 1168 keys 17 + 28 us.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <stdexcept>
#include <string>

#include "pdl.cuh"
#include "sm100.cuh"
#include "tree.h"

namespace b200 {
namespace {

using bf16 = __nv_bfloat16;

constexpr int kThreads = 256, kPer = 4;               // chunks of 16 values a thread has in flight
constexpr int kPiece = kThreads * kPer;               // chunks of one piece of work
// CTAs launched for each SM.  A CTA has a piece of a block (16 KB) at a time; with 8, sequences that hold a few
// pieces more than they have CTAs take twice as long (1168 keys 45.7 us instead of 44.9, 8208 keys 176 instead of 170).
constexpr int kCtasPerSm = 32;

struct Stage {
  bf16* kv;          // [seqs * max_blocks][k | v][kv_heads][block_size][D]
  float* scales;     // [seqs][kv_heads][k | v][key_stride]
  int* tables;       // [seqs][max_blocks]: a block's place in the stage
  int key_stride;
};

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

// 32 bytes in one store: two of 16 would each write half of every sector
__device__ __forceinline__ void st32(void* p, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
               ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// Four int8 values as fp32: a biased byte in the low mantissa bits of 2^23, minus 2^23 + 128.
__device__ __forceinline__ void four(uint32_t w, float* f) {
  w ^= 0x80808080u;
#pragma unroll
  for (int e = 0; e < 4; ++e) f[e] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 + e)) - 8388736.f;
}

template <int D, bool CHAN>
__global__ void __launch_bounds__(kThreads) tree_stage_kernel(const TreeAttnArgs a, const Stage o) {
  const int b = blockIdx.y, bs = a.block_size, nkv = a.num_kv_heads;
  const int q0 = a.cu_seqlens_q[b], q1 = a.cu_seqlens_q[b + 1], len = a.seq_lens[b];
  // (a tree that does not fit is left out and reported by the attention)
  if (q0 == q1 || !tree_fits(q0, q1, a.rows, a.max_q_len, len) || len > (int64_t)a.max_blocks * bs) return;
  const int nb = (len + bs - 1) / bs;
  const int64_t plane = (int64_t)nkv * bs * D;
  const int chunks = (int)(plane / 16), pieces = (chunks + kPiece - 1) / kPiece;
  const int64_t items = (int64_t)nb * 2 * pieces;
  for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
    const int piece = (int)(it % pieces), kv = (int)(it / pieces) & 1, j = (int)(it / pieces / 2);
    const int id = a.block_tables[b * a.table_stride + j];
    const bool ok = id >= 0 && id < a.num_blocks;
    const int64_t slot = (int64_t)b * a.max_blocks + j;
    const uint4* src = reinterpret_cast<const uint4*>(static_cast<const int8_t*>(kv ? a.v_cache : a.k_cache) +
                                                      (ok ? id : 0) * a.block_stride);
    uint4* dst = reinterpret_cast<uint4*>(o.kv + (slot * 2 + kv) * plane);
    uint4 raw[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int c = piece * kPiece + i * kThreads + threadIdx.x;
      raw[i] = make_uint4(0, 0, 0, 0);
      if (ok && c < chunks) raw[i] = __ldg(src + c);
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int c = piece * kPiece + i * kThreads + threadIdx.x;
      if (c >= chunks) continue;
      const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
      float f[16];
#pragma unroll
      for (int e = 0; e < 4; ++e) four(w[e], f + 4 * e);
      uint32_t out[8];
      if constexpr (CHAN) {
        const int y = c / (D / 16), h = y / bs, d0 = c % (D / 16) * 16;
        const float4* ds = reinterpret_cast<const float4*>(a.ch.dscale + ((int64_t)kv * nkv + h) * D + d0);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float4 s = __ldg(ds + e);
          f[4 * e] *= s.x;
          f[4 * e + 1] *= s.y;
          f[4 * e + 2] *= s.z;
          f[4 * e + 3] *= s.w;
        }
        const bf16* side = static_cast<const bf16*>(kv ? a.ch.side_v : a.ch.side_k) + (ok ? id : 0) * a.ch.side_block_stride +
                           (int64_t)y * kKvNoutMax;
        const int n_out = ok ? min(a.ch.n_out[h], kKvNoutMax) : 0;
        for (int k = 0; k < n_out; ++k) {
          const int d = a.ch.out_idx[h * kKvNoutMax + k] - d0;
          if (d < 0 || d >= 16) continue;
          const float x = __bfloat162float(side[k]);
#pragma unroll
          for (int e = 0; e < 16; ++e) f[e] = d == e ? x : f[e];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) out[e] = pack2(f[2 * e], f[2 * e + 1]);
      } else {
        // at most eight significant bits: the upper half of an fp32 is the bf16
#pragma unroll
        for (int e = 0; e < 8; ++e) out[e] = __byte_perm(__float_as_uint(f[2 * e]), __float_as_uint(f[2 * e + 1]), 0x7632);
      }
      st32(dst + 2 * c, out);
    }
    if (piece > 0) continue;
    if (threadIdx.x == 0 && kv == 0) {
      o.tables[slot] = (int)slot;
      if (!ok) record_status(a.status, kStatusBadShape);
    }
    if constexpr (!CHAN) {
      // the factors, zero behind the sequence up to the end of its last key tile
      const int rows = j == nb - 1 ? max(bs, ((len + 63) & ~63) - j * bs) : bs;
      const float* sc = (kv ? a.v_scale : a.k_scale) + (ok ? id : 0) * a.scale_block_stride;
      for (int i = threadIdx.x; i < nkv * rows; i += kThreads) {
        const int h = i / rows, y = i % rows, key = j * bs + y;
        o.scales[(((int64_t)b * nkv + h) * 2 + kv) * o.key_stride + key] = ok && key < len ? sc[h * bs + y] : 0.f;
      }
    }
  }
}

int key_stride(const TreeAttnArgs& a) { return (int)(((int64_t)a.max_blocks * a.block_size + 63) / 64 * 64); }

int64_t round16(int64_t n) { return (n + 15) / 16 * 16; }

}  // namespace

int64_t tree_stage_bytes(const TreeAttnArgs& a, int seqs) {
  const int64_t blocks = (int64_t)seqs * a.max_blocks;
  return blocks * 4 * a.num_kv_heads * a.block_size * a.head_dim +
         (int64_t)seqs * a.num_kv_heads * 2 * key_stride(a) * 4 + round16(blocks * 4);
}

int tree_attn_staged(const TreeAttnArgs& a, const TreeAttnTcPlan& p, int seqs, void* stage, cudaStream_t s) {
  const int64_t plane = (int64_t)a.num_kv_heads * a.block_size * a.head_dim;
  int launches = 0;
  for (int b0 = 0; b0 < a.batch; b0 += seqs) {
    TreeAttnArgs x = a;
    x.batch = std::min(seqs, a.batch - b0);
    x.cu_seqlens_q += b0;
    x.seq_lens += b0;
    x.block_tables += b0 * a.table_stride;
    const int64_t blocks = (int64_t)x.batch * a.max_blocks;
    Stage o;
    o.kv = static_cast<bf16*>(stage);
    o.scales = reinterpret_cast<float*>(o.kv + blocks * 2 * plane);
    o.key_stride = key_stride(a);
    o.tables = reinterpret_cast<int*>(o.scales + (int64_t)x.batch * a.num_kv_heads * 2 * o.key_stride);
    const int64_t pieces = (plane / 16 + kPiece - 1) / kPiece, most = (int64_t)a.max_blocks * 2 * pieces;
    const int each = (device_sm_count() * kCtasPerSm + x.batch - 1) / x.batch;
    const dim3 grid((unsigned)std::min<int64_t>(most, each), x.batch);
    if (a.head_dim == 128) {
      if (a.kv_int8 == 2) tree_stage_kernel<128, true><<<grid, kThreads, 0, s>>>(x, o);
      else tree_stage_kernel<128, false><<<grid, kThreads, 0, s>>>(x, o);
    } else {
      if (a.kv_int8 == 2) tree_stage_kernel<64, true><<<grid, kThreads, 0, s>>>(x, o);
      else tree_stage_kernel<64, false><<<grid, kThreads, 0, s>>>(x, o);
    }
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) throw std::runtime_error(std::string("tree_attn stage: ") + cudaGetErrorString(e));
    TreeAttnTcPlan q = p;
    if (a.kv_int8 == 1) {
      q.key_scales = o.scales;
      q.key_stride = o.key_stride;
    }
    x.kv_int8 = 0;
    x.k_cache = o.kv;
    x.v_cache = o.kv + plane;
    x.block_tables = o.tables;
    x.table_stride = a.max_blocks;
    x.block_stride = 2 * plane;
    x.num_blocks = (int)blocks;
    launches += 1 + tree_attn_tc(x, q, s);
  }
  return launches;
}

}  // namespace b200
