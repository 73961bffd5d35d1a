// A whole MoE layer for a few tokens (a decode step of one request, the nodes of a few
// drafted trees) in one launch:
//
//   logits = bf16(x Wr^T),  p = softmax(logits),  top-k (lowest id wins a tie),
//   w_k = bf16(p_k / sum p),
//   out = sum_k w_k Wd_e ( silu(Wg_e x) * (Wu_e x) ),   e = the token's k-th expert
//
// The grid is launched cooperatively, one CTA per SM, and synchronises twice: after
// the logits and after the experts' hidden rows.  Rounding points: the logits and the
// routing weights are rounded to bf16 (those of the model's router), the output once;
// an e4m3 weight enters as exactly q * scale.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <stdexcept>
#include <string>

#include "moe_few.h"
#include "pdl.cuh"
#include "sm100.cuh"

namespace b200 {
namespace {

namespace cg = cooperative_groups;
using bf16 = __nv_bfloat16;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;

// fp64 -> bf16 in one rounding: fp32 with round-to-odd keeps the bit that decides a tie.
__device__ __forceinline__ float bf16_of(double v) {
  float f = __double2float_rz(v);
  if ((double)f != v && !isnan(v)) f = __uint_as_float(__float_as_uint(f) | 1u);
  return __bfloat162float(__float2bfloat16(f));
}

struct Shared {
  uint64_t mask[kFewMaxExperts];        // tokens of each expert
  int start[kFewMaxExperts + 1];        // first pair of each expert
  int touched[kFewMaxExperts];          // experts with at least one token
  int n_touched;
  short pair[kFewMaxTokens * kFewMaxTopk];   // pairs (token * topk + k) in (expert, token) order
  short sel_e[kFewMaxTokens * kFewMaxTopk];
  float sel_w[kFewMaxTokens * kFewMaxTopk];
};

// Logits of experts blockIdx.x, blockIdx.x + gridDim.x, ...: a product of two bf16 is exact in
// fp32 and the sum of four stays so for nearly all of them; beyond that the sum runs in fp64,
// because a logit is rounded to bf16 and a wrong last bit there can change the experts.
__device__ void few_logits(const MoeFewArgs& a) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int e = blockIdx.x; e < a.E; e += gridDim.x) {
    const bf16* wr = static_cast<const bf16*>(a.router) + (int64_t)e * a.H;
    for (int t = warp; t < a.T; t += kWarps) {
      const bf16* xr = static_cast<const bf16*>(a.x) + (int64_t)t * a.H;
      double acc = 0.0;
      for (int c = lane * 8; c < a.H; c += 256) {
        const uint4 wv = *reinterpret_cast<const uint4*>(wr + c), xv = *reinterpret_cast<const uint4*>(xr + c);
        const uint32_t wu[4] = {wv.x, wv.y, wv.z, wv.w}, xu[4] = {xv.x, xv.y, xv.z, xv.w};
        float p[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[2 * i] = __uint_as_float(wu[i] << 16) * __uint_as_float(xu[i] << 16);
          p[2 * i + 1] = __uint_as_float(wu[i] & 0xffff0000u) * __uint_as_float(xu[i] & 0xffff0000u);
        }
        acc += (double)((p[0] + p[1]) + (p[2] + p[3]));
        acc += (double)((p[4] + p[5]) + (p[6] + p[7]));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
      if (lane == 0) a.logits[t * a.E + e] = bf16_of(acc);
    }
  }
}

// Top-k and weights of every token and the pairs in expert order; every CTA does all of it.
__device__ void few_route(const MoeFewArgs& a, Shared& s) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int EPL = kFewMaxExperts / 32;
  for (int e = threadIdx.x; e < a.E; e += kThreads) s.mask[e] = 0;
  for (int t = warp; t < a.T; t += kWarps) {
    float v[EPL];
    uint32_t key[EPL];
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      const int e = j * 32 + lane;
      v[j] = e < a.E ? __ldcg(a.logits + t * a.E + e) : -INFINITY;
      // (logit, lowest id first) as one unsigned key: bf16 bits in order, then 0xffff - id
      uint32_t u = __float_as_uint(v[j]) >> 16;
      u = (u & 0x8000u) ? (0xffffu ^ u) : (u | 0x8000u);
      key[j] = e < a.E ? (u << 16) | (0xffffu - e) : 0u;
    }
    int pick = 0;
    float mx = 0.f, w = 0.f, wsum = 0.f, sum = 0.f;
    for (int k = 0; k < a.topk; ++k) {
      uint32_t best = 0;
#pragma unroll
      for (int j = 0; j < EPL; ++j) best = max(best, key[j]);
      best = __reduce_max_sync(0xffffffffu, best);
      const int e = 0xffff - (int)(best & 0xffffu);
      uint32_t u = best >> 16;
      u = (u & 0x8000u) ? (u & 0x7fffu) : (0xffffu ^ u);
      const float l = __uint_as_float(u << 16);
      if (k == 0) {
        mx = l;
#pragma unroll
        for (int j = 0; j < EPL; ++j) sum += j * 32 + lane < a.E ? expf(v[j] - mx) : 0.f;
        sum = warp_sum(sum);
      }
      const float p = expf(l - mx) / sum;
      wsum += p;
      if (lane == k) { pick = e; w = p; }
#pragma unroll
      for (int j = 0; j < EPL; ++j)
        if (key[j] == best) key[j] = 0u;
    }
    if (lane < a.topk) {
      if (a.renorm) w /= wsum;
      w = __bfloat162float(__float2bfloat16(w));
      const int p = t * a.topk + lane;
      s.sel_e[p] = (short)pick;
      s.sel_w[p] = w;
      if (blockIdx.x == 0) {
        if (a.ids != nullptr) a.ids[p] = pick;
        if (a.weights != nullptr) a.weights[p] = w;
      }
    }
  }
  __syncthreads();
  const int pairs = a.T * a.topk;
  for (int p = threadIdx.x; p < pairs; p += kThreads)
    atomicOr(reinterpret_cast<unsigned long long*>(&s.mask[s.sel_e[p]]), 1ull << (p / a.topk));
  __syncthreads();
  if (warp == 0) {
    int at = 0, nt = 0;
    for (int e0 = 0; e0 < a.E; e0 += 32) {
      const int e = e0 + lane;
      const int c = e < a.E ? __popcll(s.mask[e]) : 0;
      int incl = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
      }
      if (e < a.E) s.start[e] = at + incl - c;
      const unsigned has = __ballot_sync(0xffffffffu, c > 0);
      if (c > 0) s.touched[nt + __popc(has & ((1u << lane) - 1))] = e;
      nt += __popc(has);
      at += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) { s.start[a.E] = at; s.n_touched = nt; }
  }
  __syncthreads();
  for (int p = threadIdx.x; p < pairs; p += kThreads) {
    const int e = s.sel_e[p], t = p / a.topk;
    s.pair[s.start[e] + __popcll(s.mask[e] & ((1ull << t) - 1))] = (short)p;
  }
  __syncthreads();
}

// Weight (row, col) of expert e as the number it stands for.
__device__ __forceinline__ float few_weight(const MoeFewArgs& a, const void* w, const float* s, int N, int K, int e,
                                            int row, int col) {
  if (!a.fp8) return __bfloat162float(static_cast<const bf16*>(w)[((int64_t)e * N + row) * K + col]);
  int64_t at;
  if (a.tiled) {
    const int r = row & 127, u = ((col >> 4) & 3) ^ ((r >> 1) & 3);
    at = (((int64_t)e * (N >> 7) + (row >> 7)) * (K >> 6) + (col >> 6)) * 8192 + r * 64 + u * 16 + (col & 15);
  } else {
    at = ((int64_t)e * N + row) * K + col;
  }
  const __nv_fp8_e4m3 q = static_cast<const __nv_fp8_e4m3*>(w)[at];
  return (float)q * s[((int64_t)e * (N >> 7) + (row >> 7)) * (K >> 7) + (col >> 7)];
}

__global__ void __launch_bounds__(kThreads, 1) moe_few_kernel(const MoeFewArgs a) {
  __shared__ Shared s;
  cg::grid_group grid = cg::this_grid();
  const int lane = threadIdx.x & 31;
  const int wid = blockIdx.x * kWarps + (threadIdx.x >> 5), nw = gridDim.x * kWarps;
  few_logits(a);
  grid.sync();
  few_route(a, s);
  float* h = static_cast<float*>(a.h);
  // hidden rows: a warp per (touched expert, hidden unit)
  for (int it = wid; it < s.n_touched * a.I; it += nw) {
    const int e = s.touched[it / a.I], i = it % a.I;
    for (int j = s.start[e]; j < s.start[e + 1]; ++j) {
      const int p = s.pair[j];
      const bf16* xr = static_cast<const bf16*>(a.x) + (int64_t)(p / a.topk) * a.H;
      float g = 0.f, u = 0.f;
      for (int c = lane; c < a.H; c += 32) {
        const float xv = __bfloat162float(xr[c]);
        g = fmaf(few_weight(a, a.w13, a.s13, 2 * a.I, a.H, e, i, c), xv, g);
        u = fmaf(few_weight(a, a.w13, a.s13, 2 * a.I, a.H, e, a.I + i, c), xv, u);
      }
      g = warp_sum(g);
      u = warp_sum(u);
      if (lane == 0) h[(int64_t)p * a.I + i] = g / (1.f + expf(-g)) * u;
    }
  }
  grid.sync();
  // outputs: a warp per (token, column), its experts in the order of the top-k
  for (int it = wid; it < a.T * a.H; it += nw) {
    const int t = it / a.H, c = it % a.H;
    float y = 0.f;
    for (int k = 0; k < a.topk; ++k) {
      const int p = t * a.topk + k, e = s.sel_e[p];
      float v = 0.f;
      for (int i = lane; i < a.I; i += 32)
        v = fmaf(few_weight(a, a.w2, a.s2, a.H, a.I, e, c, i), __ldcg(h + (int64_t)p * a.I + i), v);
      y = fmaf(warp_sum(v), s.sel_w[p], y);
    }
    if (lane == 0) static_cast<bf16*>(a.out)[(int64_t)t * a.H + c] = __float2bfloat16(y);
  }
}

}  // namespace

void moe_few(const MoeFewArgs& a, cudaStream_t s) {
  if (a.T == 0) return;
  MoeFewArgs args = a;
  void* params[] = {&args};
  // every CTA waits for the others: a cooperative launch places all of them at once or fails
  const cudaError_t e = cudaLaunchCooperativeKernel(reinterpret_cast<const void*>(moe_few_kernel),
                                                    dim3(device_sm_count()), dim3(kThreads), params, 0, s);
  if (e != cudaSuccess) throw std::runtime_error(std::string("moe_few: ") + cudaGetErrorString(e));
}

}  // namespace b200
