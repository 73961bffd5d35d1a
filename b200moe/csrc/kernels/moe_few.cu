// A whole MoE layer for a few tokens (a decode step of one request, the nodes of a few
// drafted trees) in one launch:
//
//   logits = bf16(x Wr^T),  p = softmax(logits),  top-k (lowest id wins a tie),
//   w_k = bf16(p_k / sum p),
//   out = sum_k w_k Wd_e ( silu(Wg_e x) * (Wu_e x) ),   e = the token's k-th expert
//
// The grid is launched cooperatively, one CTA per SM, and synchronises after the logits and
// after the experts' hidden rows, above 16 tokens also between top-k and its tables, above 4
// tokens in front of the last sums.
//
// Nearly all the time goes into reading the touched experts' weights once, so the
// kernel is built around that stream.  A team of four, two or one warps takes 32 weight
// rows of one expert -- 16 gate and the 16 up rows beside them, or 32 rows of Wd -- and
// each warp its part of K, for up to 8 of its tokens at a time.  Every lane brings what it multiplies
// itself, weights and tokens alike, into its own places of a ring per warp (16-byte
// asynchronous copies): no bank conflict lies on the way, any weight layout is an address
// rule, and nothing that comes from memory is waited for in a register.  The ring is
// refilled across items.  (Bulk copies of 1 KB by a thread of each warp were bound by their
// issue.)  The products are warp-level MMAs with the weights as the 16-row operand and the
// tokens as columns.  K is permuted alike in both operands so that a lane's operand is 16
// weights of a row.
//
// Operand types, e4m3 weights.  The first product takes them as they are.  A bf16 value has 8 significant
// bits and an e4m3 value 4, so a token enters as two e4m3 terms: x / f = hi + lo / 16 with f the power of
// two that brings the row's largest value to [2^7, 2^8).  That is exact down to 2^-14 of the largest value
// and off by at most 2^-21 of it below.  (f16 operands would need a conversion of every weight, which cost
// more instructions than all the rest of the loop.)  Hidden values keep 11 bits: f16 with a factor for
// each 16 of them, against weights converted to f16 exactly.  Factors and block scales multiply fp32 sums
// of 64 products, so a weight counts as exactly q * scale.  bf16 weights meet x as it is and a hidden
// value as two bf16, value and rest.
//
// The parts of K are added in order through shared memory.  The rows of Wd write fp32 (token, k) slots.
// A token's slots are added in the order of the top-k: with up to 4 tokens by the team that finishes the
// last expert of a tile of 128 columns, above by the whole grid behind one more barrier (at 64 tokens one
// warp per tile needed 47 us for them).
//
// Bound by the weight stream where it is long: 16 tokens of 128 experts (hidden 2048, inner 768, top-8)
// read 390 MB in 92 us, 64 tokens 595 MB in 143 us, 4.2 TB/s with about 15 us of logits, routing and
// barriers.  One token (38 MB, 27 us) and small layers (12.5 us) are bound by the chain of launch, logits,
// barrier, routing, two dependent streams and the last sums.  (Kernel times, 18 calls in a graph; in a long
// row of calls 95, 152, 28.8 and 14.3 us, the 64 tokens at the clock that the card sustains.)
//
// Rounding points: the logits (fp64 sums) and the routing weights are rounded to bf16 (those of the
// model's router), the output once.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <stdexcept>
#include <string>
#include <type_traits>

#include "moe_few.h"
#include "pdl.cuh"
#include "sm100.cuh"

namespace b200 {
namespace {

namespace cg = cooperative_groups;
using bf16 = __nv_bfloat16;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kRingBytes = 12832;        // of a warp
constexpr int kCols = 8;                 // tokens of one pass
// Tokens up to which the last team of a tile adds the slots, a warp each (3 tokens: 44.7 us, by the grid
// behind a barrier 45.8; at 8 the grid is as fast, at 64 far faster).
constexpr int kLastAdds = 4;

// fp64 -> bf16 in one rounding: fp32 with round-to-odd keeps the bit that decides a tie.
__device__ __forceinline__ float bf16_of(double v) {
  float f = __double2float_rz(v);
  if ((double)f != v && !isnan(v)) f = __uint_as_float(__float_as_uint(f) | 1u);
  return __bfloat162float(__float2bfloat16(f));
}

constexpr int kPairs = kFewMaxTokens * kFewMaxTopk;

// Routing tables.  A pass is up to kCols tokens of one expert; passes are in expert order.
struct Shared {
  uint32_t mask[2][kFewMaxExperts];     // tokens of each expert, 32 to a word
  int2 warp_sums[kFewMaxExperts / 32];
  int passes;
  short start[kFewMaxExperts + 2];      // first pair of each expert
  uint8_t pass_e[kPairs];               // expert of each pass
  short pass_first[kPairs];             // its first pair and how many
  uint8_t pass_cnt[kPairs];
  uint8_t token[kPairs];                // token of each pair, in (expert, token) order
  short pair[kPairs];                   // token * topk + k of each pair
  uint8_t sel_e[kPairs];
  float sel_w[kPairs];
};

// The sum of eight products of bf16 pairs: exact in fp32 each (above its smallest normal number), and added
// in fp64.  (Sums of four in fp32 dropped a bit in 1 of 50, and with it the side of a bf16 border on
// which a logit lies.)
__device__ __forceinline__ double dot8(const uint4& w, const uint4& x, double acc) {
  const uint32_t wu[4] = {w.x, w.y, w.z, w.w}, xu[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    acc += (double)(__uint_as_float(wu[i] << 16) * __uint_as_float(xu[i] << 16));
    acc += (double)(__uint_as_float(wu[i] & 0xffff0000u) * __uint_as_float(xu[i] & 0xffff0000u));
  }
  return acc;
}

// Values 2 q and 2 q + 1 of eight bf16.
__device__ __forceinline__ void two_of(const uint4& v, int q, double (&d)[2]) {
  const uint32_t u = q == 0 ? v.x : q == 1 ? v.y : q == 2 ? v.z : v.w;
  d[0] = (double)__uint_as_float(u << 16);
  d[1] = (double)__uint_as_float(u & 0xffff0000u);
}

// Logits of experts blockIdx.x + gridDim.x, ..., summed in fp64: a logit is rounded to bf16, and
// a wrong last bit there can change the experts.
__device__ void few_logits(const MoeFewArgs& a, double* red) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (a.T > kWarps) {
    // many tokens: tiles of 16 tokens x 4 experts, so x is not read once per expert; a warp takes 4 tokens and
    // a quarter of K, which converts half a value per product (1 with a token per warp: 2.5 us more at 64 tokens)
    const int groups = (a.T + kWarps - 1) / kWarps, tiles = groups * ((a.E + 3) / 4);
    for (int i = blockIdx.x; i < tiles; i += gridDim.x) {
      const int t0 = i % groups * kWarps + (warp & 3) * 4, e0 = i / groups * 4;
      double acc[16] = {};                       // [token][expert]; the last rows are repeated
      if (t0 < a.T) {
        for (int c = (warp >> 2) * 256 + lane * 8; c < a.H; c += 1024) {
          uint4 xv[4], wv[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            xv[j] = *reinterpret_cast<const uint4*>(static_cast<const bf16*>(a.x) + min(t0 + j, a.T - 1) * a.H + c);
            wv[j] = __ldg(reinterpret_cast<const uint4*>(static_cast<const bf16*>(a.router) + min(e0 + j, a.E - 1) * a.H + c));
          }
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            double xd[4][2];
#pragma unroll
            for (int j = 0; j < 4; ++j) two_of(xv[j], q, xd[j]);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              double wd[2];
              two_of(wv[k], q, wd);
#pragma unroll
              for (int j = 0; j < 4; ++j) acc[j * 4 + k] = fma(xd[j][1], wd[1], fma(xd[j][0], wd[0], acc[j * 4 + k]));
            }
          }
        }
        // lane l < 16 gets sum l of the warp: halves of the sums are exchanged
#pragma unroll
        for (int n = 8; n > 0; n >>= 1) {
          const bool up = lane & n;
#pragma unroll
          for (int j = 0; j < n; ++j) {
            const double give = up ? acc[j] : acc[j + n];
            acc[j] = (up ? acc[j + n] : acc[j]) + __shfl_xor_sync(0xffffffffu, give, n);
          }
        }
        acc[0] += __shfl_xor_sync(0xffffffffu, acc[0], 16);
        if (lane < 16) red[warp * 16 + lane] = acc[0];
      }
      __syncthreads();
      if (threadIdx.x < 64) {                    // 16 tokens x 4 experts, the quarters of K in order
        const int t = i % groups * kWarps + (threadIdx.x >> 2), e = e0 + (threadIdx.x & 3);
        double sum = 0.0;
#pragma unroll
        for (int q = 0; q < 4; ++q) sum += red[(q * 4 + (threadIdx.x >> 4)) * 16 + (threadIdx.x & 15)];
        if (t < a.T && e < a.E) a.logits[t * a.E + e] = bf16_of(sum);
      }
      __syncthreads();
    }
    return;
  }
  // few tokens: several warps share one, a part of K each
  const int share = a.T > 8 ? 1 : a.T > 4 ? 2 : a.T > 2 ? 4 : a.T > 1 ? 8 : 16;
  const int sub = warp % share;
  for (int e = blockIdx.x; e < a.E; e += gridDim.x) {
    const bf16* wr = static_cast<const bf16*>(a.router) + (int64_t)e * a.H;
    for (int t = warp / share; t < a.T; t += kWarps / share) {
      const bf16* xr = static_cast<const bf16*>(a.x) + (int64_t)t * a.H;
      double acc = 0.0;
#pragma unroll 8
      for (int c = (sub * 32 + lane) * 8; c < a.H; c += share * 256) {
        acc = dot8(*reinterpret_cast<const uint4*>(wr + c), *reinterpret_cast<const uint4*>(xr + c), acc);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
      if (share == 1) {
        if (lane == 0) a.logits[t * a.E + e] = bf16_of(acc);
      } else if (lane == 0) {
        red[warp] = acc;
      }
    }
    if (share > 1) {
      __syncthreads();
      if (threadIdx.x < a.T) {
        double acc = 0.0;
        for (int i = 0; i < share; ++i) acc += red[threadIdx.x * share + i];
        a.logits[threadIdx.x * a.E + e] = bf16_of(acc);
      }
      __syncthreads();
    }
  }
}

// The power of two f with |v| / f in [2^top, 2^(top + 1)) for the largest |v| = m of a row; 1 where m is
// not finite, the smallest normal number where it is zero or tiny.
__device__ __forceinline__ float factor_of(float m, int top) {
  const int e = (int)(__float_as_uint(m) >> 23);   // biased exponent, sign is 0
  return e == 255 ? 1.f : __uint_as_float((uint32_t)max(e - top, 1) << 23);
}

// The two e4m3 terms of x and the rows' factors: row t by CTA gridDim.x - 1 - t.
__device__ void few_rows(const MoeFewArgs& a, float* red) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int t = gridDim.x - 1 - blockIdx.x; t < a.T; t += gridDim.x) {
    const bf16* xr = static_cast<const bf16*>(a.x) + (int64_t)t * a.H;
    uint32_t top = 0;   // largest |x| as bits: an infinity or NaN is above every number
    for (int c = threadIdx.x * 2; c < a.H; c += kThreads * 2) {
      const uint32_t v = *reinterpret_cast<const uint32_t*>(xr + c) & 0x7fff7fffu;
      top = max(top, max(v << 16, v & 0xffff0000u));
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) red[warp] = __uint_as_float(top);
    __syncthreads();
    top = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) top = max(top, __float_as_uint(red[i]));
    const float f = factor_of(__uint_as_float(top), 7), inv = 1.f / f;   // a power of two: exact
    uint16_t* hi = reinterpret_cast<uint16_t*>(static_cast<uint8_t*>(a.x8) + (int64_t)t * 2 * a.H);
    for (int c = threadIdx.x * 2; c < a.H; c += kThreads * 2) {
      const float2 v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(xr + c));
      const float2 w = make_float2(v.x * inv, v.y * inv);
      const uint16_t h = __nv_cvt_float2_to_fp8x2(w, __NV_NOSAT, __NV_E4M3);
      const __half2_raw hr = __nv_cvt_fp8x2_to_halfraw2(h, __NV_E4M3);
      const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&hr));
      hi[c / 2] = h;
      hi[(c + a.H) / 2] = __nv_cvt_float2_to_fp8x2(make_float2((w.x - back.x) * 16.f, (w.y - back.y) * 16.f), __NV_NOSAT, __NV_E4M3);
    }
    if (threadIdx.x == 0) a.x_factor[t] = f;
    __syncthreads();
  }
}

// n / d for 0 <= n < 2^24, without the compiler's division.
__device__ __forceinline__ int quotient(int n, int d) {
  int q = (int)__fdividef((float)n, (float)d);
  const int r = n - q * d;
  if (r < 0) --q;
  if (r >= d) ++q;
  return q;
}

// Top-k and weights of token t by one warp: lane k < topk gets the k-th expert and its weight.
template <int EPL>
__device__ __forceinline__ void few_topk(const MoeFewArgs& a, int t, int lane, int& pick, float& w) {
  float v[EPL];
  uint32_t key[EPL];
#pragma unroll
  for (int j = 0; j < EPL; ++j) v[j] = j * 32 + lane < a.E ? __ldcg(a.logits + t * a.E + j * 32 + lane) : -INFINITY;
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    const int e = j * 32 + lane;
    // (logit, lowest id first) as one unsigned key: bf16 bits in order (-0 as 0), then 0xffff - id
    uint32_t u = __float_as_uint(v[j] + 0.f) >> 16;
    u = (u & 0x8000u) ? (0xffffu ^ u) : (u | 0x8000u);
    key[j] = e < a.E ? (u << 16) | (0xffffu - e) : 0u;
  }
  uint32_t mine = 0;               // lane k: the k-th key
  uint32_t first = 0;
  for (int k = 0; k < a.topk; ++k) {
    uint32_t best = key[0];
#pragma unroll
    for (int j = 1; j < EPL; ++j) best = max(best, key[j]);
    best = __reduce_max_sync(0xffffffffu, best);
    if (k == 0) first = best;
    if (lane == k) mine = best;
#pragma unroll
    for (int j = 0; j < EPL; ++j)
      if (key[j] == best) key[j] = 0u;
  }
  auto logit_of = [](uint32_t k) {
    const uint32_t u = k >> 16;
    return __uint_as_float(((u & 0x8000u) ? (u & 0x7fffu) : (0xffffu ^ u)) << 16);
  };
  const float mx = logit_of(first);
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < EPL; ++j) sum += expf(v[j] - mx);       // no expert: exp(-inf) = 0
  sum = warp_sum(sum);
  w = lane < a.topk ? expf(logit_of(mine) - mx) / sum : 0.f;
  const float wsum = warp_sum(w);
  if (a.renorm) w /= wsum;
  w = __bfloat162float(__float2bfloat16(w));
  pick = 0xffff - (int)(mine & 0xffffu);
}

// The routing tables, in every CTA.  Up to 16 tokens every CTA does the top-k of all; more tokens are
// spread over the CTAs and exchanged, which costs a barrier and saves a CTA the later rounds of 16.
template <int EPL>
__device__ void few_route(const MoeFewArgs& a, Shared& s, cg::grid_group& grid) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int e = threadIdx.x; e < 2 * kFewMaxExperts; e += kThreads) (&s.mask[0][0])[e] = 0;
  const bool spread = a.T > kWarps;
  if (spread) {
    const int t = blockIdx.x + warp * gridDim.x;             // tokens side by side on different SMs
    if (t < a.T) {
      int pick;
      float w;
      few_topk<EPL>(a, t, lane, pick, w);
      if (lane < a.topk) {
        __stcg(a.sel + t * a.topk + lane, make_int2(pick, __float_as_int(w)));
        if (a.ids != nullptr) a.ids[t * a.topk + lane] = pick;
        if (a.weights != nullptr) a.weights[t * a.topk + lane] = w;
      }
    }
    grid.sync();
  }
  __syncthreads();
  auto take = [&](int t, int p, int pick, float w) {
    s.sel_e[p] = (uint8_t)pick;
    s.sel_w[p] = w;
    atomicOr(&s.mask[t >> 5][pick], 1u << (t & 31));
  };
  if (spread) {
    for (int p = threadIdx.x; p < a.T * a.topk; p += kThreads) {
      const int2 x = __ldcg(a.sel + p);
      take(quotient(p, a.topk), p, x.x, __int_as_float(x.y));
    }
  } else if (warp < a.T) {
    int pick;
    float w;
    few_topk<EPL>(a, warp, lane, pick, w);
    if (lane < a.topk) {
      const int p = warp * a.topk + lane;
      take(warp, p, pick, w);
      if (blockIdx.x == 0) {
        if (a.ids != nullptr) a.ids[p] = pick;
        if (a.weights != nullptr) a.weights[p] = w;
      }
    }
  }
  __syncthreads();
  // first pair and passes of every expert: a thread per expert
  const int e = threadIdx.x;
  int c = 0, np = 0, ci = 0, ni = 0;
  if (e < kFewMaxExperts) {
    c = ci = __popc(s.mask[0][e]) + __popc(s.mask[1][e]);
    np = ni = (c + kCols - 1) / kCols;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int cu = __shfl_up_sync(0xffffffffu, ci, o), nu = __shfl_up_sync(0xffffffffu, ni, o);
      if (lane >= o) { ci += cu; ni += nu; }
    }
    if (lane == 31) s.warp_sums[warp] = make_int2(ci, ni);
  }
  __syncthreads();
  if (e < kFewMaxExperts) {
#pragma unroll
    for (int i = 0; i < kFewMaxExperts / 32; ++i) {
      const int2 x = s.warp_sums[i];
      if (i < warp) { ci += x.x; ni += x.y; }
    }
    s.start[e] = (short)(ci - c);
    for (int i = 0; i < np; ++i) {
      const int q = ni - np + i;
      s.pass_e[q] = (uint8_t)e;
      s.pass_first[q] = (short)(ci - c + i * kCols);
      s.pass_cnt[q] = (uint8_t)min(kCols, c - i * kCols);
    }
    if (e == kFewMaxExperts - 1) s.passes = ni;
  }
  __syncthreads();
  for (int p = threadIdx.x; p < a.T * a.topk; p += kThreads) {
    const int x = s.sel_e[p], t = quotient(p, a.topk);
    const uint32_t below = (1u << (t & 31)) - 1;
    const int at = s.start[x] + (t < 32 ? __popc(s.mask[0][x] & below) : __popc(s.mask[0][x]) + __popc(s.mask[1][x] & below));
    s.pair[at] = (short)p;
    s.token[at] = (uint8_t)t;
  }
  __syncthreads();
}

constexpr int kRing = kWarps * kRingBytes;
constexpr int kRed = kRing;                                  // [kWarps][8][32] floats
constexpr int kShared = kRed + kWarps * 8 * 32 * 4;          // Shared
constexpr int kSmem = kShared + (int)sizeof(Shared);
static_assert(kSmem <= 232448, "shared memory budget");

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// all but the newest N groups have landed
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
               "{%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_e4m3(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
               "{%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
               "{%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Two e4m3 -> two f16, exactly (NaN stays NaN).
__device__ __forceinline__ uint32_t f16x2_of(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two), __NV_E4M3);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <bool FP8>
struct Few {
  static constexpr int PER = FP8 ? 1 : 2;              // 16-byte pieces of a lane's 16 weights
  // A stage of the ring holds two runs of 64 K, so that their products overlap.  A run: weights
  // [4 * PER][32 lanes] x 16 bytes, tokens [2 or 4][32] x 16 bytes and, for e4m3, the hidden values'
  // factors [32]; behind the stages the block scales, two for each run.
  static constexpr int KPS = FP8 ? 2 : 1;
  static constexpr int W = 2048 * PER, B = FP8 ? 1024 : 2048;
  static constexpr int kRunBytes = FP8 ? W + B + 128 : W + B, kStages = 2;
  static_assert(kStages * KPS * (kRunBytes + (FP8 ? 8 : 0)) <= kRingBytes, "ring");
  const MoeFewArgs& a;
  Shared& s;
  uint8_t* ring;
  int lane, part, kw, team, teams;  // part: of the kw parts of K; team: over the grid

  // ------------------------------------------------------------ the stream of items
  // An item is a pass against a block of rows: 16 gate and up rows (phase 0) or 32 rows of Wd (phase 1).
  // Blocks are parts of a tile of 128 rows.  Order of phase 0: pass, tile, block; of phase 1: tile, pass,
  // block, so that the sums of 128 outputs are over early.  A team takes the team-th of equal runs of
  // either order, and within a tile only addresses move on.
  __device__ __forceinline__ int tiles(int phase) const { return (phase ? a.H : a.I) >> 7; }
  __device__ __forceinline__ static constexpr int subs(int phase) { return phase ? 4 : 8; }
  // warps of a team (4, 2 or 1): the least rounds of items, each its runs and about one run's time more
  // (with 8 among them at most 1 % is gained, and 10 tokens take 80 us instead of 73)
  __device__ __forceinline__ int team_warps(int phase) const {
    const int n = s.passes * tiles(phase) * subs(phase), runs = (phase ? a.I : a.H) / 64;
    int best = 4, cost = 1 << 30;
#pragma unroll
    for (int w = 4; w >= 1; w >>= 1) {
      const int t = kWarps / w * (int)gridDim.x, c = (quotient(n + t - 1, t)) * (runs / w + 1);
      if (c < cost) { cost = c; best = w; }
    }
    return best;
  }
  __device__ __forceinline__ void enter(int phase, int warp) {
    kw = team_warps(phase);
    part = warp & (kw - 1);
    team = warp / kw * (int)gridDim.x + (int)blockIdx.x;
    teams = kWarps / kw * (int)gridDim.x;
  }
  __device__ __forceinline__ int run0(int phase) const { return (phase ? a.I : a.H) / 64 * part / kw; }
  __device__ __forceinline__ int run1(int phase) const { return (phase ? a.I : a.H) / 64 * (part + 1) / kw; }

  struct Cursor {
    int phase, left;               // phase 2: over; items left in the phase, this one among them
    int q, tile, sub;              // pass, tile of rows, block of the tile
  };
  __device__ __forceinline__ Cursor begin(int phase) const {
    Cursor c;
    c.phase = phase;
    const int n = s.passes * tiles(phase) * subs(phase), each = quotient(n, teams), over = n - each * teams;
    const int lo = each * team + min(team, over);
    c.left = each + (team < over ? 1 : 0);
    const int inner = phase ? s.passes : tiles(phase), x = lo / subs(phase), o = quotient(x, inner);
    c.sub = lo % subs(phase);
    c.q = phase ? x - o * inner : o;
    c.tile = phase ? o : x - o * inner;
    return c;
  }
  // to the next item; true: in the same tile and pass
  __device__ __forceinline__ bool next(Cursor& c) const {
    if (--c.left == 0) return false;
    if (++c.sub < subs(c.phase)) return true;
    c.sub = 0;
    if (c.phase == 0) {
      if (++c.tile == tiles(0)) { c.tile = 0; ++c.q; }
    } else {
      if (++c.q == s.passes) { c.q = 0; ++c.tile; }
    }
    return false;
  }

  // The item whose runs are being brought in.
  struct Ahead {
    Cursor c;
    int st, runs;                  // run of 64 K, runs of this warp
    const uint8_t* w0;             // this lane's weights of rows g of the two row blocks, run st
    const uint8_t* w1;
    int row8, run, block;          // bytes from row g to row g + 8, to the next run, to the next block
    const uint8_t* tok;            // this lane's token or hidden row; null: none
    int tok_run, tok_piece;        // bytes to the next run, and between its two pieces of a run
    const float* fac;              // its factors
    const float* sc;               // lanes 0 and 1: block scales of a row block
    int k0;
  };
  __device__ __forceinline__ bool more(const Ahead& h) const { return h.c.phase < 2; }
  __device__ __forceinline__ void resolve(Ahead& h) const {
    if (h.c.left <= 0 || run0(h.c.phase) == run1(h.c.phase)) { h.c.phase = 2; return; }   // nothing (more) to bring in
    const int ph = h.c.phase, e = s.pass_e[h.c.q];
    h.st = 0;
    h.k0 = run0(ph);
    h.runs = run1(ph) - h.k0;
    const int N = ph ? a.H : 2 * a.I, K = ph ? a.I : a.H;
    // rows of the first block of the tile, and of the block's second half
    const uint32_t r0 = (uint32_t)(e * N + h.c.tile * 128), r1 = ph ? r0 : r0 + a.I;
    const int g = lane >> 2, t = lane & 3;
    const uint8_t* w = static_cast<const uint8_t*>(ph ? a.w2 : a.w13);
    const int rows = ph ? 32 : 16;                     // of a block in either half
    uint32_t row;                                      // bytes of a row
    if (FP8 && a.tiled) {
      // [row / 128][K / 64][128][64]; 16-byte chunk u of a row at u ^ ((row >> 1) & 3)
      row = 64;
      h.run = 8192;
      w += g * 64 + ((t ^ ((g >> 1) & 3)) << 4);
      h.w0 = w + (uint64_t)((r0 >> 7) * (K >> 6) + h.k0) * 8192;
      h.w1 = w + (uint64_t)((r1 >> 7) * (K >> 6) + h.k0) * 8192;
    } else {
      row = K * (FP8 ? 1 : 2);
      h.run = FP8 ? 64 : 128;
      w += h.k0 * h.run + t * 16;
      h.w0 = w + (uint64_t)(r0 + g) * row;
      h.w1 = w + (uint64_t)(r1 + g) * row;
    }
    h.row8 = 8 * row;
    h.block = rows * row;
    h.w0 += h.c.sub * h.block;
    h.w1 += h.c.sub * h.block + (ph ? 16 * row : 0);
    h.block -= h.runs * h.run;                         // from behind the last run
    h.tok = nullptr;
    if (g < s.pass_cnt[h.c.q]) {
      const int at = s.pass_first[h.c.q] + g;
      if (FP8 && ph == 0) {          // two terms of 16 values
        h.tok = static_cast<const uint8_t*>(a.x8) + s.token[at] * 2 * a.H + h.k0 * 64 + t * 16;
        h.tok_run = 64;
        h.tok_piece = a.H;
      } else {                       // 16 values of two bytes
        h.tok = ph == 0 ? static_cast<const uint8_t*>(a.x) + s.token[at] * a.H * 2
                        : static_cast<const uint8_t*>(a.h) + s.pair[at] * a.I * 2;
        h.tok += h.k0 * 128 + t * (FP8 ? 32 : 16);
        h.tok_run = 128;
        h.tok_piece = FP8 ? 16 : 64;
      }
      if (FP8) h.fac = a.h_factor + s.pair[at] * (a.I / 16) + h.k0 * 4 + t;
    }
    if (FP8) h.sc = (ph ? a.s2 : a.s13) + (uint64_t)((lane == 0 ? r0 : r1) >> 7) * (K >> 7);
  }
  // run st of the item into place r of the ring
  __device__ __forceinline__ void copy_run(const Ahead& h, int r, int64_t plane) const {
    const uint32_t dst = smem_u32(ring + r * kRunBytes + lane * 16);
#pragma unroll
    for (int v = 0; v < PER; ++v) {
      copy16(dst + (0 * PER + v) * 512, h.w0 + v * 64);
      copy16(dst + (1 * PER + v) * 512, h.w0 + h.row8 + v * 64);
      copy16(dst + (2 * PER + v) * 512, h.w1 + v * 64);
      copy16(dst + (3 * PER + v) * 512, h.w1 + h.row8 + v * 64);
    }
    if (FP8 && lane < 2) copy4(smem_u32(ring + kStages * KPS * kRunBytes + r * 8 + lane * 4), h.sc + ((h.k0 + h.st) >> 1));
    // A lane without a token leaves its place as it is: what stands there makes a column nobody reads.
    if (h.tok == nullptr) return;
    const uint8_t* src = h.tok + h.st * h.tok_run;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      copy16(dst + W + v * 512, src + v * h.tok_piece);
      if (!FP8 && h.c.phase == 1) copy16(dst + W + (2 + v) * 512, src + plane * 2 + v * 64);
    }
    if (FP8 && h.c.phase == 1) copy4(smem_u32(ring + r * kRunBytes + W + B + lane * 4), h.fac + h.st * 4);
  }
  // to the next run; true: of the same item
  __device__ __forceinline__ bool step(Ahead& h) const {
    h.w0 += h.run;
    h.w1 += h.run;
    if (++h.st < h.runs) return true;
    if (next(h.c)) {
      h.st = 0;
      h.w0 += h.block;
      h.w1 += h.block;
    } else {
      resolve(h);
    }
    return false;
  }

  // acc[m] += 16 weight rows x 8 tokens of a stage's n runs (the products of a missing one are dropped)
  template <int P>
  __device__ __forceinline__ void multiply(int slot, int n, float (&acc)[2][4]) const {
    constexpr int PLANES = !FP8 && P == 1 ? 2 : 1;
    const int t = lane & 3;
    uint4 b[KPS][PLANES][2];
    float sc[KPS][2][2];             // factors of the sums: [row block][column of this lane]
#pragma unroll
    for (int k = 0; k < KPS; ++k) {
      const int r = slot * KPS + k;
      const uint8_t* src = ring + r * kRunBytes + lane * 16;
#pragma unroll
      for (int p = 0; p < PLANES; ++p)
#pragma unroll
        for (int v = 0; v < 2; ++v) b[k][p][v] = *reinterpret_cast<const uint4*>(src + W + (p * 2 + v) * 512);
      if constexpr (FP8) {
        const float2 bs = *reinterpret_cast<const float2*>(ring + kStages * KPS * kRunBytes + r * 8);
        sc[k][0][0] = sc[k][0][1] = bs.x;
        sc[k][1][0] = sc[k][1][1] = bs.y;
        if constexpr (P == 1) {
          // Each lane of a token holds 16 hidden values with a factor of their own: bring the four to
          // the largest (a value that vanishes there is below 2^-24 of the others' largest).
          const float f = *reinterpret_cast<const float*>(ring + r * kRunBytes + W + B + lane * 4);
          float m = fmaxf(f, __shfl_xor_sync(0xffffffffu, f, 1));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
          const int d = (int)(__float_as_uint(f) >> 23) - (int)(__float_as_uint(m) >> 23);   // <= 0
          const __half2 h = __float2half2_rn(d < -30 ? 0.f : __uint_as_float((uint32_t)(127 + d) << 23));
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            __half2* x = reinterpret_cast<__half2*>(&b[k][0][v]);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = __hmul2(x[i], h);
          }
          const float top0 = __shfl_sync(0xffffffffu, m, t * 8), top1 = __shfl_sync(0xffffffffu, m, t * 8 + 4);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            sc[k][i][0] *= top0;
            sc[k][i][1] *= top1;
          }
        }
      }
    }
    constexpr bool E4 = FP8 && P == 0;
    float sum[KPS][2][4], low[E4 ? KPS : 1][2][4];
#pragma unroll
    for (int k = 0; k < KPS; ++k)
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sum[k][m][i] = 0.f;
          if constexpr (E4) low[k][m][i] = 0.f;
        }
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      uint4 w[KPS][2][PER];          // rows g and g + 8: 16 weights
#pragma unroll
      for (int k = 0; k < KPS; ++k)
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int v = 0; v < PER; ++v)
            w[k][r][v] = *reinterpret_cast<const uint4*>(ring + (slot * KPS + k) * kRunBytes + lane * 16 + ((m * 2 + r) * PER + v) * 512);
      if constexpr (E4) {             // 32 of the 64 K at a time: two words of each lane's 16 weights
#pragma unroll
        for (int k = 0; k < KPS; ++k) {
          const uint4 &lo = w[k][0][0], &hi = w[k][1][0], &bh = b[k][0][0], &bl = b[k][0][1];
          mma_e4m3(sum[k][m], lo.x, hi.x, lo.y, hi.y, bh.x, bh.y);
          mma_e4m3(low[k][m], lo.x, hi.x, lo.y, hi.y, bl.x, bl.y);
          mma_e4m3(sum[k][m], lo.z, hi.z, lo.w, hi.w, bh.z, bh.w);
          mma_e4m3(low[k][m], lo.z, hi.z, lo.w, hi.w, bl.z, bl.w);
        }
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)     // 16 of the 64 K: weights 4 q .. 4 q + 3 of each lane's 16
#pragma unroll
          for (int k = 0; k < KPS; ++k) {
            uint32_t af[4];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              if constexpr (FP8) {
                const uint4& y = w[k][r][0];
                const uint32_t x = q == 0 ? y.x : q == 1 ? y.y : q == 2 ? y.z : y.w;
                af[r] = f16x2_of(x & 0xffffu);
                af[r + 2] = f16x2_of(x >> 16);
              } else {
                const uint4& x = w[k][r][q >> 1];
                af[r] = q & 1 ? x.z : x.x;
                af[r + 2] = q & 1 ? x.w : x.y;
              }
            }
#pragma unroll
            for (int p = 0; p < PLANES; ++p) {
              const uint4& x = b[k][p][q >> 1];
              if constexpr (FP8) mma_f16(sum[k][m], af, q & 1 ? x.z : x.x, q & 1 ? x.w : x.y);
              else mma_bf16(sum[k][m], af, q & 1 ? x.z : x.x, q & 1 ? x.w : x.y);
            }
          }
      }
    }
#pragma unroll
    for (int k = 0; k < KPS; ++k) {
      if (k >= n) break;
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float v = sum[k][m][i];
          if constexpr (E4) v = fmaf(low[k][m][i], 0.0625f, v);
          acc[m][i] = FP8 ? fmaf(v, sc[k][m][i & 1], acc[m][i]) : acc[m][i] + v;
        }
    }
  }
};

// out[t, c .. c + 3]: the token's slots in the order of the top-k
__device__ __forceinline__ void few_add(const MoeFewArgs& a, const Shared& s, int t, int c) {
  float4 v[kFewMaxTopk];
#pragma unroll
  for (int k = 0; k < kFewMaxTopk; ++k)
    if (k < a.topk) v[k] = __ldcg(reinterpret_cast<const float4*>(a.slots + (int64_t)(t * a.topk + k) * a.H + c));
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int k = 0; k < kFewMaxTopk; ++k)
    if (k < a.topk) {
      const float w = s.sel_w[t * a.topk + k];
      y.x = fmaf(v[k].x, w, y.x);
      y.y = fmaf(v[k].y, w, y.y);
      y.z = fmaf(v[k].z, w, y.z);
      y.w = fmaf(v[k].w, w, y.w);
    }
  const __nv_bfloat162 lo = __floats2bfloat162_rn(y.x, y.y), hi = __floats2bfloat162_rn(y.z, y.w);
  uint2 o;
  o.x = *reinterpret_cast<const uint32_t*>(&lo);
  o.y = *reinterpret_cast<const uint32_t*>(&hi);
  *reinterpret_cast<uint2*>(static_cast<bf16*>(a.out) + (int64_t)t * a.H + c) = o;
}

template <bool FP8>
__global__ void __launch_bounds__(kThreads, 1)
moe_few_kernel(const MoeFewArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int last_s[kWarps];
  Shared& s = *reinterpret_cast<Shared*>(smem + kShared);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  cg::grid_group grid = cg::this_grid();
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < a.H / 128; i += kThreads) a.done[i] = 0;
  few_logits(a, reinterpret_cast<double*>(smem + kRed));
  if (FP8) few_rows(a, reinterpret_cast<float*>(smem + kRed));
  grid.sync();
  if (a.E <= 128) few_route<4>(a, s, grid);
  else few_route<kFewMaxExperts / 32>(a, s, grid);

  Few<FP8> few{a, s, smem + warp * kRingBytes, lane};
  using Cursor = typename Few<FP8>::Cursor;
  using Ahead = typename Few<FP8>::Ahead;
  constexpr int kStages = Few<FP8>::kStages, KPS = Few<FP8>::KPS;
  uint16_t* hid = static_cast<uint16_t*>(a.h);
  const int64_t hplane = (int64_t)a.T * a.topk * a.I;

  // One barrier more spreads the last sums over the grid; with a few tokens the team that brings the
  // last product of a tile is sooner done with them.
  const bool last_adds = a.T <= kLastAdds;

  Ahead ahead{};
  auto run_phase = [&](auto phase_c) {
    constexpr int P = decltype(phase_c)::value;
    few.enter(P, warp);
    const int kw = few.kw, team_in = warp / kw, tt = threadIdx.x & (kw * 32 - 1);
    float* red = reinterpret_cast<float*>(smem + kRed) + team_in * kw * 256;   // [kw][8][32]
    Cursor at = few.begin(P);
    ahead.c = at;
    few.resolve(ahead);
    const int runs = few.run1(P) - few.run0(P), stages = (runs + KPS - 1) / KPS;
    int slot = 0;                                // the ring's next stage
    int fill = kStages;                          // stages to bring in before the first is used
    int summed = 0;                              // items of the tile that this team has finished
#pragma unroll 1
    while (at.left > 0) {
      const int first = s.pass_first[at.q], cnt = s.pass_cnt[at.q];
      const int col = at.tile * 128 + at.sub * (P ? 32 : 16);
      float acc[2][4] = {};
#pragma unroll 1
      for (int k = -fill; k < stages; ++k) {
        if (k >= 0) {
          copies_wait<kStages - 1>();
          __syncwarp();                          // the scales come in through two lanes
          few.template multiply<P>(slot, runs - k * KPS, acc);
          __syncwarp();
        }
        if (few.more(ahead)) {                   // the next runs; an empty group behind the last
          few.copy_run(ahead, slot * KPS, hplane);
          if (few.step(ahead) && KPS > 1) {
            few.copy_run(ahead, slot * KPS + KPS - 1, hplane);
            few.step(ahead);
          }
        }
        copies_commit();
        slot ^= 1;
      }
      fill = 0;
      // the parts of K, added in order
      auto team_sync = [&]() {
        if (kw == 1) __syncwarp();
        else named_barrier_sync(1 + team_in, kw * 32);
      };
      team_sync();                               // the last sums have been read
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) red[few.part * 256 + (m * 4 + i) * 32 + lane] = acc[m][i];
      team_sync();
#pragma unroll 1
      for (int idx = tt; idx < 128; idx += kw * 32) {
        // (token, row): the 16 rows of a token side by side
        const int n = idx >> 4, row = idx & 15;
        if (n >= cnt) break;                     // all of a half-warp
        const int ri = (row >> 3) * 2 + (n & 1), rl = (row & 7) * 4 + (n >> 1);
        float v[2] = {0.f, 0.f};
        for (int q = 0; q < kw; ++q) {
          v[0] += red[q * 256 + ri * 32 + rl];
          v[1] += red[q * 256 + (4 + ri) * 32 + rl];
        }
        const int p = s.pair[first + n];
        if constexpr (P == 0) {
          if (FP8) {
            const float f = a.x_factor[s.token[first + n]];
            v[0] *= f;
            v[1] *= f;
          }
          const float hv = v[0] / (1.f + expf(-v[0])) * v[1];
          if constexpr (FP8) {
            const unsigned half = 0xffffu << (lane & 16);
            uint32_t top = __float_as_uint(hv) & 0x7fffffffu;   // NaN and infinity are above every number
            top = __reduce_max_sync(half, top);
            const float f = factor_of(__uint_as_float(top), 14);
            reinterpret_cast<__half*>(hid)[p * a.I + col + row] = __float2half_rn(hv * (1.f / f));
            if (row == 0) a.h_factor[p * (a.I / 16) + (col >> 4)] = f;
          } else {
            const bf16 top = __float2bfloat16(hv);
            bf16* dst = reinterpret_cast<bf16*>(hid) + p * a.I + col + row;
            dst[0] = top;
            dst[hplane] = __float2bfloat16(hv - __bfloat162float(top));
          }
        } else {
          float* dst = a.slots + (int64_t)p * a.H + col + row;
          dst[0] = v[0];
          dst[16] = v[1];
        }
      }
      __syncwarp();
      const int tile = at.tile;
      few.next(at);
      if constexpr (P == 1) {
        ++summed;
        if (last_adds && (at.left == 0 || at.tile != tile)) {
          // Items of a tile are counted when a team leaves it; the team that brings the last ones
          // adds the slots of its columns.
          __threadfence();
          team_sync();
          if (tt == 0) last_s[team_in] = atomicAdd(&a.done[tile], summed) + summed == s.passes * 4;
          team_sync();
          summed = 0;
          if (last_s[team_in]) {
            __threadfence();
            for (int t = tt >> 5; t < a.T; t += kw) few_add(a, s, t, tile * 128 + (tt & 31) * 4);
          }
        }
      }
    }
  };
  run_phase(std::integral_constant<int, 0>{});
  grid.sync();
  copies_wait<0>();
  run_phase(std::integral_constant<int, 1>{});
  if (!last_adds) {
    grid.sync();
    for (int i = blockIdx.x + gridDim.x * warp; i < a.T * (a.H >> 7); i += gridDim.x * kWarps) {
      const int t = quotient(i, a.H >> 7);
      few_add(a, s, t, (i - t * (a.H >> 7)) * 128 + lane * 4);
    }
  }
}

template <bool FP8>
void launch(const MoeFewArgs& a, cudaStream_t s) {
  MoeFewArgs args = a;
  smem_opt_in(moe_few_kernel<FP8>, kSmem);
  void* params[] = {&args};
  // every CTA waits for the others: a cooperative launch places all of them at once or fails
  const cudaError_t e = cudaLaunchCooperativeKernel(reinterpret_cast<const void*>(moe_few_kernel<FP8>),
                                                    dim3(device_sm_count()), dim3(kThreads), params, kSmem, s);
  if (e != cudaSuccess) throw std::runtime_error(std::string("moe_few: ") + cudaGetErrorString(e));
}

}  // namespace

void moe_few(const MoeFewArgs& a, cudaStream_t s) {
  if (a.T == 0) return;
  if (a.fp8) launch<true>(a, s);
  else launch<false>(a, s);
}

}  // namespace b200
