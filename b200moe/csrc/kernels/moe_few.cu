// A whole MoE layer for a few tokens (a decode step of one request, the nodes of a few
// drafted trees) in one launch:
//
//   logits = bf16(x Wr^T),  p = softmax(logits),  top-k (lowest id wins a tie),
//   w_k = bf16(p_k / sum p),
//   out = sum_k w_k Wd_e ( silu(Wg_e x) * (Wu_e x) ),   e = the token's k-th expert
//
// The grid is launched cooperatively, one CTA per SM, and synchronises twice: after the
// logits and after the experts' hidden rows.
//
// Nearly all the time goes into reading the touched experts' weights once, so the
// kernel is built around that stream.  Four warps (a team) take 32 weight rows of one
// expert -- 16 gate and the 16 up rows beside them, or 32 rows of Wd -- and a quarter of
// K each.  Every warp brings its own weights into its own ring of three 4 KB stages
// with bulk copies that its first lane issues, so nothing but the two grid barriers
// ever drains the stream: a ring is refilled across items, and in front of the second
// barrier with the first rows of Wd.  16 warps x 12 KB keep up to 192 KB per SM in
// flight.  The products are warp-level MMAs with the weights as the 16-row operand and
// up to 16 tokens as columns.  K is permuted alike in both operands so that a lane's
// operand is 16 contiguous weights of a row.  e4m3 becomes bf16 exactly; the block
// scale multiplies the fp32 sum of each 64 weights, so a weight counts as exactly
// q * scale.  Hidden values enter the second product as two bf16 (value and rest),
// 16 bits of each.  The quarters of K are added in order through shared memory.  The
// rows of Wd write fp32 (token, k) slots, and the team that finishes the last expert of
// a block of 32 columns adds the token's slots in the order of the top-k.
//
// Rounding points: the logits and the routing weights are rounded to bf16 (those of the
// model's router), the output once.  Every wait for a copy is bounded (sm100.cuh); after
// one gives up the warps run on without waiting and the status word says so.
#include <cooperative_groups.h>
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

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
constexpr int kTeam = 4;                 // warps of a team, each a part of K
constexpr int kTeams = kWarps / kTeam;
constexpr int kStages = 3, kStageBytes = 4096;

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

constexpr int kRing = kWarps * kStages * kStageBytes;
constexpr int kRed = kRing;                                  // [kWarps][8][32] floats
constexpr int kBars = kRed + kWarps * 8 * 32 * 4;            // [kWarps][kStages]
constexpr int kShared = kBars + kWarps * kStages * 8 + 64;   // Shared
constexpr int kSmem = kShared + (int)sizeof(Shared) + 1024;
static_assert(kSmem <= 232448, "shared memory budget");

__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
               "{%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Two e4m3 -> two bf16, exactly (every e4m3 value is a bf16 value; NaN stays NaN).
__device__ __forceinline__ uint32_t bf16x2_of(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two), __NV_E4M3);
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
  const __nv_bfloat162 b = __floats2bfloat162_rn(f.x, f.y);
  return *reinterpret_cast<const uint32_t*>(&b);
}

// One pass of a team over 32 weight rows of an expert for up to 16 of its tokens.
struct Item {
  int e, block;        // expert; block of 16 hidden units (phase 0) or of 32 outputs (phase 1)
  int first, cnt;      // pairs [first, first + cnt) of the expert-ordered list
};

template <bool FP8>
struct Few {
  static constexpr int KPS = FP8 ? 2 : 1;              // runs of 64 K per stage
  static constexpr int BLOCK = FP8 ? 1024 : 2048;      // 16 rows of one run
  const MoeFewArgs& a;
  const CUtensorMap& m13;
  const CUtensorMap& m2;
  Shared& s;
  uint8_t* ring;                   // this warp's stages
  uint64_t* bars;
  volatile int* abort_flag;
  int lane, part, team, teams;     // part: quarter of K; team: over the grid

  // ------------------------------------------------------------ the stream of items
  // Items of phase 0 (gate and up rows) and phase 1 (rows of Wd); each is a run of passes.
  __device__ __forceinline__ int blocks(int phase) const { return phase ? a.H / 32 : a.I / 16; }
  __device__ __forceinline__ int k_runs(int phase) const { return (phase ? a.I : a.H) / 64; }
  __device__ __forceinline__ int run0(int phase) const { return k_runs(phase) * part / kTeam; }
  __device__ __forceinline__ int run1(int phase) const { return k_runs(phase) * (part + 1) / kTeam; }
  __device__ __forceinline__ int stages(int phase) const { return (run1(phase) - run0(phase) + KPS - 1) / KPS; }

  struct Cursor {
    int phase, i, pass, st;        // item of the phase, pass of 16 tokens, stage; phase 2: over
  };
  __device__ __forceinline__ Item item(const Cursor& c) const {
    Item it;
    int x;
    if (c.phase == 0) {            // an expert's blocks side by side on different SMs
      x = c.i / blocks(0);
      it.block = c.i - x * blocks(0);
    } else {                       // a block's experts together, so its sum is over early
      it.block = c.i / s.n_touched;
      x = c.i - it.block * s.n_touched;
    }
    it.e = s.touched[x];
    it.first = s.start[it.e] + c.pass * 16;
    it.cnt = min(16, s.start[it.e + 1] - it.first);
    return it;
  }
  __device__ __forceinline__ int passes(const Cursor& c) const {
    const int e = s.touched[c.phase == 0 ? c.i / blocks(0) : c.i % s.n_touched];
    return (s.start[e + 1] - s.start[e] + 15) / 16;
  }
  __device__ __forceinline__ bool settle(Cursor& c) const {   // to the first item at or behind c.i; false: over
    while (c.phase < 2 && c.i >= s.n_touched * blocks(c.phase)) {
      ++c.phase;
      c.i = team;
    }
    return c.phase < 2;
  }
  // next stage of this warp in stream order (items in which it has no K are passed over)
  __device__ __forceinline__ bool to_stage(Cursor& c) const {
    while (settle(c)) {
      if (c.st < stages(c.phase)) return true;
      c.st = 0;
      if (++c.pass >= passes(c)) { c.pass = 0; c.i += teams; }
    }
    return false;
  }

  // the copies of one stage (one lane)
  __device__ __forceinline__ void issue(const Cursor& c, int slot) const {
    const Item it = item(c);
    const int k0 = run0(c.phase) + c.st * KPS, n = min(KPS, run1(c.phase) - k0);
    uint8_t* dst = ring + slot * kStageBytes;
    uint64_t* bar = &bars[slot];
    mbar_arrive_expect_tx(bar, n * 2 * BLOCK);
    const int N = c.phase ? a.H : 2 * a.I, K = c.phase ? a.I : a.H;
    const int row0 = c.phase ? it.block * 32 : it.block * 16, row1 = c.phase ? row0 + 16 : a.I + row0;
    for (int k = 0; k < n; ++k) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int row = b ? row1 : row0;
        uint8_t* d = dst + (k * 2 + b) * BLOCK;
        if (FP8 && a.tiled) {
          const uint8_t* w = static_cast<const uint8_t*>(c.phase ? a.w2 : a.w13);
          bulk_load(d, w + (((int64_t)it.e * (N >> 7) + (row >> 7)) * (K >> 6) + k0 + k) * 8192 + (row & 127) * 64, BLOCK, bar);
        } else {
          tma_load_2d(d, c.phase ? &m2 : &m13, bar, (k0 + k) * 64, it.e * N + row);
        }
      }
    }
  }

  // ------------------------------------------------------------ products
  // acc[m][n] += 16 rows x 8 tokens of this warp's K; B: bf16 rows of K elements, `planes` of them
  // (value and rest) `plane` elements apart.
  template <int NT, int PLANES, typename Load>
  __device__ __forceinline__ void stage_mma(const Cursor& c, const Item& it, int slot, uint32_t parity, float (&acc)[2][NT][4],
                                            const bf16* const (&rows)[NT], int64_t plane, Load load) {
    const int k0 = run0(c.phase) + c.st * KPS, n = min(KPS, run1(c.phase) - k0);
    const int g = lane >> 2, t = lane & 3;
    uint4 b[KPS][NT][PLANES][2];
#pragma unroll
    for (int k = 0; k < KPS; ++k)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int p = 0; p < PLANES; ++p)
#pragma unroll
          for (int v = 0; v < 2; ++v)
            b[k][j][p][v] = k < n && rows[j] != nullptr ? load(rows[j] + p * plane + (k0 + k) * 64 + t * 16 + v * 8)
                                                        : make_uint4(0, 0, 0, 0);
    float sc[KPS][2];
    if constexpr (FP8) {
      const int N = c.phase ? a.H : 2 * a.I, kb = (c.phase ? a.I : a.H) / 128;
      const int row0 = c.phase ? it.block * 32 : it.block * 16, row1 = c.phase ? row0 + 16 : a.I + row0;
      const float* sp = (c.phase ? a.s2 : a.s13) + (int64_t)it.e * (N / 128) * kb;
#pragma unroll
      for (int k = 0; k < KPS; ++k) {
        const int at = min(k0 + k, k_runs(c.phase) - 1) >> 1;
        sc[k][0] = __ldg(sp + (row0 >> 7) * kb + at);
        sc[k][1] = __ldg(sp + (row1 >> 7) * kb + at);
      }
    }
    mbar_wait(&bars[slot], parity, a.status, kStatusTimeoutFull, abort_flag);
    const uint8_t* src = ring + slot * kStageBytes;
#pragma unroll
    for (int k = 0; k < KPS; ++k) {
      if (k >= n) break;
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const uint8_t* blk = src + (k * 2 + m) * BLOCK;
        float part_acc[NT][4];
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) part_acc[j][i] = 0.f;
        uint4 w[2][FP8 ? 1 : 2];     // rows g and g + 8: 16 weights
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int row = g + 8 * r;
          if constexpr (FP8) {
            w[r][0] = *reinterpret_cast<const uint4*>(blk + row * 64 + ((t ^ ((row >> 1) & 3)) << 4));
          } else {
#pragma unroll
            for (int v = 0; v < 2; ++v)
              w[r][v] = *reinterpret_cast<const uint4*>(blk + row * 128 + (((2 * t + v) ^ (row & 7)) << 4));
          }
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {   // 16 of the 64 K: weights 4 q .. 4 q + 3 of each lane's 16
          uint32_t af[4];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            if constexpr (FP8) {
              const uint32_t x = q == 0 ? w[r][0].x : q == 1 ? w[r][0].y : q == 2 ? w[r][0].z : w[r][0].w;
              af[r] = bf16x2_of(x & 0xffffu);
              af[r + 2] = bf16x2_of(x >> 16);
            } else {
              const uint4& x = w[r][q >> 1];
              af[r] = q & 1 ? x.z : x.x;
              af[r + 2] = q & 1 ? x.w : x.y;
            }
          }
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int p = 0; p < PLANES; ++p) {
              const uint4& x = b[k][j][p][q >> 1];
              mma_bf16(part_acc[j], af, q & 1 ? x.z : x.x, q & 1 ? x.w : x.y);
            }
        }
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if constexpr (FP8) acc[m][j][i] = fmaf(part_acc[j][i], sc[k][m], acc[m][j][i]);
            else acc[m][j][i] += part_acc[j][i];
          }
      }
    }
  }
};

template <bool FP8>
__global__ void __launch_bounds__(kThreads, 1)
moe_few_kernel(const __grid_constant__ CUtensorMap m13, const __grid_constant__ CUtensorMap m2, const MoeFewArgs a) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Shared& s = *reinterpret_cast<Shared*>(smem + kShared);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + kBars + kWarps * kStages * 8);
  int* last_s = reinterpret_cast<int*>(smem + kBars + kWarps * kStages * 8 + 4);   // [kTeams]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int team_in = warp / kTeam, tt = threadIdx.x % (kTeam * 32);
  cg::grid_group grid = cg::this_grid();
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kBars) + warp * kStages;
  if (lane == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(&bars[i], 1);
    if (warp == 0) *abort_flag = 0;
    fence_barrier_init();
  }
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < a.H / 32; i += kThreads) a.done[i] = 0;
  few_logits(a);
  grid.sync();
  few_route(a, s);

  Few<FP8> few{a, m13, m2, s, smem + warp * kStages * kStageBytes, bars, abort_flag, lane, warp % kTeam,
               team_in * (int)gridDim.x + (int)blockIdx.x, kTeams * (int)gridDim.x};
  using Cursor = typename Few<FP8>::Cursor;
  Cursor ahead{0, few.team, 0, 0}, at{0, few.team, 0, 0};
  int issued = 0, used = 0;
  auto refill = [&]() {   // keep the ring full, across items and phases
    while (issued < used + kStages && few.to_stage(ahead)) {
      if (lane == 0 && !*abort_flag) few.issue(ahead, issued % kStages);
      ++issued;
      ++ahead.st;
    }
  };
  refill();

  float* red = reinterpret_cast<float*>(smem + kRed) + team_in * (kTeam * 256);   // [kTeam][8][32]
  bf16* hid = static_cast<bf16*>(a.h);
  const int64_t hplane = (int64_t)a.T * a.topk * a.I;
  const int g = lane >> 2;

  auto run_phase = [&](auto phase_c) {
    constexpr int P = decltype(phase_c)::value;
    while (few.settle(at) && at.phase == P) {
      const Item it = few.item(at);
      auto pass = [&](auto nt_c) {
        constexpr int NT = decltype(nt_c)::value;
        float acc[2][NT][4];
        const bf16* rows[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
#pragma unroll
          for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[m][j][i] = 0.f;
          const int n = j * 8 + g;
          rows[j] = nullptr;
          if (n < it.cnt) {
            const int p = s.pair[it.first + n];
            rows[j] = P ? hid + (int64_t)p * a.I : static_cast<const bf16*>(a.x) + (int64_t)(p / a.topk) * a.H;
          }
        }
        for (at.st = 0; at.st < few.stages(P); ++at.st) {
          const int slot = used % kStages;
          const uint32_t parity = (used / kStages) & 1;
          if constexpr (P == 0)
            few.template stage_mma<NT, 1>(at, it, slot, parity, acc, rows, 0,
                                          [](const bf16* p) { return __ldg(reinterpret_cast<const uint4*>(p)); });
          else
            few.template stage_mma<NT, 2>(at, it, slot, parity, acc, rows, hplane,
                                          [](const bf16* p) { return __ldcg(reinterpret_cast<const uint4*>(p)); });
          __syncwarp();
          ++used;
          refill();
        }
        at.st = 0;
        // the quarters of K, added in order: thread = (accumulator register, lane)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          named_barrier_sync(1 + team_in, kTeam * 32);    // the last sums have been read
#pragma unroll
          for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) red[(warp % kTeam) * 256 + (m * 4 + i) * 32 + lane] = acc[m][j][i];
          named_barrier_sync(1 + team_in, kTeam * 32);
          const int i = tt >> 5, l = tt & 31;
          float v[2];
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            v[m] = 0.f;
#pragma unroll
            for (int q = 0; q < kTeam; ++q) v[m] += red[q * 256 + (m * 4 + i) * 32 + l];
          }
          const int n = j * 8 + (l & 3) * 2 + (i & 1), row = (l >> 2) + 8 * (i >> 1);
          if (n < it.cnt) {
            const int64_t p = s.pair[it.first + n];
            if constexpr (P == 0) {
              const float hv = v[0] / (1.f + expf(-v[0])) * v[1];
              const bf16 top = __float2bfloat16(hv);
              bf16* dst = hid + p * a.I + it.block * 16 + row;
              dst[0] = top;
              dst[hplane] = __float2bfloat16(hv - __bfloat162float(top));
            } else {
              float* dst = a.slots + p * a.H + it.block * 32 + row;
              dst[0] = v[0];
              dst[16] = v[1];
            }
          }
        }
      };
      if (it.cnt <= 8) pass(std::integral_constant<int, 1>{});
      else pass(std::integral_constant<int, 2>{});
      const bool over = at.pass + 1 >= few.passes(at);
      if constexpr (P == 1) {
        if (over) {
          // the team that brings a block's last expert adds the slots of every token
          __threadfence();
          named_barrier_sync(1 + team_in, kTeam * 32);
          if (tt == 0) last_s[team_in] = atomicAdd(&a.done[it.block], 1) == s.n_touched - 1;
          named_barrier_sync(1 + team_in, kTeam * 32);
          if (last_s[team_in]) {
            __threadfence();
            const int c = it.block * 32 + (tt & 7) * 4;
            for (int t = tt >> 3; t < a.T; t += kTeam * 4) {
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
          }
        }
      }
      if (over) { at.pass = 0; at.i += few.teams; } else { ++at.pass; }
    }
  };
  run_phase(std::integral_constant<int, 0>{});
  grid.sync();
  run_phase(std::integral_constant<int, 1>{});
  if (*abort_flag) {
    // a wait gave up: let the copies already issued land before the CTA exits
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 1000000ull) __nanosleep(1000);
  }
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    cudaDriverEntryPointQueryResult q;
    void* p = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess || p == nullptr)
      throw std::runtime_error("cuTensorMapEncodeTiled entry point not available");
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }();
  return fn;
}

// Row-major weights [rows, K]: boxes of 64 K x 16 rows, in the swizzle the lanes read without
// bank conflicts (64-byte rows for e4m3, 128-byte rows for bf16).
void weight_map(CUtensorMap* map, const void* w, bool fp8, int64_t rows, int K) {
  const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)K * (fp8 ? 1 : 2)};
  const cuuint32_t box[2] = {64, 16}, estr[2] = {1, 1};
  const CUresult r = encode_fn()(map, fp8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
                                 const_cast<void*>(w), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                 fp8 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                                 CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) throw std::runtime_error("moe_few weight map: encode failed " + std::to_string((int)r));
}

template <bool FP8>
void launch(const MoeFewArgs& a, cudaStream_t s) {
  MoeFewArgs args = a;
  CUtensorMap m13{}, m2{};
  if (!(FP8 && a.tiled)) {
    weight_map(&m13, a.w13, FP8, (int64_t)a.E * 2 * a.I, a.H);
    weight_map(&m2, a.w2, FP8, (int64_t)a.E * a.H, a.I);
  }
  smem_opt_in(moe_few_kernel<FP8>, kSmem);
  void* params[] = {&m13, &m2, &args};
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
