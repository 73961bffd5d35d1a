// Attention of drafted trees on the 5th-generation tensor cores (bf16 pool, head_dim 64
// or 128): the same function as tree_attn.cu, for the shapes a server runs.
//
// Rows and keys.  The n nodes of a sequence times the G query heads of one KV head are
// packed into tiles of 128 rows (row = node * G + head), keys into tiles of 128.  A
// unit of work is one key tile against one pair of row tiles:
//
//   two row tiles (n * G > 128)   softmax group w of the CTA takes row tile w,
//   one row tile                  the groups take alternate key tiles and their two
//                                 results are joined in the epilogue,
//
// so both groups work on either shape and a K/V tile is read once for up to 256 rows.
//
// Split.  Units are ordered (sequence, KV head, key chunk, row pair, key tile), and
// CTA c of the persistent grid takes the c-th of equal shares of that order: long
// contexts, few requests and ragged batches all fill every SM, without the host
// knowing a length.  A chunk is at least a share long and is the same for all row pairs
// of a KV head, so the CTAs that read the same keys do so at about the same time and
// the L2 serves all but the first.  A share that cuts an item leaves an unnormalised
// fp32 result with its running maximum and sum; after a grid-wide barrier the warps
// join those (softmax over the parts).
//
// Roles per CTA (12 warps): a TMA producer; two MMA issuers, one per softmax group
// (S = Q K^T, then O += P V with P read from TMEM, where it overlays its S); a cleaner
// of the last V tiles; two softmax groups of four warps, a thread per row, so the row
// statistics need no shuffles.  The running maximum moves only when a row grows by
// more than 2^8, so O is rarely rescaled.  P is rounded to bf16 for the MMA and the sum
// that divides O adds the rounded values, which cancels that rounding where few keys
// carry the weight.
//
// A masked place never reaches the result: scores are selected, not added to, and a V
// row is cleaned in front of the MMA (0 * NaN is NaN) -- rows behind the sequence become
// zero, and where a node's V is not finite those elements become zero and are added back
// for the rows that see the node.
//
// Every wait is bounded (sm100.cuh).  The grid is launched cooperatively because its
// CTAs wait for one another once.
#include <cooperative_groups.h>
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <cstdint>
#include <stdexcept>
#include <string>

#include "pdl.cuh"
#include "sm100.cuh"
#include "tree.h"

namespace b200 {
namespace {

namespace cg = cooperative_groups;
using bf16 = __nv_bfloat16;

constexpr int kRows = 128, kKeys = 128;
constexpr int kThreads = 384;
constexpr float kLazyLog2 = 8.f;
constexpr int kAncWords = kTreeMaxNodes / 32;
constexpr int kDirtyBufs = 4;

template <int D>
struct Lay {
  static constexpr int TILE = kKeys * D * 2;       // a K, V or Q tile: D / 64 halves of [128][64]
  static constexpr int HALF = kKeys * 64 * 2;
  static constexpr int SLOTS = D == 128 ? 2 : 4;   // K tiles, and V tiles, in flight
  static constexpr int Q = 0;                      // two row tiles
  static constexpr int K = Q + 2 * TILE;
  static constexpr int V = K + SLOTS * TILE;
  static constexpr int STAGE = V + SLOTS * TILE;   // join of the two groups: 2 x [4][128] float4
  static constexpr int ANC = STAGE + 2 * 8192;     // [nodes][kAncWords] ancestor bits
  static constexpr int PAR = ANC + kTreeMaxNodes * kAncWords * 4;
  static constexpr int ML = PAR + kTreeMaxNodes * 4;          // [2][128] (max, sum)
  static constexpr int DIRTY = ML + 2 * kRows * 8;
  static constexpr int BARS = DIRTY + kDirtyBufs * kAncWords * 4;
  static constexpr int NBARS = 5 * SLOTS + 2 + 6 + 3;
  static constexpr int PU = BARS + NBARS * 8 + 16;            // [batch + 1] units before a sequence
  static int smem(int batch) { return PU + (batch + 1) * 4 + 1024; }
};

struct TcArgs {
  TreeAttnArgs a;
  float* part_o;     // [grid][2][part_rows][D]
  float2* part_ml;   // [grid][2][part_rows]
  int part_rows;     // 128 or 256
  int sub_rows;
};

__device__ __forceinline__ uint32_t sw_off(int r, int u) { return r * 128 + ((u ^ (r & 7)) << 4); }

__device__ __forceinline__ void tma_4d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// MN-major operand in 128-byte swizzle: rows = K index, 64 contiguous elements each;
// lbo = bytes between 64-wide chunks, 1024 bytes between groups of 8 rows.
__device__ __forceinline__ uint64_t sdesc_mn(uint32_t addr, uint32_t lbo) {
  return umma_sdesc_sw128(addr) & ~(uint64_t(0x3FFF) << 16) | (uint64_t((lbo >> 4) & 0x3FFFu) << 16);
}

template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t addr, float* v);
template <>
__device__ __forceinline__ void tmem_ld<32>(uint32_t addr, float* v) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Key chunks of a sequence with nt key tiles, [start(i), start(i + 1)): at least `share` tiles each
// (one chunk where the sequence is shorter), so a CTA's share never holds a chunk strictly inside.
struct Chunks {
  int n, nt;
  __device__ __forceinline__ int start(int i) const { return (int)((int64_t)i * nt / n); }
  __device__ __forceinline__ int of(int tile) const { return (int)(((int64_t)(tile + 1) * n - 1) / nt); }
};
__device__ __forceinline__ Chunks chunks_of(int nt, int pairs, int share) {
  return {pairs == 1 || nt <= share ? 1 : nt / share, nt};
}

// What a sequence adds to the order of units.
struct Seq {
  int q0, n, len;      // first row, nodes, keys
  int nt, pairs;       // key tiles, pairs of row tiles
};
__device__ __forceinline__ Seq seq_of(const TreeAttnArgs& a, int b) {
  Seq s;
  s.q0 = a.cu_seqlens_q[b];
  s.n = a.cu_seqlens_q[b + 1] - s.q0;
  s.len = a.seq_lens[b];
  s.nt = (s.len + kKeys - 1) / kKeys;
  const int per = kRows / a.group;  // nodes per row tile
  s.pairs = ((s.n + per - 1) / per + 1) / 2;
  return s;
}

// A run of key tiles [t0, t1) of one item (sequence, KV head, row pair) inside a CTA's share.
struct Seg {
  Seq s;
  int b, h, pair, t0, t1;
  int two;             // two row tiles
  int whole;           // covers all of the item's keys
  int next;            // first unit behind it
};
__device__ __forceinline__ Seg seg_at(const TreeAttnArgs& a, const int* pu, int share, int u, int hi) {
  Seg g;
  int lo = 0, up = a.batch;
  while (up - lo > 1) {
    const int mid = (lo + up) >> 1;
    if (pu[mid] <= u) lo = mid; else up = mid;
  }
  g.b = lo;
  g.s = seq_of(a, lo);
  int r = u - pu[lo];
  const int per_head = g.s.nt * g.s.pairs;
  g.h = r / per_head;
  r -= g.h * per_head;
  const Chunks c = chunks_of(g.s.nt, g.s.pairs, share);
  const int ci = c.of(r / g.s.pairs), start = c.start(ci), end = c.start(ci + 1), clen = end - start;
  r -= start * g.s.pairs;
  g.pair = r / clen;
  g.t0 = start + r % clen;
  g.t1 = min(end, g.t0 + (hi - u));
  g.next = u + (g.t1 - g.t0);
  g.whole = g.t0 == 0 && g.t1 == g.s.nt;
  const int per = kRows / a.group;
  g.two = g.s.n > (2 * g.pair + 1) * per;
  return g;
}

// CTA c's share of W units.
__device__ __forceinline__ int share_lo(int c, int W, int grid) { return (int)((int64_t)c * W / grid); }

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
tree_attn_tc_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                    const __grid_constant__ CUtensorMap q_map, const TcArgs t) {
  using L = Lay<D>;
  constexpr int kHalves = D / 64, kSlots = L::SLOTS;
  const TreeAttnArgs& a = t.a;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + L::BARS);
  uint64_t* k_empty = k_full + kSlots;
  uint64_t* v_full = k_empty + kSlots;    // landed
  uint64_t* v_ready = v_full + kSlots;    // cleaned where it had to be
  uint64_t* v_empty = v_ready + kSlots;
  uint64_t* q_full = v_empty + kSlots;
  uint64_t* q_empty = q_full + 1;
  uint64_t* s_full = q_empty + 1;         // [2] per softmax group
  uint64_t* p_full = s_full + 2;
  uint64_t* pv_done = p_full + 2;
  uint64_t* fin = pv_done + 2;            // [2] an issuer's last products
  uint64_t* both = fin + 2;               // the eight softmax warps
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(both + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* s_max_nt = reinterpret_cast<int*>(tmem_slot + 2);
  int* pu = reinterpret_cast<int*>(smem + L::PU);
  uint32_t* anc = reinterpret_cast<uint32_t*>(smem + L::ANC);
  int* s_par = reinterpret_cast<int*>(smem + L::PAR);
  float2* s_ml = reinterpret_cast<float2*>(smem + L::ML);
  uint32_t* dirty = reinterpret_cast<uint32_t*>(smem + L::DIRTY);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = a.group, per = kRows / G;   // nodes per row tile
  int* status = a.status;

  // ---- units before each sequence; a tree that does not fit counts none
  if (threadIdx.x == 0) *s_max_nt = 0;
  __syncthreads();
  for (int b = threadIdx.x; b < a.batch; b += kThreads) {
    const Seq s = seq_of(a, b);
    const bool bad = s.n < 0 || s.n > a.max_q_len || s.q0 < 0 || s.q0 + s.n > a.rows ||
                     (s.n > 0 && (s.len < s.n || s.len > (int64_t)a.max_blocks * a.block_size));
    if (bad && blockIdx.x == 0) record_status(status, kStatusBadShape);
    const bool none = bad || s.n == 0;
    pu[b + 1] = none ? 0 : s.nt * s.pairs * a.num_kv_heads;
    if (!none) atomicMax(s_max_nt, s.nt);
  }
  if (threadIdx.x == 32) {
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 2);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_ready[i], 1);
      mbar_init(&v_empty[i], 2);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 2);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&pv_done[i], 1);
      mbar_init(&fin[i], 1);
    }
    mbar_init(both, 8);
    fence_barrier_init();
    *abort_flag = 0;
  }
  __syncthreads();
  if (warp == 0) {
    int at = 0;
    if (lane == 0) pu[0] = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 32) {
      const int b = b0 + lane;
      int v = b < a.batch ? pu[b + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += up;
      }
      if (b < a.batch) pu[b + 1] = at + v;
      at += __shfl_sync(0xffffffffu, v, 31);
    }
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;   // S0 | S1 | O0 | O1, 128 columns each
  const int W = pu[a.batch];
  const int grid = gridDim.x;
  const int share = (W + grid - 1) / grid;
  const int u_lo = share_lo(blockIdx.x, W, grid), u_hi = share_lo(blockIdx.x + 1, W, grid);

  if (warp == 0) {
    // ================================================================ TMA producer
    if (lane == 0) {
      tma_prefetch_desc(&k_map);
      tma_prefetch_desc(&v_map);
      tma_prefetch_desc(&q_map);
      const int nsub = kKeys / t.sub_rows;
      int gt = 0, sg = 0;   // tiles, segments
      bool ok = true, bad = false;
      for (int u = u_lo; u < u_hi && ok; ++sg) {
        const Seg g = seg_at(a, pu, share, u, u_hi);
        u = g.next;
        if (!mbar_wait(q_empty, (sg & 1) ^ 1, status, kStatusTimeoutEmpty, abort_flag)) break;
        const int tiles = g.two ? 2 : 1;
        mbar_arrive_expect_tx(q_full, tiles * kHalves * per * G * 128);
        for (int i = 0; i < tiles; ++i)
#pragma unroll
          for (int hf = 0; hf < kHalves; ++hf)
            tma_3d(smem_u32(smem + L::Q + i * L::TILE + hf * L::HALF), &q_map, q_full, hf * 64, g.h * G,
                   g.s.q0 + (2 * g.pair + i) * per);
        const int* tab = a.block_tables + (int64_t)g.b * a.max_blocks;
        for (int j = g.t0; j < g.t1 && ok; ++j, ++gt) {
          const int slot = gt % kSlots;
          const uint32_t ph = (gt / kSlots) & 1;
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            uint64_t* full = kv ? &v_full[slot] : &k_full[slot];
            if (!mbar_wait(kv ? &v_empty[slot] : &k_empty[slot], ph ^ 1, status, kStatusTimeoutEmpty, abort_flag)) {
              ok = false;
              break;
            }
            mbar_arrive_expect_tx(full, L::TILE);
            const uint32_t dst = smem_u32(smem + (kv ? L::V : L::K) + slot * L::TILE);
            for (int sub = 0; sub < nsub; ++sub) {
              const int key = j * kKeys + sub * t.sub_rows;
              int blk = a.num_blocks;      // out of range: zero fill
              if (key < g.s.len) {
                const int bi = key / a.block_size;
                const int id = bi < a.max_blocks ? tab[bi] : -1;
                if (id >= 0 && id < a.num_blocks) blk = id;
                else bad = true;
              }
#pragma unroll
              for (int hf = 0; hf < kHalves; ++hf)
                tma_4d(dst + hf * L::HALF + sub * t.sub_rows * 128, kv ? &v_map : &k_map, full, hf * 64,
                       key % a.block_size, g.h, blk);
            }
          }
        }
      }
      if (bad) record_status(status, kStatusBadShape);
      if (*abort_flag) {
        // a wait gave up: let the copies already issued land before the CTA exits
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 1000000ull) __nanosleep(1000);
      }
    }
    __syncwarp();
  } else if (warp <= 2) {
    // ================================================================ MMA issuer of group w
    if (lane == 0) {
      const int w = warp - 1;
      const uint32_t idesc_s = umma_idesc_bf16(kRows, kKeys);
      const uint32_t idesc_pv = umma_idesc_bf16(kRows, D) | (1u << 16);  // B (V) is MN-major
      const uint32_t tS = tmem + w * 128, tO = tmem + 256 + w * 128;
      int gt = 0, sg = 0, mine = 0;   // tiles of the CTA, segments, tiles of this group
      bool ok = true;
      for (int u = u_lo; u < u_hi && ok; ++sg) {
        const Seg g = seg_at(a, pu, share, u, u_hi);
        u = g.next;
        if (!mbar_wait(q_full, sg & 1, status, kStatusTimeoutFull, abort_flag)) { ok = false; break; }
        const uint32_t qa = smem_u32(smem + L::Q + (g.two ? w : 0) * L::TILE);
        bool first = true;
        for (int j = g.t0; j < g.t1; ++j, ++gt) {
          if (!g.two && (gt & 1) != w) continue;
          const int slot = gt % kSlots;
          const uint32_t ph = (gt / kSlots) & 1;
          // S overlays the group's last P: that product has to be done
          if (mine > 0 && !mbar_wait(&pv_done[w], (mine - 1) & 1, status, kStatusTimeoutAccEmpty, abort_flag)) { ok = false; break; }
          if (!mbar_wait(&k_full[slot], ph, status, kStatusTimeoutFull, abort_flag)) { ok = false; break; }
          tc_fence_after();
          const uint32_t kb = smem_u32(smem + L::K + slot * L::TILE);
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t off = (k >> 2) * L::HALF + (k & 3) * 32;
            umma_f16_ss(tS, umma_sdesc_sw128(qa + off), umma_sdesc_sw128(kb + off), idesc_s, k > 0 ? 1u : 0u);
          }
          umma_commit(&s_full[w]);
          umma_commit(&k_empty[slot]);
          if (!g.two) umma_commit(&k_empty[slot]);   // the other group does not read this tile
          if (!mbar_wait(&p_full[w], mine & 1, status, kStatusTimeoutConv, abort_flag)) { ok = false; break; }
          if (!mbar_wait(&v_ready[slot], ph, status, kStatusTimeoutFull, abort_flag)) { ok = false; break; }
          tc_fence_after();
          const uint32_t vb = smem_u32(smem + L::V + slot * L::TILE);
#pragma unroll
          for (int k = 0; k < kKeys / 16; ++k)
            umma_f16_ts(tO, tS + k * 8, sdesc_mn(vb + k * 16 * 128, L::HALF), idesc_pv, (!first || k > 0) ? 1u : 0u);
          umma_commit(&pv_done[w]);
          umma_commit(&v_empty[slot]);
          if (!g.two) umma_commit(&v_empty[slot]);
          first = false;
          ++mine;
        }
        if (!ok) break;
        // the segment's products are done (its Q, and every K and V phase before the next)
        umma_commit(q_empty);
      }
      // every product issued so far ends before TMEM is released
      umma_commit(&fin[w]);
      mbar_wait(&fin[w], 0, status, kStatusTimeoutAccEmpty, nullptr);
    }
    __syncwarp();
  } else if (warp == 3) {
    // ================================================================ V cleaner
    int gt = 0, sg = 0;
    bool ok = true;
    for (int u = u_lo; u < u_hi && ok; ++sg) {
      const Seg g = seg_at(a, pu, share, u, u_hi);
      u = g.next;
      uint32_t* dirt = dirty + (sg % kDirtyBufs) * kAncWords;
      if (lane < kAncWords) dirt[lane] = 0;
      __syncwarp();
      const int prefix = g.s.len - g.s.n;
      for (int j = g.t0; j < g.t1; ++j, ++gt) {
        const int slot = gt % kSlots;
        ok = mbar_wait(&v_full[slot], (gt / kSlots) & 1, status, kStatusTimeoutFull, abort_flag);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        if ((j + 1) * kKeys > prefix) {
          uint8_t* vt = smem + L::V + slot * L::TILE;
          for (int r = lane; r < kKeys; r += 32) {
            const int node = j * kKeys + r - prefix;
            if (node < 0) continue;
            const bool behind = node >= g.s.n;
            bool bad = false;
#pragma unroll 1
            for (int c = 0; c < D / 8; ++c) {
              uint4* p = reinterpret_cast<uint4*>(vt + (c >> 3) * L::HALF + sw_off(r, c & 7));
              if (behind) {
                *p = make_uint4(0, 0, 0, 0);
                continue;
              }
              const uint4 v = *p;
              uint32_t e[4] = {v.x, v.y, v.z, v.w};
              bool hit = false;
#pragma unroll
              for (int i = 0; i < 4; ++i) {   // all exponent bits set: infinite or NaN
                if ((e[i] & 0x7f80u) == 0x7f80u) { e[i] &= 0xffff0000u; hit = true; }
                if ((e[i] & 0x7f800000u) == 0x7f800000u) { e[i] &= 0xffffu; hit = true; }
              }
              if (hit) { *p = make_uint4(e[0], e[1], e[2], e[3]); bad = true; }
            }
            if (bad) atomicOr(&dirt[node >> 5], 1u << (node & 31));
          }
          fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_ready[slot]);
      }
    }
  } else {
    // ================================================================ softmax group w
    const int w = (warp - 4) >> 2;
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const int tid = threadIdx.x - 128;        // over both groups
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const uint32_t tS = tmem + w * 128 + lane_base, tO = tmem + 256 + w * 128 + lane_base;
    const float sl2 = a.scale * 1.4426950408889634f;
    const int nq = a.num_kv_heads * G;
    int gt = 0, sg = 0, mine = 0, seen_b = -1, syncs = 0;
    bool ok = true;
    // both groups meet; false once a wait has given up somewhere (bounded, unlike bar.sync)
    auto meet = [&]() {
      __syncwarp();
      if (lane == 0) mbar_arrive(both);
      const bool here = mbar_wait(both, syncs++ & 1, status, kStatusTimeoutFlag, abort_flag);
      return __all_sync(0xffffffffu, here) != 0;
    };
    for (int u = u_lo; u < u_hi && ok; ++sg) {
      const Seg g = seg_at(a, pu, share, u, u_hi);
      const int slot_id = u == u_lo ? 0 : 1;
      u = g.next;
      const int prefix = g.s.len - g.s.n;
      if (g.b != seen_b) {
        // ancestor bits of the sequence's nodes, by walking the parents in shared memory
        if (!meet()) break;
        for (int i = tid; i < g.s.n; i += 256) s_par[i] = a.parents[g.s.q0 + i];
        for (int i = tid; i < g.s.n * kAncWords; i += 256) anc[i] = 0;
        if (!meet()) break;
        for (int i = tid; i < g.s.n; i += 256) {
          for (int at = i; at >= 0;) {          // a parent that is not in front of its child ends the walk
            anc[i * kAncWords + (at >> 5)] |= 1u << (at & 31);
            const int up = s_par[at];
            at = up < at ? up : -1;
          }
        }
        if (!meet()) break;
        seen_b = g.b;
      }
      const int tile = 2 * g.pair + (g.two ? w : 0);
      const int node = tile * per + r / G, head = g.h * G + r % G;
      const bool valid = r < per * G && node < g.s.n;
      const bool any = __any_sync(0xffffffffu, valid);
      float m = -INFINITY, l = 0.f;
      int done = 0;                              // tiles of this group in the segment
      for (int j = g.t0; j < g.t1; ++j, ++gt) {
        if (!g.two && (gt & 1) != w) continue;
        ok = mbar_wait(&s_full[w], mine & 1, status, kStatusTimeoutAccFull, abort_flag);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        tc_fence_after();
        if (any) {
          float s[kKeys];
#pragma unroll
          for (int c = 0; c < kKeys / 32; ++c) tmem_ld<32>(tS + c * 32, s + c * 32);
          tmem_ld_wait();
          const int kb = j * kKeys;
          if (kb + kKeys > prefix) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const int t0 = kb + q * 32 - prefix;        // node of the word's first column
              uint32_t see = t0 >= 0 ? 0u : t0 <= -32 ? 0xffffffffu : (1u << -t0) - 1u;
              if (t0 > -32 && valid) {
                const int i = t0 >> 5;
                const uint32_t* row = anc + node * kAncWords;
                const uint32_t lo = i >= 0 && i < kAncWords ? row[i] : 0u;
                const uint32_t up = i + 1 < kAncWords ? row[i + 1] : 0u;
                see |= __funnelshift_r(lo, up, t0 & 31);
              }
#pragma unroll
              for (int c = 0; c < 32; ++c)
                if (!((see >> c) & 1u)) s[q * 32 + c] = -INFINITY;
            }
          }
          float mx = fmaxf(s[0], s[1]);
#pragma unroll
          for (int c = 2; c < kKeys; ++c) mx = fmaxf(mx, s[c]);
          mx *= sl2;
          const bool grow = mx > m + kLazyLog2;
          if (__any_sync(0xffffffffu, grow)) {
            float alpha = 1.f;
            if (grow) {
              alpha = m == -INFINITY ? 1.f : ex2(m - mx);
              m = mx;
              l *= alpha;
            }
            if (done > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll 1
              for (int c = 0; c < D / 16; ++c) {
                float o[16];
                tmem_ld16(tO + c * 16, o);
                tmem_ld_wait();
                uint32_t ou[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) ou[i] = __float_as_uint(o[i] * alpha);
                tmem_st16(tO + c * 16, ou);
              }
            }
          }
          const float mu = m == -INFINITY ? 0.f : m;
          float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
          for (int c = 0; c < kKeys / 32; ++c) {
            uint32_t p[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              p[i] = pack2(ex2(fmaf(s[c * 32 + 2 * i], sl2, -mu)), ex2(fmaf(s[c * 32 + 2 * i + 1], sl2, -mu)));
              sum0 += __uint_as_float(p[i] << 16);
              sum1 += __uint_as_float(p[i] & 0xffff0000u);
            }
            tmem_st16(tS + c * 16, p);
          }
          l += sum0 + sum1;
          tmem_st_wait();
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[w]);
        ++mine;
        ++done;
      }
      if (!ok) break;
      // ---------------------------------------------------------------- epilogue
      const bool join = !g.two && g.t1 - g.t0 > 1;   // both groups hold a part of every row
      if (done > 0) {
        ok = mbar_wait(&pv_done[w], (mine - 1) & 1, status, kStatusTimeoutAccEmpty, abort_flag);
        if (!__all_sync(0xffffffffu, ok)) break;
        tc_fence_after();
      }
      float fac = 1.f;
      if (join) {
        s_ml[w * kRows + r] = make_float2(m, l);
        if (!meet()) break;
        const float2 other = s_ml[(w ^ 1) * kRows + r];
        const float top = fmaxf(m, other.x);
        fac = m == -INFINITY ? 0.f : ex2(m - top);
        const float ofac = other.x == -INFINITY ? 0.f : ex2(other.x - top);
        l = l * fac + other.y * ofac;
        m = top;
      }
      // columns this thread writes: all of its row, or its half of a joined row
      const int c0 = join ? w * (D / 32) : 0, c1 = join ? (w + 1) * (D / 32) : done > 0 ? D / 16 : 0;
      const float inv = l > 0.f ? 1.f / l : 0.f;
      const int prow = (g.two ? w : 0) * kRows + r;
      const int64_t pslot = (int64_t)(blockIdx.x * 2 + slot_id) * t.part_rows + prow;
      if (!g.whole && valid && c1 > 0 && (!join || w == 0)) t.part_ml[pslot] = make_float2(m, l);
      const uint32_t* dirt = dirty + (sg % kDirtyBufs) * kAncWords;
      bool dirt_any = false;
#pragma unroll
      for (int i = 0; i < kAncWords; ++i) dirt_any |= dirt[i] != 0;
      float4* stage = reinterpret_cast<float4*>(smem + L::STAGE);
#pragma unroll 1
      for (int i = 0; i < D / 16; ++i) {
        if (join && i >= D / 32) break;
        float o[16];
        if (join) {
          // hand the other group its columns of this row, take this group's columns of the other part
          tmem_ld16(tO + ((w ^ 1) * (D / 32) + i) * 16, o);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 4; ++e)
            stage[w * 512 + e * 128 + r] = make_float4(o[4 * e] * fac, o[4 * e + 1] * fac, o[4 * e + 2] * fac, o[4 * e + 3] * fac);
          if (!(ok = meet())) break;
        }
        if (c0 + i < c1) {
          tmem_ld16(tO + (c0 + i) * 16, o);
          tmem_ld_wait();
          if (join) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float4 v = stage[(w ^ 1) * 512 + e * 128 + r];
              o[4 * e] = o[4 * e] * fac + v.x;
              o[4 * e + 1] = o[4 * e + 1] * fac + v.y;
              o[4 * e + 2] = o[4 * e + 2] * fac + v.z;
              o[4 * e + 3] = o[4 * e + 3] * fac + v.w;
            }
          }
          if (valid) {
            if (dirt_any) {
              // V elements that were not finite count for the rows that see their node
              for (int d = 0; d < g.s.n; ++d) {
                if (!((dirt[d >> 5] & anc[node * kAncWords + (d >> 5)]) >> (d & 31) & 1u)) continue;
                const int key = prefix + d, id = a.block_tables[(int64_t)g.b * a.max_blocks + key / a.block_size];
                const bf16* v = static_cast<const bf16*>(a.v_cache) + (int64_t)id * a.block_stride +
                                ((int64_t)g.h * a.block_size + key % a.block_size) * D + (c0 + i) * 16;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                  const float x = __bfloat162float(v[e]);
                  if (!isfinite(x)) o[e] += x;
                }
              }
            }
            if (g.whole) {
              uint4* dst = reinterpret_cast<uint4*>(static_cast<bf16*>(a.out) +
                                                    ((int64_t)(g.s.q0 + node) * nq + head) * D + (c0 + i) * 16);
#pragma unroll
              for (int e = 0; e < 2; ++e)
                dst[e] = make_uint4(pack2(o[8 * e] * inv, o[8 * e + 1] * inv), pack2(o[8 * e + 2] * inv, o[8 * e + 3] * inv),
                                    pack2(o[8 * e + 4] * inv, o[8 * e + 5] * inv), pack2(o[8 * e + 6] * inv, o[8 * e + 7] * inv));
            } else {
              float4* dst = reinterpret_cast<float4*>(t.part_o + pslot * D + (c0 + i) * 16);
#pragma unroll
              for (int e = 0; e < 4; ++e) dst[e] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
            }
          }
        }
        if (join && !(ok = meet())) break;
      }
      tc_fence_before();  // O is read before the next segment's first product overwrites it
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }

  // ---- join the parts of items that a share cut (none where every item is one tile)
  if (*s_max_nt <= 1) return;
  cg::this_grid().sync();
  const int nq = a.num_kv_heads * G;
  for (int64_t it = (int64_t)blockIdx.x * (kThreads / 32) + warp; it < (int64_t)a.rows * nq;
       it += (int64_t)grid * (kThreads / 32)) {
    const int row = (int)(it / nq), head = (int)(it % nq), h = head / G;
    int lo = 0, up = a.batch;
    while (up - lo > 1) {
      const int mid = (lo + up) >> 1;
      if (a.cu_seqlens_q[mid] <= row) lo = mid; else up = mid;
    }
    const int b = lo;
    if (pu[b + 1] == pu[b]) continue;                      // no keys, or a tree that was left out
    const Seq s = seq_of(a, b);
    const int node = row - s.q0;
    if (node < 0 || node >= s.n) continue;                 // rows behind the last sequence
    const int rt = node / per, pair = rt / 2;
    const bool two = s.n > (2 * pair + 1) * per;
    const int prow = (two ? rt & 1 : 0) * kRows + (node % per) * G + head % G;
    const Chunks c = chunks_of(s.nt, s.pairs, share);
    constexpr int V = D / 32;
    float acc[V], top = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
    bool whole = false;
    for (int ci = 0; ci < c.n && !whole; ++ci) {
      const int start = c.start(ci), clen = c.start(ci + 1) - start;
      const int u0 = pu[b] + (h * s.nt + start) * s.pairs + pair * clen, u1 = u0 + clen;
      // the CTA whose share holds u0: the largest x with x * W / grid <= u0
      int x = (int)(((int64_t)u0 * grid + grid - 1) / W);
      while (share_lo(x, W, grid) > u0) --x;
      while (share_lo(x + 1, W, grid) <= u0) ++x;
      for (; x < grid && share_lo(x, W, grid) < u1; ++x) {
        const int lo_x = share_lo(x, W, grid);
        if (share_lo(x + 1, W, grid) == lo_x) continue;    // an empty share
        if (c.n == 1 && lo_x <= u0 && share_lo(x + 1, W, grid) >= u1) { whole = true; break; }
        const int64_t ps = (int64_t)(x * 2 + (lo_x >= u0 ? 0 : 1)) * t.part_rows + prow;
        const float2 ml = __ldcg(t.part_ml + ps);
        const float* po = t.part_o + ps * D + lane * V;
        float v[V];
        if constexpr (V == 4) {
          const float4 f = __ldcg(reinterpret_cast<const float4*>(po));
          v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
        } else {
          const float2 f = __ldcg(reinterpret_cast<const float2*>(po));
          v[0] = f.x; v[1] = f.y;
        }
        const float nt = fmaxf(top, ml.x);
        const float fa = top == -INFINITY ? 0.f : ex2(top - nt), fb = ml.x == -INFINITY ? 0.f : ex2(ml.x - nt);
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = acc[i] * fa + v[i] * fb;
        l = l * fa + ml.y * fb;
        top = nt;
      }
    }
    if (whole) continue;
    const float inv = l > 0.f ? 1.f / l : 0.f;
    uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<bf16*>(a.out) + ((int64_t)row * nq + head) * D + lane * V);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) dst[i] = pack2(acc[2 * i] * inv, acc[2 * i + 1] * inv);
  }
}

// ------------------------------------------------------------------ host side
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

void encode(CUtensorMap* map, int rank, const void* base, const cuuint64_t* dims, const cuuint64_t* strides,
            const cuuint32_t* box) {
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUresult r = encode_fn()(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(base), dims, strides, box,
                                 estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                 CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) throw std::runtime_error("tree attention tensor map: encode failed " + std::to_string((int)r));
}

template <int D>
void launch(const TreeAttnArgs& a, const TreeAttnTcPlan& p, cudaStream_t s) {
  CUtensorMap km, vm, qm;
  const cuuint64_t kd[4] = {(cuuint64_t)D, (cuuint64_t)a.block_size, (cuuint64_t)a.num_kv_heads, (cuuint64_t)a.num_blocks};
  const cuuint64_t ks[3] = {(cuuint64_t)D * 2, (cuuint64_t)a.block_size * D * 2, (cuuint64_t)a.block_stride * 2};
  const cuuint32_t kb[4] = {64, (cuuint32_t)p.sub_rows, 1, 1};
  encode(&km, 4, a.k_cache, kd, ks, kb);
  encode(&vm, 4, a.v_cache, kd, ks, kb);
  const int nq = a.num_kv_heads * a.group;
  const cuuint64_t qd[3] = {(cuuint64_t)D, (cuuint64_t)nq, (cuuint64_t)a.rows};
  const cuuint64_t qs[2] = {(cuuint64_t)D * 2, (cuuint64_t)nq * D * 2};
  const cuuint32_t qb[3] = {64, (cuuint32_t)a.group, (cuuint32_t)(kRows / a.group)};
  encode(&qm, 3, a.q, qd, qs, qb);
  TcArgs t{};
  t.a = a;
  t.part_rows = p.part_rows;
  t.sub_rows = p.sub_rows;
  t.part_o = static_cast<float*>(p.workspace);
  t.part_ml = reinterpret_cast<float2*>(t.part_o + (int64_t)p.grid * 2 * p.part_rows * D);
  // slices of the batch that fit the shared table of units (one launch for up to kTreeTcBatch sequences)
  for (int b0 = 0; b0 < a.batch; b0 += kTreeTcBatch) {
    t.a.batch = std::min(kTreeTcBatch, a.batch - b0);
    t.a.cu_seqlens_q = a.cu_seqlens_q + b0;
    t.a.seq_lens = a.seq_lens + b0;
    t.a.block_tables = a.block_tables + (int64_t)b0 * a.max_blocks;
    const int smem = Lay<D>::smem(kTreeTcBatch);
    smem_opt_in(tree_attn_tc_kernel<D>, smem);
    void* params[] = {&km, &vm, &qm, &t};
    const cudaError_t e = cudaLaunchCooperativeKernel(reinterpret_cast<const void*>(tree_attn_tc_kernel<D>), dim3(p.grid),
                                                      dim3(kThreads), params, smem, s);
    if (e != cudaSuccess) throw std::runtime_error(std::string("tree_attn: ") + cudaGetErrorString(e));
  }
}

}  // namespace

bool tree_attn_tc_plan(const TreeAttnArgs& a, int max_q_len, TreeAttnTcPlan* p) {
  if (a.kv_int8 || (a.head_dim != 64 && a.head_dim != 128) || a.group > kRows || a.num_blocks <= 0) return false;
  if (a.block_size % kKeys == 0) p->sub_rows = kKeys;
  else if (kKeys % a.block_size == 0 && a.block_size % 8 == 0) p->sub_rows = a.block_size;
  else return false;
  // units are counted in 32 bits
  const int64_t tiles = ((int64_t)a.max_blocks * a.block_size + kKeys - 1) / kKeys;
  const int per = kRows / a.group, pairs = ((max_q_len + per - 1) / per + 1) / 2;
  if (tiles * pairs * a.num_kv_heads * std::min(a.batch, kTreeTcBatch) >= (1ll << 31)) return false;
  p->part_rows = max_q_len > per ? 2 * kRows : kRows;
  p->grid = device_sm_count();
  p->workspace_bytes = (int64_t)p->grid * 2 * p->part_rows * (a.head_dim * 4 + 8);
  return true;
}

void tree_attn_tc(const TreeAttnArgs& a, const TreeAttnTcPlan& p, cudaStream_t s) {
  if (a.head_dim == 128) launch<128>(a, p, s);
  else launch<64>(a, p, s);
}

}  // namespace b200
