// Attention of drafted trees on the 5th-generation tensor cores (head_dim 64 or 128; bf16
// pool, or the stage of an int8 one): the same function as tree_attn.cu, for the shapes a
// server runs.
//
// Rows and keys.  The n nodes of a sequence times the G query heads of one KV head are
// packed into tiles of 128 rows (row = node * G + head), keys into tiles of 64.  A
// unit of work is one key tile against one pair of row tiles:
//
//   two row tiles (n * G > 128)   softmax group w of the CTA takes row tile w,
//   one row tile                  the groups take alternate key tiles and their two
//                                 results are joined in the epilogue,
//
// so both groups work on either shape and a K/V tile is read once for up to 256 rows.
//
// Split, without the host knowing a length.  An item is the keys of one (sequence, KV head,
// row pair).  Small batches give every CTA whole items; batches with fewer items than SMs
// cut each item in equal parts, one to a CTA; larger ones order the units (sequence, KV
// head, key chunk, row pair, key tile), and CTA c of the persistent grid takes the c-th of
// equal shares of that order.  A chunk is at least a share long and is the same for all row pairs
// of a KV head, so the CTAs that read the same keys do so at about the same time and
// the L2 serves all but the first.  A cut item leaves an unnormalised
// fp32 result with its running maximum and sum; after a grid-wide barrier the warps
// join those (softmax over the parts).
//
// Roles per CTA (12 warps): two TMA producers, one of Q and K and one of V, because a
// copy with its wait costs its thread about 650 cycles and one thread alone held the
// whole kernel at 4.9 TB/s; two MMA issuers, one per softmax group (S = Q K^T, then
// O += P V with P read from TMEM, where it overlays its S); two softmax groups of four
// warps, a thread per row, so the row statistics need no shuffles.  The running maximum moves only when a row grows by
// more than 2^8, so O is rarely rescaled.  P is rounded to bf16 for the MMA and the sum
// that divides O adds the rounded values, which cancels that rounding where few keys
// carry the weight.
//
// What bounds it (kernel times, 18 calls in a graph on a card that was idle before; calls in a long row of
// them in brackets).  64 chains of 4 nodes at 4k context: the cache, 542 MB in 96.7 us, 5.6 TB/s [110 to 113].
// 4 trees of 64 nodes at 32k, 16 query heads on a KV head: 272 GFLOP in 300 us, 0.56 of the bf16 burst peak
// [353: 1000 W hold the card at 1.52 GHz, 0.56 of the bf16 peak that it sustains]; a tile's chain S, softmax,
// P V, next S is as long as the softmax of a tile (about 2,100 cycles), and TMEM has no room for a third S.
// Smaller calls: setup, first loads, epilogue, barrier and join, 10 to 12 us (one request at 500 context
// 12.4 us [14.3], 32 at 1.1k 26.8 [28.7]; 13 ragged ones 17.3 to 22.3 by card [18.5]).
//
// A masked place never reaches the result: scores are selected, not added to, and a V
// row is cleaned by its producer in front of the MMA (0 * NaN is NaN) -- rows behind the sequence become
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

constexpr int kRows = 128, kKeys = 64;    // of a tile
constexpr int kThreads = 384;
constexpr float kLazyLog2 = 8.f;
constexpr int kAncWords = kTreeMaxNodes / 32;
// What a way of splitting costs beside its longest run of tiles, in bytes of K.  Cut items: partial results, a
// grid barrier and the join (4 items of 12 tiles at D = 128: 15.2 us cut, 17.2 whole; 26 of 11 tiles at
// D = 64: 17.3 cut, 13.8 whole).  Shares that end inside items: a second segment for some CTAs (48 items of
// 51 tiles at D = 128: 28.4 us in parts, 31.5 in shares; with 256 KB 160 items of 24 tiles would go whole,
// 50.7 us instead of 45.7).
constexpr int kCutBytes = 128 << 10, kShareBytes = 192 << 10;
constexpr int kParts = 4;         // partial results in flight per lane when parts are joined
constexpr int kRing = 4;          // segments known ahead, and their dirty bits

template <int D>
struct Lay {
  static constexpr int QTILE = kRows * D * 2, QHALF = kRows * 64 * 2;   // D / 64 halves of [128][64]
  static constexpr int TILE = kKeys * D * 2, HALF = kKeys * 64 * 2;     // of K or V: halves of [64][64]
  static constexpr int SLOTS = D == 128 ? 4 : 8;   // K tiles, and V tiles, in flight (even: see the issuers)
  static constexpr int Q = 0;                      // two row tiles; the second also carries the join
  static constexpr int K = Q + 2 * QTILE;
  static constexpr int V = K + SLOTS * TILE;
  static constexpr int ANC = V + SLOTS * TILE;     // [nodes][kAncWords] ancestor bits
  static constexpr int PAR = ANC + kTreeMaxNodes * kAncWords * 4;
  static constexpr int ML = PAR + kTreeMaxNodes * 4;          // [2][128] (max, sum)
  static constexpr int DIRTY = ML + 2 * kRows * 8;
  static constexpr int SEG = DIRTY + kRing * kAncWords * 4;   // [kRing] segments
  static constexpr int BARS = SEG + kRing * 64;
  static constexpr int NBARS = 5 * SLOTS + 2 + 12 + 3 + 2 * kRing;
  static constexpr int TAB = BARS + NBARS * 8 + 32;           // per sequence: Row, then one more
  static int smem(int batch) { return TAB + (batch + 1) * 16 + 1024; }
};

struct TcArgs {
  TreeAttnArgs a;
  float* part_o;     // [grid][2][part_rows][D]
  float2* part_ml;   // [grid][2][part_rows]
  int part_rows;     // 128 or 256
  int sub_rows;
  const float* key_scales;   // SCALED: [batch][kv_heads][k | v][key_stride]
  int key_stride;
};

__device__ __forceinline__ uint32_t sw_off(int r, int u) { return r * 128 + ((u ^ (r & 7)) << 4); }

// Whether a phase has completed, without waiting.
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

__device__ __forceinline__ void tma_5d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int half, int z,
                                       int w) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(half), "r"(z), "r"(w)
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
template <>
__device__ __forceinline__ void tmem_ld<16>(uint32_t addr, float* v) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
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
// 32 bytes in one store
__device__ __forceinline__ void st32(void* p, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
               ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
// two fp32 operations in one instruction, each rounded to nearest
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 ra, rb, rc, rd;\n\t"
      "mov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmov.b64 rc, {%6, %7};\n\t"
      "fma.rn.f32x2 rd, ra, rb, rc;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
      "add.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
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
  // (n is at most the grid, and nt * n below 2^32: the host has checked the number of units)
  __device__ __forceinline__ int start(int i) const { return n == 1 ? i * nt : (int)((uint32_t)i * (uint32_t)nt / (uint32_t)n); }
  __device__ __forceinline__ int of(int tile) const { return (int)(((uint32_t)(tile + 1) * (uint32_t)n - 1) / (uint32_t)nt); }
};

// Per sequence, in shared memory.
struct Row {
  int q0, len;         // first row, keys
  int unit, item;      // units (parts, see Plan) and items in front of it
};

// First sequence with work that holds a row, else the last.  Not inlined: that cost the ragged batch 0.15 us.
__device__ __noinline__ int holder(const Row* rows, int batch, int row) {
  int b = 0;
  while (b < batch - 1 && !(rows[b + 1].unit != rows[b].unit && rows[b].q0 <= row && row < rows[b + 1].q0)) ++b;
  return b;
}

// The grid's work, in one of three ways:
//   whole items    nothing is cut, several items to a CTA;
//   parts          every item in equal parts of at most `parts` tiles, one part to a CTA (fewer items than CTAs);
//   equal shares   of the units, a share may begin and end inside an item.
struct Plan {
  const Row* rows;     // [batch + 1]
  int batch, kvh, per; // sequences, KV heads, nodes per row tile
  int W, items;        // units and items in all
  int grid, share;     // CTAs with work, units of the largest share
  int whole;           // whole items
  int parts;           // tiles of a part, 0: not in parts
  int base, rem;       // quotient and remainder of W (items) by the CTAs

  __device__ __forceinline__ int nodes(int b) const { return rows[b + 1].q0 - rows[b].q0; }
  __device__ __forceinline__ int tiles(int b) const { return (rows[b].len + kKeys - 1) / kKeys; }
  __device__ __forceinline__ int pairs(int b) const { return ((nodes(b) + per - 1) / per + 1) >> 1; }
  __device__ __forceinline__ int cuts(int nt) const { return (nt + parts - 1) / parts; }
  __device__ __forceinline__ Chunks chunks(int nt, int pr) const {
    return {whole || pr == 1 || nt <= share ? 1 : nt / share, nt};
  }
  // last sequence with at most x units (items) in front of it
  __device__ __forceinline__ int at(int x, bool by_item) const {
    int lo = 0, up = batch;
    while (up - lo > 1) {
      const int mid = (lo + up) >> 1;
      if ((by_item ? rows[mid].item : rows[mid].unit) <= x) lo = mid; else up = mid;
    }
    return lo;
  }
  // first unit of CTA c
  __device__ __forceinline__ int lo(int c) const {
    if (parts) return min(c, grid);
    if (c >= grid) return W;
    const int x = c * base + min(c, rem);
    if (!whole || x >= items) return whole ? W : x;
    const int b = at(x, true);
    return rows[b].unit + (x - rows[b].item) * tiles(b);
  }
  // the CTA whose share holds unit u (shares of units)
  __device__ __forceinline__ int cta(int u) const {
    const int edge = rem * (base + 1);
    return u < edge ? u / (base + 1) : rem + (u - edge) / base;
  }
};

// A run of key tiles [t0, t1) of one item (sequence, KV head, row pair) inside a CTA's share.
struct Seg {
  int b, h, pair, q0, n, len;
  int t0, t1;          // t1 = 0: no more segments
  int two;             // two row tiles
  int whole;           // covers all of the item's keys
  int slot;            // partial result of the CTA
  int pad[5];
};
static_assert(sizeof(Seg) == 64, "segment ring");

// The key tiles of a segment that softmax group w takes.
struct Own {
  int first, step, n;
  __device__ __forceinline__ Own(const Seg& g, int gt, int w) {
    step = g.two ? 1 : 2;
    first = g.two || (gt & 1) == w ? g.t0 : g.t0 + 1;
    n = first < g.t1 ? (g.t1 - 1 - first) / step + 1 : 0;
  }
  __device__ __forceinline__ int tile(int s) const { return first + s * step; }
};

__device__ __forceinline__ Seg seg_at(const Plan& p, int u, int lo, int hi) {
  Seg g;
  g.b = p.at(u, false);
  const Row row = p.rows[g.b];
  g.q0 = row.q0;
  g.len = row.len;
  g.n = p.nodes(g.b);
  const int nt = p.tiles(g.b), pr = p.pairs(g.b);
  int r = u - row.unit;
  if (p.parts) {
    const int cuts = p.cuts(nt), item = r / cuts;
    r -= item * cuts;
    g.h = item / pr;
    g.pair = item - g.h * pr;
    g.t0 = (r * nt) / cuts;
    g.t1 = ((r + 1) * nt) / cuts;
  } else {
    const int per_head = nt * pr;
    g.h = r / per_head;
    r -= g.h * per_head;
    const Chunks c = p.chunks(nt, pr);
    int start = 0, end = nt;
    if (c.n > 1) {
      const int ci = c.of(r / pr);
      start = c.start(ci);
      end = c.start(ci + 1);
    }
    r -= start * pr;
    g.pair = pr == 1 ? 0 : r / (end - start);
    g.t0 = start + r - g.pair * (end - start);
    g.t1 = min(end, g.t0 + (hi - u));
  }
  g.whole = g.t0 == 0 && g.t1 == nt;
  g.two = g.n > (2 * g.pair + 1) * p.per;
  g.slot = u == lo ? 0 : 1;
  return g;
}

// Block ids of a sequence's table by the lanes of a warp, 32 at a time and the next 32 on their way:
// a load per tile in front of its copies cost more than the copies.  Also copies a tile of keys.
struct Blocks {
  const int* tab;
  int max_blocks, num_blocks, block_size, sub_rows, len;
  int bi, y;             // block and row of the next tile's first key
  int window, ids, ids_next;
  bool bad;
  __device__ __forceinline__ int entry(int i) const { return i < max_blocks ? __ldg(tab + i) : -1; }
  __device__ __forceinline__ void start(const TreeAttnArgs& a, int b, int key, int keys, int lane) {
    tab = a.block_tables + b * a.table_stride;
    len = keys;
    bi = key / block_size;
    y = key - bi * block_size;
    window = bi;
    ids = entry(window + lane);
    ids_next = entry(window + 32 + lane);
  }
  // keys [key, key + kKeys) of KV head h, in boxes of sub_rows; the whole warp
  template <int D>
  __device__ __forceinline__ void copy(const CUtensorMap* map, uint64_t* bar, uint8_t* tile, int key, int h, int lane) {
    using L = Lay<D>;
    while (bi >= window + 32) {
      window += 32;
      ids = ids_next;
      ids_next = entry(window + 32 + lane);
    }
    const uint32_t dst = smem_u32(tile);
    if (sub_rows == kKeys) {
      // a box of the whole tile
      const int id = __shfl_sync(0xffffffffu, ids, bi - window);
      const bool in = id >= 0 && id < num_blocks;
      if (!in) bad = true;
      if (lane == 0) tma_5d(dst, map, bar, 0, y, 0, h, in ? id : num_blocks);   // out of range: zero fill
      y += kKeys;
      if (y >= block_size) { y = 0; ++bi; }
    } else {
      // whole blocks, at most eight, each half of the columns by a lane of its own: one lane's copies
      // one after the other held pages of 16 keys at 4.1 TB/s
      const int row = lane / (D / 64) * sub_rows, hf = lane % (D / 64);
      const int d = bi - window + lane / (D / 64);
      const int a0 = __shfl_sync(0xffffffffu, ids, d & 31), a1 = __shfl_sync(0xffffffffu, ids_next, d & 31);
      if (row < kKeys) {
        const int id = d < 32 ? a0 : a1;
        int blk = num_blocks;
        if (key + row < len) {
          if (id >= 0 && id < num_blocks) blk = id;
          else bad = true;
        }
        tma_5d(dst + hf * L::HALF + row * 128, map, bar, 0, 0, hf, h, blk);
      }
      __syncwarp();
      bi += kKeys / sub_rows;
    }
  }
};

// SCALED: K and V hold int8 values (exact in bf16), one factor for each key and one for each value row
// apply to the scores and to P.
template <int D, bool SCALED>
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
  uint64_t* v_ready = k_empty + kSlots;   // landed, and cleaned where it had to be
  uint64_t* v_full = v_ready + kSlots;    // landed, of the tiles that have to be cleaned
  uint64_t* v_empty = v_full + kSlots;
  uint64_t* q_full = v_empty + kSlots;
  uint64_t* q_empty = q_full + 1;
  uint64_t* s_full = q_empty + 1;         // [2][2] per softmax group and score buffer
  uint64_t* p_full = s_full + 4;          // [2][2]
  uint64_t* pv_done = p_full + 4;         // [2][2]
  uint64_t* fin = pv_done + 4;            // [2] an issuer's last products
  uint64_t* both = fin + 2;               // the eight softmax warps meet
  uint64_t* joined = both + 1;            // [kRing] the softmax warps are done with the segment's join
  uint64_t* seg_full = joined + kRing;    // [kRing]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(seg_full + kRing);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* s_max_nt = reinterpret_cast<int*>(tmem_slot + 2);
  int* s_parts = s_max_nt + 1;
  int* s_bad = s_max_nt + 2;              // a tree does not fit
  Row* rows = reinterpret_cast<Row*>(smem + L::TAB);
  volatile Seg* segs = reinterpret_cast<volatile Seg*>(smem + L::SEG);
  uint32_t* anc = reinterpret_cast<uint32_t*>(smem + L::ANC);
  int* s_par = reinterpret_cast<int*>(smem + L::PAR);
  float2* s_ml = reinterpret_cast<float2*>(smem + L::ML);
  uint32_t* dirty = reinterpret_cast<uint32_t*>(smem + L::DIRTY);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = a.group, per = kRows / G;   // nodes per row tile
  int* status = a.status;

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&k_map);
    tma_prefetch_desc(&v_map);
    tma_prefetch_desc(&q_map);
  }
  // ---- the work of every sequence; a tree that does not fit has none
  if (threadIdx.x == 0) *s_max_nt = *s_bad = 0;
  __syncthreads();
  for (int b = threadIdx.x; b < a.batch; b += kThreads) {
    const int q0 = a.cu_seqlens_q[b], q1 = a.cu_seqlens_q[b + 1], len = a.seq_lens[b];
    const bool bad = !tree_fits(q0, q1, a.rows, a.max_q_len, len) ||
                     (q0 < q1 && len > (int64_t)a.max_blocks * a.block_size);
    if (bad && blockIdx.x == 0) record_status(status, kStatusBadShape);
    Row r{q0, len, 0, 0};
    if (!bad && q0 < q1) {
      const int nt = (len + kKeys - 1) / kKeys;
      r.item = ((q1 - q0 + per - 1) / per + 1) / 2 * a.num_kv_heads;
      r.unit = r.item * nt;
      atomicMax(s_max_nt, nt);
    }
    if (bad) *s_bad = 1;
    rows[b] = r;
    if (b == a.batch - 1) rows[b + 1].q0 = q1;
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
      for (int k = 0; k < 2; ++k) {
        mbar_init(&s_full[2 * i + k], 1);
        mbar_init(&p_full[2 * i + k], 4);
        mbar_init(&pv_done[2 * i + k], 1);
      }
      mbar_init(&fin[i], 1);
    }
    mbar_init(both, 8);
    for (int i = 0; i < kRing; ++i) {
      mbar_init(&joined[i], 8);
      mbar_init(&seg_full[i], 1);
    }
    fence_barrier_init();
    *abort_flag = 0;
  }
  __syncthreads();
  if (warp == 0) {
    int units = 0, items = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 32) {
      const int b = b0 + lane;
      const int mu = b < a.batch ? rows[b].unit : 0, mi = b < a.batch ? rows[b].item : 0;
      int u = mu, i = mi;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int pu = __shfl_up_sync(0xffffffffu, u, o), pi = __shfl_up_sync(0xffffffffu, i, o);
        if (lane >= o) { u += pu; i += pi; }
      }
      if (b < a.batch) {
        rows[b].unit = units + u - mu;
        rows[b].item = items + i - mi;
      }
      units += __shfl_sync(0xffffffffu, u, 31);
      items += __shfl_sync(0xffffffffu, i, 31);
    }
    if (lane == 0) {
      rows[a.batch].unit = units;
      rows[a.batch].item = items;
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
  Plan plan{rows, a.batch, a.num_kv_heads, per, rows[a.batch].unit, rows[a.batch].item};
  const int max_nt = *s_max_nt;
  const int ctas = (int)gridDim.x;
  // (the integer divisions are the longest part of this, so the small batches leave before them)
  const int rounds = plan.items <= ctas ? 1 : (plan.items + ctas - 1) / ctas;
  plan.share = max_nt;
  plan.whole = rounds * max_nt <= kCutBytes / L::TILE;
  if (!plan.whole) {
    plan.share = (plan.W + ctas - 1) / ctas;
    int cut = plan.share + kShareBytes / L::TILE;
    if (plan.items < ctas && max_nt < 1 << 23) {
      // Parts of S tiles are at most W / S + items, and S (ctas - items) >= W makes that at most the CTAs.
      // (Two tiles take the two groups as long as one.)
      const int parts = max(2, (plan.W + ctas - plan.items - 1) / (ctas - plan.items));
      if (parts <= cut) cut = plan.parts = parts;
    }
    plan.whole = rounds * max_nt <= cut + kCutBytes / L::TILE;
    if (plan.whole) plan.parts = 0;
  }
  if (plan.parts) {
    // parts in front of every sequence, in the place of its units
    if (warp == 0) {
      int sum = 0;
      for (int b0 = 0; b0 < a.batch; b0 += 32) {
        const int b = b0 + lane;
        const int mine = b < a.batch ? (rows[b + 1].item - rows[b].item) * plan.cuts(plan.tiles(b)) : 0;
        int x = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int px = __shfl_up_sync(0xffffffffu, x, o);
          if (lane >= o) x += px;
        }
        if (b < a.batch) rows[b].unit = sum + x - mine;
        sum += __shfl_sync(0xffffffffu, x, 31);
      }
      if (lane == 0) *s_parts = sum;
    }
    __syncthreads();          // (every thread has read the number of units)
    plan.grid = *s_parts;
    if (threadIdx.x == 0) rows[a.batch].unit = plan.grid;
  } else {
    const int spread = plan.whole ? plan.items : plan.W;
    plan.grid = min(ctas, spread);
    plan.base = spread <= ctas ? 1 : spread / ctas;
    plan.rem = spread <= ctas ? 0 : spread - plan.base * ctas;
  }
  int edge[2] = {plan.lo(blockIdx.x), plan.lo(blockIdx.x + 1)};
  const int u_lo = edge[0], u_hi = edge[1];
  // No role is kRing segments ahead of another, so a ring of barriers tells segments apart.
  auto join_over = [&](int sg) {
    return mbar_wait(&joined[sg % kRing], (sg / kRing) & 1, status, kStatusTimeoutEmpty, abort_flag);
  };
  // segment sg of this CTA, written by the producer; none behind the last
  auto segment = [&](int sg, Seg& g) {
    if (!mbar_wait(&seg_full[sg % kRing], (sg / kRing) & 1, status, kStatusTimeoutFull, abort_flag)) return false;
    const volatile int* src = reinterpret_cast<const volatile int*>(&segs[sg % kRing]);
    int* dst = reinterpret_cast<int*>(&g);
#pragma unroll
    for (int i = 0; i < 11; ++i) dst[i] = src[i];
    return g.t1 > 0;
  };

  auto settle = [&]() {
    if (!*abort_flag) return;
    // a wait gave up: let the copies already issued land before the CTA exits
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 1000000ull) __nanosleep(1000);
  };

  if (warp == 0) {
    // ================================================================ producer of Q and K
    Blocks blocks{nullptr, a.max_blocks, a.num_blocks, a.block_size, t.sub_rows};
    int gt = 0, sg = 0;   // tiles, segments
    bool ok = true;
    for (int u = u_lo; ok; ++sg) {
      Seg g{};
      if (u < u_hi) g = seg_at(plan, u, u_lo, u_hi);
      u = plan.parts ? u_hi : u + g.t1 - g.t0;
      if (lane == 0) {
        volatile int* dst = reinterpret_cast<volatile int*>(&segs[sg % kRing]);
        const int* src = reinterpret_cast<const int*>(&g);
#pragma unroll
        for (int i = 0; i < 11; ++i) dst[i] = src[i];
        mbar_arrive(&seg_full[sg % kRing]);
      }
      if (g.t1 == 0) break;
      blocks.start(a, g.b, g.t0 * kKeys, g.len, lane);
      ok = mbar_wait(q_empty, (sg & 1) ^ 1, status, kStatusTimeoutEmpty, abort_flag);
      // its second Q tile may still carry a join
      if (ok && g.two && sg > 0) ok = join_over(sg - 1);
      if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      if (lane == 0) {
        const int tiles = g.two ? 2 : 1;
        mbar_arrive_expect_tx(q_full, tiles * kHalves * per * G * 128);
        for (int i = 0; i < tiles; ++i)
#pragma unroll
          for (int hf = 0; hf < kHalves; ++hf)
            tma_3d(smem_u32(smem + L::Q + i * L::QTILE + hf * L::QHALF), &q_map, q_full, hf * 64, g.h * G,
                   g.q0 + (2 * g.pair + i) * per);
      }
      for (int j = g.t0; j < g.t1; ++j, ++gt) {
        const int slot = gt % kSlots;
        ok = mbar_wait(&k_empty[slot], ((gt / kSlots) & 1) ^ 1, status, kStatusTimeoutEmpty, abort_flag);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        if (lane == 0) mbar_arrive_expect_tx(&k_full[slot], L::TILE);
        blocks.template copy<D>(&k_map, &k_full[slot], smem + L::K + slot * L::TILE, j * kKeys, g.h, lane);
      }
    }
    if (blocks.bad) record_status(status, kStatusBadShape);
    if (lane == 0) settle();
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
      Seg g;
      for (; ok && segment(sg, g); ++sg) {
        if (!mbar_wait(q_full, sg & 1, status, kStatusTimeoutFull, abort_flag)) break;
        const uint32_t qa = smem_u32(smem + L::Q + (g.two ? w : 0) * L::QTILE);
        const Own own(g, gt, w);
        auto issue_s = [&](int s) {
          const int slot = (gt + own.tile(s) - g.t0) % kSlots, buf = (mine + s) & 1;
          const uint32_t kb = smem_u32(smem + L::K + slot * L::TILE);
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t qo = (k >> 2) * L::QHALF + (k & 3) * 32, ko = (k >> 2) * L::HALF + (k & 3) * 32;
            umma_f16_ss(tS + buf * kKeys, umma_sdesc_sw128(qa + qo), umma_sdesc_sw128(kb + ko), idesc_s, k > 0 ? 1u : 0u);
          }
          umma_commit(&s_full[2 * w + buf]);
          umma_commit(&k_empty[slot]);
          if (!g.two) umma_commit(&k_empty[slot]);     // the other group does not read this tile
        };
        auto issue_pv = [&](int s) {
          const int slot = (gt + own.tile(s) - g.t0) % kSlots, buf = (mine + s) & 1;
          const uint32_t vb = smem_u32(smem + L::V + slot * L::TILE);
#pragma unroll
          for (int k = 0; k < kKeys / 16; ++k)
            umma_f16_ts(tO, tS + buf * kKeys + k * 8, sdesc_mn(vb + k * 16 * 128, L::HALF), idesc_pv, (s > 0 || k > 0) ? 1u : 0u);
          umma_commit(&pv_done[2 * w + buf]);
          umma_commit(&v_empty[slot]);
          if (!g.two) umma_commit(&v_empty[slot]);
        };
        // Scores run up to two tiles ahead; whichever product has its inputs goes first (waiting for
        // the next K here would hold back the product that frees a V tile).
        int si = 0, pi = 0;
        uint64_t since = 0;
        while (pi < own.n) {
          bool did = false;
          if (si < own.n && si < pi + 2) {
            const int at = gt + own.tile(si) - g.t0;
            // the scores overlay the P of the tile two before
            if ((si < 2 || mbar_test(&pv_done[2 * w + ((mine + si) & 1)], ((mine + si - 2) >> 1) & 1)) &&
                mbar_test(&k_full[at % kSlots], (at / kSlots) & 1)) {
              tc_fence_after();
              issue_s(si++);
              did = true;
            }
          }
          if (pi < si && mbar_test(&p_full[2 * w + ((mine + pi) & 1)], ((mine + pi) >> 1) & 1)) {
            const int at = gt + own.tile(pi) - g.t0;
            if (mbar_test(&v_ready[at % kSlots], (at / kSlots) & 1)) {
              tc_fence_after();
              issue_pv(pi++);
              did = true;
            }
          }
          if (did) {
            since = 0;
          } else if (since == 0) {
            since = globaltimer_ns();
          } else if (*abort_flag || globaltimer_ns() - since > kWaitLimitNs) {
            if (!*abort_flag) record_status(status, kStatusTimeoutConv);
            *abort_flag = 1;
            ok = false;
            break;
          }
        }
        if (!ok) break;
        mine += own.n;
        gt += g.t1 - g.t0;
        // the segment's products are done (its Q, and every K and V phase before the next)
        umma_commit(q_empty);
      }
      // every product issued so far ends before TMEM is released
      umma_commit(&fin[w]);
      mbar_wait(&fin[w], 0, status, kStatusTimeoutAccEmpty, nullptr);
    }
    __syncwarp();
  } else if (warp == 3) {
    // ================================================================ producer of V
    Blocks blocks{nullptr, a.max_blocks, a.num_blocks, a.block_size, t.sub_rows};
    int gt = 0, sg = 0;
    uint32_t cleaned = 0;      // parity of each slot's v_full: it counts the tiles that had to be cleaned
    bool ok = true;
    Seg g;
    for (; ok && __all_sync(0xffffffffu, segment(sg, g)); ++sg) {
      uint32_t* dirt = dirty + (sg % kRing) * kAncWords;
      if (lane < kAncWords) dirt[lane] = 0;
      __syncwarp();
      const int prefix = g.len - g.n;
      blocks.start(a, g.b, g.t0 * kKeys, g.len, lane);
      // a tile with nodes or with rows behind the sequence, in slot `slot`
      auto clean = [&](int j, int slot) {
        ok = mbar_wait(&v_full[slot], (cleaned >> slot) & 1, status, kStatusTimeoutFull, abort_flag);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; return; }
        cleaned ^= 1u << slot;
        uint8_t* vt = smem + L::V + slot * L::TILE;
        for (int r = lane; r < kKeys; r += 32) {
          const int node = j * kKeys + r - prefix;
          if (node < 0) continue;
          const bool behind = node >= g.n;
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
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_ready[slot]);
      };
      int due = -1;            // the tile before this one, if it has to be cleaned
      for (int j = g.t0; j < g.t1 && ok; ++j, ++gt) {
        const int slot = gt % kSlots;
        ok = mbar_wait(&v_empty[slot], ((gt / kSlots) & 1) ^ 1, status, kStatusTimeoutEmpty, abort_flag);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        const bool dirty_tile = (j + 1) * kKeys > prefix;
        uint64_t* bar = dirty_tile ? &v_full[slot] : &v_ready[slot];
        if (lane == 0) mbar_arrive_expect_tx(bar, L::TILE);
        blocks.template copy<D>(&v_map, bar, smem + L::V + slot * L::TILE, j * kKeys, g.h, lane);
        if (due >= 0) clean(due, (gt - 1) % kSlots);
        due = dirty_tile ? j : -1;
      }
      if (ok && due >= 0) clean(due, (gt - 1) % kSlots);
    }
    if (blocks.bad) record_status(status, kStatusBadShape);
    if (lane == 0) settle();
    __syncwarp();
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
    // product i of this group has been added to O (the one two before it is known to be)
    auto pv_over = [&](int i) {
      return mbar_wait(&pv_done[2 * w + (i & 1)], (i >> 1) & 1, status, kStatusTimeoutAccEmpty, abort_flag);
    };
    Seg g;
    while (ok && __all_sync(0xffffffffu, segment(sg, g))) {
      const int prefix = g.len - g.n;
      if (g.t1 * kKeys > prefix && g.b != seen_b) {
        // ancestor bits of the sequence's nodes, by walking the parents in shared memory
        if (!meet()) break;
        if (tid < g.n) s_par[tid] = a.parents[g.q0 + tid];
        if (!meet()) break;
        if (tid < g.n) {
          uint32_t bits[kAncWords] = {};
          for (int at = tid; at >= 0;) {        // a parent that is not in front of its child ends the walk
#pragma unroll
            for (int i = 0; i < kAncWords; ++i) bits[i] |= (at >> 5) == i ? 1u << (at & 31) : 0u;
            const int up = s_par[at];
            at = up < at ? up : -1;
          }
          uint4* dst = reinterpret_cast<uint4*>(anc + tid * kAncWords);
          dst[0] = make_uint4(bits[0], bits[1], bits[2], bits[3]);
          dst[1] = make_uint4(bits[4], bits[5], bits[6], bits[7]);
        }
        if (!meet()) break;
        seen_b = g.b;
      }
      const int tile = 2 * g.pair + (g.two ? w : 0);
      const int node = tile * per + r / G, head = g.h * G + r % G;
      const bool valid = r < per * G && node < g.n;
      const bool any = __any_sync(0xffffffffu, valid);
      // columns [c, c + 32) of key tile j that this row sees
      auto sees = [&](int kb, int c) -> uint32_t {
        const int t0 = kb + c - prefix;                 // node of the first column
        uint32_t see = t0 >= 0 ? 0u : t0 <= -32 ? 0xffffffffu : (1u << -t0) - 1u;
        if (t0 > -32 && valid) {
          const int i = t0 >> 5;
          const uint32_t* row = anc + node * kAncWords;
          const uint32_t lo = i >= 0 && i < kAncWords ? row[i] : 0u;
          const uint32_t up = i + 1 < kAncWords ? row[i + 1] : 0u;
          see |= __funnelshift_r(lo, up, t0 & 31);
        }
        return see;
      };
      float m = -INFINITY, l = 0.f;
      const Own own(g, gt, w);
      const int done = own.n;
      const float* factors = SCALED ? t.key_scales + ((int64_t)g.b * a.num_kv_heads + g.h) * 2 * t.key_stride : nullptr;
#pragma unroll 1
      for (int i = 0; i < own.n; ++i, ++mine) {
        const int buf = mine & 1;
        const uint32_t tb = tS + buf * kKeys;
        ok = mbar_wait(&s_full[2 * w + buf], (mine >> 1) & 1, status, kStatusTimeoutAccFull, abort_flag);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        tc_fence_after();
        if (any) {
          const int kb = own.tile(i) * kKeys;
          float s[kKeys];
          tmem_ld<32>(tb, s);
          tmem_ld<32>(tb + 32, s + 32);
          tmem_ld_wait();
          if constexpr (SCALED) {
#pragma unroll
            for (int e = 0; e < kKeys; e += 4) {
              const float4 f = __ldg(reinterpret_cast<const float4*>(factors + kb + e));
              s[e] *= f.x;
              s[e + 1] *= f.y;
              s[e + 2] *= f.z;
              s[e + 3] *= f.w;
            }
          }
          if (kb + kKeys > prefix) {
            const uint32_t lo = sees(kb, 0), hi = sees(kb, 32);
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              if (!((lo >> e) & 1u)) s[e] = -INFINITY;
              if (!((hi >> e) & 1u)) s[32 + e] = -INFINITY;
            }
          }
          float x[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = fmaxf(s[e], s[8 + e]);
#pragma unroll
          for (int q = 2; q < 8; ++q)
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = fmaxf(x[e], s[8 * q + e]);
          const float mx = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7]))) * sl2;
          const bool grow = mx > m + kLazyLog2;
          if (__any_sync(0xffffffffu, grow)) {
            float alpha = 1.f;
            if (grow) {
              alpha = m == -INFINITY ? 1.f : ex2(m - mx);
              m = mx;
              l *= alpha;
            }
            if (i > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
              // the product before this one may still be adding to O
              ok = pv_over(mine - 1);
              if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
              tc_fence_after();
#pragma unroll 1
              for (int c = 0; c < D / 16; ++c) {
                float o[16];
                tmem_ld<16>(tO + c * 16, o);
                tmem_ld_wait();
                uint32_t ou[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) ou[e] = __float_as_uint(o[e] * alpha);
                tmem_st16(tO + c * 16, ou);
              }
            }
          }
          const float2 k2 = make_float2(sl2, sl2);
          const float mu = m == -INFINITY ? 0.f : -m;
          const float2 mu2 = make_float2(mu, mu);
          float2 sum0 = make_float2(0.f, 0.f), sum1 = sum0;
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            uint32_t p[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float2 z = fma2(make_float2(s[q * 32 + 2 * e], s[q * 32 + 2 * e + 1]), k2, mu2);
              if constexpr (SCALED) {
                // (the sum takes P as it is; a place without weight takes no part, whatever its factor)
                const float2 x = make_float2(ex2(z.x), ex2(z.y));
                const float2 f = __ldg(reinterpret_cast<const float2*>(factors + t.key_stride + kb + q * 32 + 2 * e));
                p[e] = pack2(x.x == 0.f ? 0.f : x.x * f.x, x.y == 0.f ? 0.f : x.y * f.y);
                if (e & 1) sum1 = add2(sum1, x); else sum0 = add2(sum0, x);
              } else {
                p[e] = pack2(ex2(z.x), ex2(z.y));
                const float2 back = make_float2(__uint_as_float(p[e] << 16), __uint_as_float(p[e] & 0xffff0000u));
                if (e & 1) sum1 = add2(sum1, back); else sum0 = add2(sum0, back);
              }
            }
            tmem_st16(tb + q * 16, p);           // P overlays its scores, which this thread has read
          }
          l += (sum0.x + sum0.y) + (sum1.x + sum1.y);
          tmem_st_wait();
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[2 * w + buf]);
      }
      gt += g.t1 - g.t0;
      if (!ok) break;
      // ---------------------------------------------------------------- epilogue
      const bool join = !g.two && g.t1 - g.t0 > 1;   // both groups hold a part of every row
      if (done > 0) {
        ok = pv_over(mine - 1);
        if (!__all_sync(0xffffffffu, ok)) break;
        tc_fence_after();
      }
      // Where both groups hold a part, each hands the other half of its columns, D / 4 at a time,
      // through the second Q tile (not in use by a segment with one row tile).
      constexpr int kHand = D / 4;
      float4* stage = reinterpret_cast<float4*>(smem + L::Q + L::QTILE);   // [2][kHand / 4][128]
      auto hand = [&](int round) {
        float o[kHand];
        tmem_ld<kHand>(tO + ((w ^ 1) * 2 + round) * kHand, o);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < kHand / 4; ++e)
          stage[(w * (kHand / 4) + e) * kRows + r] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
      };
      float fac = 1.f, ofac = 0.f;
      if (join) {
        if (sg > 0) {
          ok = join_over(sg - 1);   // the other group has read what the last join handed over
          if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        }
        s_ml[w * kRows + r] = make_float2(m, l);
        hand(0);
        if (!(ok = meet())) break;
        const float2 other = s_ml[(w ^ 1) * kRows + r];
        const float top = fmaxf(m, other.x);
        fac = m == -INFINITY ? 0.f : ex2(m - top);
        ofac = other.x == -INFINITY ? 0.f : ex2(other.x - top);
        l = l * fac + other.y * ofac;
        m = top;
      }
      const float inv = 1.f / l;   // every score -inf: l and O are 0, the row NaN
      const int64_t pblk = blockIdx.x * 2 + g.slot;
      const int prow = (g.two ? w : 0) * kRows + r;
      if (!g.whole && valid && done > 0 && (!join || w == 0)) t.part_ml[pblk * t.part_rows + prow] = make_float2(m, l);
      const uint32_t* dirt = dirty + (sg % kRing) * kAncWords;
      bool dirt_any = false;
#pragma unroll
      for (int i = 0; i < kAncWords; ++i) dirt_any |= dirt[i] != 0;
      // columns this thread writes: all of its row, or its half of a joined row
      const int c_end = join ? (w + 1) * (D / 2) : done > 0 ? D : 0;
#pragma unroll 1
      for (int c = join ? w * (D / 2) : 0; c < c_end; c += kHand) {
        if (join && c != w * (D / 2)) {
          if (!(ok = meet())) break;
          hand(1);
          if (!(ok = meet())) break;
        }
        float o[kHand];
        __syncwarp();
        tmem_ld<kHand>(tO + c, o);
        tmem_ld_wait();
        if (join) {
#pragma unroll
          for (int e = 0; e < kHand / 4; ++e) {
            const float4 v = stage[((w ^ 1) * (kHand / 4) + e) * kRows + r];
            o[4 * e] = o[4 * e] * fac + v.x * ofac;
            o[4 * e + 1] = o[4 * e + 1] * fac + v.y * ofac;
            o[4 * e + 2] = o[4 * e + 2] * fac + v.z * ofac;
            o[4 * e + 3] = o[4 * e + 3] * fac + v.w * ofac;
          }
        }
        if (valid) {
          if (dirt_any) {
            // V elements that were not finite count for the rows that see their node
            for (int d = 0; d < g.n; ++d) {
              if (!((dirt[d >> 5] & anc[node * kAncWords + (d >> 5)]) >> (d & 31) & 1u)) continue;
              const int key = prefix + d, id = a.block_tables[g.b * a.table_stride + key / a.block_size];
              const bf16* v = static_cast<const bf16*>(a.v_cache) + (int64_t)id * a.block_stride +
                              ((int64_t)g.h * a.block_size + key % a.block_size) * D + c;
#pragma unroll 1
              for (int e = 0; e < kHand; ++e) {
                const float x = __bfloat162float(v[e]);
#pragma unroll
                for (int f = 0; f < kHand; ++f)
                  if (f == e && !isfinite(x)) o[f] += x;
              }
            }
          }
          if (g.whole) {
            uint32_t v[kHand / 2];
#pragma unroll
            for (int e = 0; e < kHand / 2; ++e) v[e] = pack2(o[2 * e] * inv, o[2 * e + 1] * inv);
#pragma unroll
            for (int e = 0; e < kHand; e += 16)
              st32(static_cast<bf16*>(a.out) + ((int64_t)(g.q0 + node) * nq + head) * D + c + e, v + e / 2);
          } else {
            // columns by fours, rows inside: a warp's stores are contiguous
            float4* dst = reinterpret_cast<float4*>(t.part_o) + (pblk * (D / 4) + c / 4) * t.part_rows + prow;
#pragma unroll
            for (int e = 0; e < kHand / 4; ++e)
              dst[e * t.part_rows] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
          }
        }
      }
      if (!ok) break;
      if (join) fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&joined[sg % kRing]);
      tc_fence_before();  // O is read before the next segment's first product overwrites it
      ++sg;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }

  // ---- join the parts of items that a share cut: a lane per row (node and query head) and 16 columns
  if (plan.whole) return;
  const bool any_bad = *s_bad;
  cg::this_grid().sync();
  const int nq = a.num_kv_heads * G, qrows = a.rows * G, groups = (qrows + 31) / 32;
  const int tasks = groups * a.num_kv_heads * (D / 16);
  for (int it = blockIdx.x + gridDim.x * warp; it < tasks; it += gridDim.x * (kThreads / 32)) {
    const int c4 = it % (D / 16) * 4, x = it / (D / 16), h = x - x / a.num_kv_heads * a.num_kv_heads;
    const int qr = x / a.num_kv_heads * 32 + lane;
    if (qr >= qrows) continue;
    const int row = qr / G, hg = qr - row * G;
    int lo = 0, up = a.batch;
    while (up - lo > 1) {
      const int mid = (lo + up) >> 1;
      if (rows[mid].q0 <= row) lo = mid; else up = mid;
    }
    if (any_bad) lo = holder(rows, a.batch, row);   // (offsets of a bad tree may lead that search astray)
    const int b = lo, unit0 = rows[b].unit;
    const int node = row - rows[b].q0;
    // nothing to do for a tree that was left out and for rows behind the last sequence
    if (rows[b + 1].unit == unit0 || node < 0 || node >= plan.nodes(b)) continue;
    const int nt = plan.tiles(b), pr = plan.pairs(b);
    const int rt = node / per, pair = rt / 2;
    const bool two = plan.nodes(b) > (2 * pair + 1) * per;
    const int prow = (two ? rt & 1 : 0) * kRows + (node - rt * per) * G + hg;
    const Chunks c = plan.parts ? Chunks{1, nt} : plan.chunks(nt, pr);
    float acc[16], top = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = 0.f;
    bool whole = false;
    for (int ci = 0; ci < c.n && !whole; ++ci) {
      const int start = c.start(ci), clen = c.start(ci + 1) - start;
      int x0, x1, begun = 0;      // CTAs; whether the first one's share begins in front of this chunk
      if (plan.parts) {
        const int cuts = plan.cuts(nt);
        x0 = unit0 + (h * pr + pair) * cuts;
        x1 = x0 + cuts - 1;
      } else {
        const int u0 = unit0 + (h * nt + start) * pr + pair * clen;
        x0 = plan.cta(u0);
        x1 = plan.cta(u0 + clen - 1);
        begun = x0 * plan.base + min(x0, plan.rem) < u0;
      }
      if (c.n == 1 && x0 == x1) { whole = true; break; }
      for (int x = x0; x <= x1; x += kParts) {
        float2 ml[kParts];
        float4 v[kParts][4];
#pragma unroll
        for (int k = 0; k < kParts; ++k) {
          ml[k] = make_float2(-INFINITY, 0.f);
          if (x + k > x1) continue;
          const int pblk = (x + k) * 2 + (x + k == x0 ? begun : 0);
          ml[k] = __ldcg(t.part_ml + pblk * t.part_rows + prow);
          const float4* po = reinterpret_cast<const float4*>(t.part_o) + ((int64_t)pblk * (D / 4) + c4) * t.part_rows + prow;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[k][e] = __ldcg(po + e * t.part_rows);
        }
        float mt = top;
#pragma unroll
        for (int k = 0; k < kParts; ++k) mt = fmaxf(mt, ml[k].x);
        const float fa = top == -INFINITY ? 0.f : ex2(top - mt);
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[e] *= fa;
        l *= fa;
#pragma unroll
        for (int k = 0; k < kParts; ++k) {
          if (x + k > x1) continue;
          const float fb = ml[k].x == -INFINITY ? 0.f : ex2(ml[k].x - mt);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            acc[4 * e] += v[k][e].x * fb;
            acc[4 * e + 1] += v[k][e].y * fb;
            acc[4 * e + 2] += v[k][e].z * fb;
            acc[4 * e + 3] += v[k][e].w * fb;
          }
          l += ml[k].y * fb;
        }
        top = mt;
      }
    }
    if (whole) continue;
    const float inv = 1.f / l;
    uint32_t v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = pack2(acc[2 * e] * inv, acc[2 * e + 1] * inv);
    st32(static_cast<bf16*>(a.out) + ((int64_t)row * nq + h * G + hg) * D + c4 * 4, v);
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
  const cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  const CUresult r = encode_fn()(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(base), dims, strides, box,
                                 estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                 CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) throw std::runtime_error("tree attention tensor map: encode failed " + std::to_string((int)r));
}

template <int D, bool SCALED>
int launch(const TreeAttnArgs& a, const TreeAttnTcPlan& p, cudaStream_t s) {
  CUtensorMap km, vm, qm;
  // columns as (64, D / 64): one copy brings both halves of a tile
  const cuuint64_t kd[5] = {64, (cuuint64_t)a.block_size, D / 64, (cuuint64_t)a.num_kv_heads, (cuuint64_t)a.num_blocks};
  const cuuint64_t ks[4] = {(cuuint64_t)D * 2, 128, (cuuint64_t)a.block_size * D * 2, (cuuint64_t)a.block_stride * 2};
  const cuuint32_t kb[5] = {64, (cuuint32_t)p.sub_rows, (cuuint32_t)(p.sub_rows == kKeys ? D / 64 : 1), 1, 1};
  encode(&km, 5, a.k_cache, kd, ks, kb);
  encode(&vm, 5, a.v_cache, kd, ks, kb);
  const int nq = a.num_kv_heads * a.group;
  const cuuint64_t qd[3] = {(cuuint64_t)D, (cuuint64_t)nq, (cuuint64_t)a.rows};
  const cuuint64_t qs[2] = {(cuuint64_t)D * 2, (cuuint64_t)nq * D * 2};
  const cuuint32_t qb[3] = {64, (cuuint32_t)a.group, (cuuint32_t)(kRows / a.group)};
  encode(&qm, 3, a.q, qd, qs, qb);
  TcArgs t{};
  t.a = a;
  t.part_rows = p.part_rows;
  t.sub_rows = p.sub_rows;
  t.key_scales = p.key_scales;
  t.key_stride = p.key_stride;
  t.part_o = static_cast<float*>(p.workspace);
  t.part_ml = reinterpret_cast<float2*>(t.part_o + (int64_t)p.grid * 2 * p.part_rows * D);
  // slices of the batch that fit the shared table of units (one launch for up to kTreeTcBatch sequences)
  int launches = 0;
  for (int b0 = 0; b0 < a.batch; b0 += kTreeTcBatch, ++launches) {
    t.a.batch = std::min(kTreeTcBatch, a.batch - b0);
    t.a.cu_seqlens_q = a.cu_seqlens_q + b0;
    t.a.seq_lens = a.seq_lens + b0;
    t.a.block_tables = a.block_tables + b0 * a.table_stride;
    const int smem = Lay<D>::smem(kTreeTcBatch);
    smem_opt_in(tree_attn_tc_kernel<D, SCALED>, smem);
    void* params[] = {&km, &vm, &qm, &t};
    const cudaError_t e = cudaLaunchCooperativeKernel(reinterpret_cast<const void*>(tree_attn_tc_kernel<D, SCALED>),
                                                      dim3(p.grid), dim3(kThreads), params, smem, s);
    if (e != cudaSuccess) throw std::runtime_error(std::string("tree_attn: ") + cudaGetErrorString(e));
  }
  return launches;
}

}  // namespace

bool tree_attn_tc_plan(const TreeAttnArgs& a, int max_q_len, TreeAttnTcPlan* p) {
  if ((a.head_dim != 64 && a.head_dim != 128) || a.group > kRows || a.num_blocks <= 0) return false;
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

int tree_attn_tc(const TreeAttnArgs& a, const TreeAttnTcPlan& p, cudaStream_t s) {
  if (p.key_scales != nullptr) return a.head_dim == 128 ? launch<128, true>(a, p, s) : launch<64, true>(a, p, s);
  return a.head_dim == 128 ? launch<128, false>(a, p, s) : launch<64, false>(a, p, s);
}

}  // namespace b200
