// Commit of the accepted path of every drafted tree, one launch for all layers.
//
// The model scored a tree of n nodes per sequence; node i holds drafted token
// draft[i] and target[i] is the token the model picks behind node i.  Node 0 is the
// last token already emitted.  The accepted path is
//
//   path[0] = 0,  path[j + 1] = min { c > path[j] : parents[c] == path[j],
//                                      draft[c] == target[path[j]] }
//
// and the step emits target[path[0]], target[path[1]], ...  The cache rows of the
// path, written at positions P + path[j] (P = committed prefix), move to P + j, so
// the cache holds exactly the committed tokens again.
//
// A CTA owns a slice of a sequence's planes (layer, k|v, kv head).  Every CTA walks the
// tree itself (one warp, the tree in shared memory: a ballot per step), which costs
// less than a second launch or a flag; then its threads move rows.  A thread owns
// fixed 16-byte (scales: 4-byte) columns of its planes and takes the path in ascending
// order.  path[j] >= j and path ascends, so a row is read before the step that writes
// its place (j' = path[j] > j), and moving in place is safe without a copy.
//
// Bound by latency: table, tree, walk and rows are four dependent reads.  One request of 8 nodes over 48
// layers takes 4.1 us (kernel in a graph, 5.1 on the slowest card), 32 requests of up to 32 nodes (22 MB read and
// written) 8.5 to 10.6 us, 24 requests on an int8 pool with its scales 7.1 to 8.1 us.  Calls in a row take 8.1,
// 10.2 and 8.3 us, because the host needs 8.7 us for one: its checks, three outputs, the launch.  A CTA takes 8 planes: with 4 the walks of twice the CTAs cost more than the
// copies gain (10.9 us for the 32 requests), with 16 the one request takes 5.0 us.
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

constexpr int kThreads = 128;

template <typename V>
__device__ __forceinline__ void move_rows(uint8_t* base, int row_bytes, int p0, int p1, int planes, int bs,
                                          const int2* moves, int n_moves, int tid, int nthreads) {
  const int vpr = row_bytes / (int)sizeof(V);
  V* b = reinterpret_cast<V*>(base);
  const int64_t plane_v = (int64_t)bs * vpr, block_v = (int64_t)planes * plane_v;
  for (int u = tid; u < (p1 - p0) * vpr; u += nthreads) {
    V* col = b + (int64_t)(p0 + u / vpr) * plane_v + u % vpr;
    for (int j0 = 0; j0 < n_moves; j0 += 4) {  // four loads in flight; their stores write earlier places
      V v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j0 + j < n_moves) {
          const int s = moves[j0 + j].x;
          v[j] = col[(int64_t)(s / bs) * block_v + (int64_t)(s % bs) * vpr];
        }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j0 + j < n_moves) {
          const int d = moves[j0 + j].y;
          col[(int64_t)(d / bs) * block_v + (int64_t)(d % bs) * vpr] = v[j];
        }
    }
  }
}

__global__ void __launch_bounds__(kThreads) tree_commit_kernel(const TreeCommitArgs a, int planes_per_cta) {
  pdl_enter();
  __shared__ int s_par[kTreeMaxNodes], s_draft[kTreeMaxNodes], s_target[kTreeMaxNodes];
  __shared__ int s_path[kTreeMaxNodes];
  __shared__ int2 s_moves[kTreeMaxNodes];  // (source, destination) slots of the pool
  __shared__ int s_len, s_moves_n;
  const int b = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
  const int q0 = a.cu_seqlens_q[b], q1 = a.cu_seqlens_q[b + 1], keys = a.seq_lens[b];
  // a malformed row (offsets outside the arrays, more nodes than keys) commits nothing
  const bool bad = !tree_fits(q0, q1, a.nodes, a.max_q_len, keys);
  const int n = bad ? 0 : q1 - q0, prefix = keys - n;
  if (bad && tid == 0) record_status(a.status, kStatusBadShape);
  for (int i = tid; i < n; i += kThreads) {
    s_par[i] = a.parents[q0 + i];
    s_draft[i] = a.draft[q0 + i];
    s_target[i] = a.target[q0 + i];
  }
  __syncthreads();
  if (tid < 32) {
    int len = 0;
    if (n > 0) {
      int cur = 0;
      while (true) {
        if (lane == 0) s_path[len] = cur;
        ++len;
        const int want = s_target[cur];
        int next = -1;
        for (int c0 = cur + 1; c0 < n && next < 0; c0 += 32) {
          const int c = c0 + lane;
          const unsigned hit = __ballot_sync(0xffffffffu, c < n && s_par[c] == cur && s_draft[c] == want);
          if (hit) next = c0 + __ffs(hit) - 1;
        }
        if (next < 0) break;
        cur = next;
      }
    }
    __syncwarp();
    // the path's rows that change places, as pool slots
    const int* tab = a.block_tables + b * a.table_stride;
    int moved = 0;
    bool out_of_range = false;
    for (int j0 = 0; j0 < len; j0 += 32) {
      const int j = j0 + lane;
      int src = -1, dst = -1;
      if (j < len && s_path[j] != j) {
        const int ps = prefix + s_path[j], pd = prefix + j;
        const int bs_i = ps / a.block_size, bd_i = pd / a.block_size;
        const int sb = bs_i < a.max_blocks ? tab[bs_i] : -1, db = bd_i < a.max_blocks ? tab[bd_i] : -1;
        if (sb >= 0 && sb < a.num_blocks && db >= 0 && db < a.num_blocks) {
          src = sb * a.block_size + ps % a.block_size;
          dst = db * a.block_size + pd % a.block_size;
        } else {
          out_of_range = true;
        }
      }
      const unsigned take = __ballot_sync(0xffffffffu, src >= 0);
      if (src >= 0) s_moves[moved + __popc(take & ((1u << lane) - 1))] = make_int2(src, dst);
      moved += __popc(take);
    }
    if (out_of_range) record_status(a.status, kStatusBadShape);
    if (lane == 0) {
      s_len = len;
      s_moves_n = moved;
    }
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    if (tid == 0) a.accepted[b] = s_len;
    for (int j = tid; j < a.max_q_len; j += kThreads) {
      const int at = j < s_len ? s_path[j] : -1;
      a.path[(int64_t)b * a.max_q_len + j] = at;
      a.tokens[(int64_t)b * a.max_q_len + j] = at >= 0 ? s_target[at] : -1;
    }
  }
  const int p0 = blockIdx.x * planes_per_cta, p1 = min(a.planes, p0 + planes_per_cta);
  for (int k = 0; k < a.kinds; ++k) {
    const TreeRows& r = a.rows[k];
    if (r.row_bytes % 16 == 0)
      move_rows<uint4>(r.base, r.row_bytes, p0, p1, a.planes, a.block_size, s_moves, s_moves_n, tid, kThreads);
    else
      move_rows<uint32_t>(r.base, r.row_bytes, p0, p1, a.planes, a.block_size, s_moves, s_moves_n, tid, kThreads);
  }
  pdl_trigger();
}

}  // namespace

int tree_commit(const TreeCommitArgs& a, cudaStream_t s) {
  const int per = 8;   // planes of a CTA
  constexpr int kMost = 65535;   // blocks of a grid in y
  int launches = 0;
  for (int b0 = 0; b0 < a.batch; b0 += kMost, ++launches) {
    TreeCommitArgs x = a;
    x.batch = std::min(kMost, a.batch - b0);
    x.cu_seqlens_q += b0;
    x.seq_lens += b0;
    x.block_tables += b0 * a.table_stride;
    x.accepted += b0;
    x.path += (int64_t)b0 * a.max_q_len;
    x.tokens += (int64_t)b0 * a.max_q_len;
    pdl_launch(tree_commit_kernel, dim3((x.planes + per - 1) / per, x.batch), kThreads, 0, s, x, per);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) throw std::runtime_error(std::string("tree_commit: ") + cudaGetErrorString(e));
  }
  return launches;
}

}  // namespace b200
