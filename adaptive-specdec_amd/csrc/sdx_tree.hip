// Trees of drafted tokens: what a step needs of a tree before the target runs (which nodes
// each node sees, its position, its slot in the paged cache), and the walk of the nodes that
// the target's choices accept afterwards. The chain form of the first is the slot formula of
// vllm_draft_spec/proposer.py:295-314, of the second the accept loop of
// specdec/engine.py:285-303.
//
// Both are bound by latency: a few KB, and loads that depend on each other (offsets, parents,
// pages; the walk one choice after another). A tree of 26 nodes: 2.0 us for each kernel; 256 trees
// of up to 64: 3.2 us for the layout, 3.1 for the walk. The host's 10 us a call are more. Trees of more
// than 64 nodes, in graphs: one of 512 8.4 us for the layout (a chain of 512: 11.8), 256 of them 11.3
// (15.0); the walk 3.8 and 4.4, and 0.43 us for every node that it keeps: a chain of 512 that is
// accepted whole takes 218.
#include "sdx_launch.hpp"

namespace sdx {

constexpr int TR_NT = 256;
constexpr int TR_NW = TR_NT / kWave;
constexpr int TR_NPL = TREE_MAX_NODES / kWave;  // nodes of a lane in the largest row
constexpr int TR_NPT = TREE_MAX_NODES / TR_NT;  // nodes of a thread

// Row b's nodes, [q0, q0 + n) of the packed ones: false where they are no part of them.
struct TrRow {
  int64_t q0, n;
  bool ok;
};
__device__ __forceinline__ TrRow tr_row(const int64_t* cu, int64_t b, int64_t tokens, int32_t max_nodes) {
  const int64_t q0 = cu[b], q1 = cu[b + 1];
  return TrRow{q0, q1 - q0, q0 >= 0 && q1 >= q0 && q1 <= tokens && q1 - q0 <= max_nodes};
}

// position and slot of node i, whose depth below a root is `depth`
template <typename I>  // uint32_t where positions fit 32 bits (a short division), or uint64_t
__device__ __forceinline__ void tr_put(const TreeLayoutArgs& a, int64_t b, int64_t t, int64_t start, int i,
                                       int depth) {
  a.positions[t] = start + depth;
  if (!a.slots) return;
  const uint64_t at = (uint64_t)start + i;
  const I pg = (I)at / (I)a.bs;
  const int32_t page = a.table[b * a.max_blocks + (int64_t)pg];
  if (page < 0) {
    a.slots[t] = a.padding_slot;
    if (a.error) *a.error = 1;
  } else {
    a.slots[t] = (int64_t)page * a.bs + (int64_t)((I)at - pg * (I)a.bs);
  }
}
// tokens of no row, or of one that is refused
__device__ __forceinline__ void tr_pad(const TreeLayoutArgs& a, int64_t t) {
  for (int w = 0; w < a.words; ++w) a.mask[t * a.words + w] = 0;
  a.positions[t] = 0;
  if (a.slots) a.slots[t] = a.padding_slot;
}
__device__ __forceinline__ bool tr_lengths(const TreeLayoutArgs& a, int64_t kv, int64_t n) {
  return kv >= n && kv <= a.max_blocks * a.bs;
}

// Masks by doubling: M holds node i's ancestors below J (itself first), and every round takes
// over those of J, until no node's J is left: rounds for the deepest node's path, log2 of it.
// Rows of up to 64 nodes: a wave each, a node per lane, and no LDS or barrier.
template <typename I>
__global__ void __launch_bounds__(TR_NT) tree_layout_wave_kernel(TreeLayoutArgs a) {
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t b = (int64_t)blockIdx.x * TR_NW + threadIdx.x / kWave;
  if (b > a.batch) return;  // uniform per wave
  if (b == a.batch) {       // tokens in front of the first row and behind the last
    const int64_t first = a.cu_q[0], last = a.cu_q[a.batch];
    for (int64_t t = lane; t < min(first, a.tokens); t += kWave) tr_pad(a, t);
    for (int64_t t = max(last, (int64_t)0) + lane; t < a.tokens; t += kWave) tr_pad(a, t);
    if (lane == 0 && a.error && (first != 0 || last > a.tokens)) *a.error = 1;
    return;
  }
  const TrRow r = tr_row(a.cu_q, b, a.tokens, kWave);
  const int64_t kv = a.kv_len[b];
  bool ok = r.ok && tr_lengths(a, kv, r.n);
  int32_t up = -1;
  const bool mine = ok && lane < r.n;
  if (mine) up = a.parents[r.q0 + lane];
  ok = ok && !__any(up < -1 || up >= lane);
  if (!ok) {  // uniform
    if (lane == 0 && a.error) *a.error = 1;
    for (int64_t t = max(r.q0, (int64_t)0) + lane; t < min(r.q0 + r.n, a.tokens); t += kWave) tr_pad(a, t);
    return;
  }
  uint32_t lo = lane < 32 ? 1u << lane : 0u, hi = lane < 32 ? 0u : 1u << (lane - 32);
  int32_t j = up;
  while (__any(j >= 0)) {  // six rounds at most: parents lie in front of their children
    const int from = max(j, 0);
    const uint32_t l = (uint32_t)__shfl((int)lo, from, kWave), h = (uint32_t)__shfl((int)hi, from, kWave);
    const int32_t k = __shfl(j, from, kWave);
    if (j >= 0) lo |= l, hi |= h, j = k;
  }
  if (!mine) return;
  const int64_t t = r.q0 + lane;
  a.mask[t] = (int64_t)((uint64_t)lo | (uint64_t)hi << 32);
  tr_put<I>(a, b, t, kv - r.n, lane, __popc(lo) + __popc(hi) - 1);
}

// Rows of up to TREE_MAX_NODES nodes: a workgroup each, the masks in LDS.
template <typename I>
__global__ void __launch_bounds__(TR_NT) tree_layout_kernel(TreeLayoutArgs a) {
  constexpr int W = TREE_MAX_NODES / 64;
  __shared__ uint64_t sMask[TREE_MAX_NODES][W + 1];  // (a word more: rows in other banks)
  __shared__ int16_t sJump[TREE_MAX_NODES];
  const int tid = threadIdx.x;
  const int64_t b = blockIdx.x;
  if (b == a.batch) {
    const int64_t first = a.cu_q[0], last = a.cu_q[a.batch];
    for (int64_t t = tid; t < min(first, a.tokens); t += TR_NT) tr_pad(a, t);
    for (int64_t t = max(last, (int64_t)0) + tid; t < a.tokens; t += TR_NT) tr_pad(a, t);
    if (tid == 0 && a.error && (first != 0 || last > a.tokens)) *a.error = 1;
    return;
  }
  const TrRow r = tr_row(a.cu_q, b, a.tokens, min(a.words * 64, TREE_MAX_NODES));
  const int64_t kv = a.kv_len[b];
  const bool ok = r.ok && tr_lengths(a, kv, r.n);
  int bad = !ok, left = 0;
  if (ok)
    for (int i = tid; i < r.n; i += TR_NT) {
      const int32_t up = a.parents[r.q0 + i];
      bad |= up < -1 || up >= i;
      sJump[i] = (int16_t)max(up, -1);
      left |= up >= 0;
#pragma unroll
      for (int w = 0; w < W; ++w) sMask[i][w] = w == i / 64 ? 1ull << (i % 64) : 0ull;
    }
  if (__syncthreads_or(bad)) {
    if (tid == 0 && a.error) *a.error = 1;
    for (int64_t t = max(r.q0, (int64_t)0) + tid; t < min(r.q0 + r.n, a.tokens); t += TR_NT) tr_pad(a, t);
    return;
  }
  while (__syncthreads_or(left)) {
    uint64_t m[TR_NPT][W];
    int16_t k[TR_NPT];
    left = 0;
#pragma unroll
    for (int e = 0; e < TR_NPT; ++e) {
      const int i = tid + e * TR_NT;
      const int j = i < r.n ? sJump[i] : -1;
      k[e] = -2;  // nothing to take over
      if (j < 0) continue;
      k[e] = sJump[j];
#pragma unroll
      for (int w = 0; w < W; ++w) m[e][w] = sMask[j][w];
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < TR_NPT; ++e) {
      const int i = tid + e * TR_NT;
      if (k[e] == -2) continue;
#pragma unroll
      for (int w = 0; w < W; ++w) sMask[i][w] |= m[e][w];
      sJump[i] = k[e];
      left |= k[e] >= 0;
    }
  }
  for (int i = tid; i < r.n; i += TR_NT) {
    const int64_t t = r.q0 + i;
    int depth = -1;
#pragma unroll
    for (int w = 0; w < W; ++w) depth += __popcll(sMask[i][w]);
    for (int w = 0; w < a.words; ++w) a.mask[t * a.words + w] = (int64_t)sMask[i][w];
    tr_put<I>(a, b, t, kv - r.n, i, depth);
  }
}

// ---- the walk: from node 0 to the lowest child whose token is the choice at the node, as far
// as there is one. A wave per row, NPL nodes per lane; a child lies behind its parent, so the
// walk ends whatever the parents hold. Up to 64 nodes a step is a ballot and two lane reads.
template <int NPL>
__device__ __forceinline__ int64_t tr_walk(const TreeAcceptArgs& a, const TrRow& r, int64_t* path,
                                           int64_t* sChoice, int64_t& y) {
  const int lane = threadIdx.x;
  int32_t up[NPL];
  int64_t tok[NPL], ch = -1;
#pragma unroll
  for (int e = 0; e < NPL; ++e) {
    const int i = lane + e * kWave;
    up[e] = -2;
    tok[e] = 0;
    if (i < r.n) {
      up[e] = a.parents[r.q0 + i];
      tok[e] = a.token_ids[r.q0 + i];
      ch = a.choice[r.q0 + i];
      if constexpr (NPL > 1) sChoice[i] = ch;
    }
  }
  if constexpr (NPL > 1) __syncthreads();  // one wave: its own stores
  int64_t keep = 0;
  for (int cur = 0;;) {
    if (lane == 0) path[keep] = cur;
    ++keep;
    if constexpr (NPL == 1)
      y = (int64_t)((uint64_t)rdlane((uint32_t)((uint64_t)ch >> 32), cur) << 32 | rdlane((uint32_t)ch, cur));
    else
      y = sChoice[cur];
    if (keep == a.max_path || y < 0) break;
    int next = -1;
#pragma unroll
    for (int e = 0; e < NPL; ++e) {
      const uint64_t hit = __ballot(up[e] == cur && tok[e] == y && lane + e * kWave > cur);
      if (next < 0 && hit) next = e * kWave + __ffsll((unsigned long long)hit) - 1;
    }
    next = __builtin_amdgcn_readfirstlane(next);
    if (next < 0) break;
    cur = next;
  }
  return keep;
}

__global__ void __launch_bounds__(kWave) tree_accept_kernel(TreeAcceptArgs a) {
  __shared__ int64_t sChoice[TREE_MAX_NODES];
  const int lane = threadIdx.x;
  const int64_t b = blockIdx.x;
  const TrRow r = tr_row(a.cu_q, b, a.tokens, TREE_MAX_NODES);
  if (lane == 0 && a.error && !r.ok) *a.error = 1;
  int64_t* const path = a.path + b * a.max_path;
  int64_t keep = 0, y = -1;
  if (r.ok && r.n > 0 && (!a.active || a.active[b]))  // uniform
    keep = r.n <= kWave ? tr_walk<1>(a, r, path, sChoice, y) : tr_walk<TR_NPL>(a, r, path, sChoice, y);
  for (int64_t i = keep + lane; i < a.max_path; i += kWave) path[i] = -1;
  if (lane == 0) {
    a.keep[b] = keep;
    a.y[b] = max(y, (int64_t)-1);
  }
}

// ---------------------------------------------------------------- launches
hipError_t launch_tree_layout(const TreeLayoutArgs& a, hipStream_t s) {
  const bool narrow = a.max_blocks * a.bs <= 0xFFFFFFFFll;
  if (a.words == 1) {
    const dim3 grid((unsigned)((a.batch + 1 + TR_NW - 1) / TR_NW));
    if (narrow) hipLaunchKernelGGL(tree_layout_wave_kernel<uint32_t>, grid, dim3(TR_NT), 0, s, a);
    else hipLaunchKernelGGL(tree_layout_wave_kernel<uint64_t>, grid, dim3(TR_NT), 0, s, a);
  } else {
    const dim3 grid((unsigned)(a.batch + 1));
    if (narrow) hipLaunchKernelGGL(tree_layout_kernel<uint32_t>, grid, dim3(TR_NT), 0, s, a);
    else hipLaunchKernelGGL(tree_layout_kernel<uint64_t>, grid, dim3(TR_NT), 0, s, a);
  }
  return hipGetLastError();
}

hipError_t launch_tree_accept(const TreeAcceptArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)a.batch);
  hipLaunchKernelGGL(tree_accept_kernel, grid, dim3(kWave), 0, s, a);
  return hipGetLastError();
}

}  // namespace sdx
