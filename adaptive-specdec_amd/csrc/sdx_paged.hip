// Layout of a batch in the paged cache, from its lengths, on the device: block tables
// of rows whose groups share a prefix's pages, the slots of the step's new tokens, and
// the append of those tokens' K/V by slot. The slot formula block_table[b, pos / bs] * bs
// + pos % bs is the proposer's (vllm_draft_spec/proposer.py:295-314); the pool is the one
// of the paged append (proposer.py:18-22).
#include "sdx_launch.hpp"

namespace sdx {

constexpr int PG_NT = 256;
constexpr int PG_LDS = 1024;  // offsets kept in LDS for a search

// Sum over the workgroup (PG_NT threads); every thread gets it. sRed: one word per wave.
__device__ __forceinline__ int64_t pg_block_sum(int64_t v, uint64_t* sRed) {
  const uint64_t w = wave_sum_u64((uint64_t)v);
  if ((threadIdx.x & (kWave - 1)) == 0) sRed[threadIdx.x / kWave] = w;
  __syncthreads();
  uint64_t t = 0;
#pragma unroll
  for (int i = 0; i < PG_NT / kWave; ++i) t += sRed[i];
  __syncthreads();  // sRed is reused
  return (int64_t)t;
}

// Every `step`-th of n + 1 ascending offsets in LDS, step the smallest that fits.
__device__ __forceinline__ int64_t pg_step(int64_t n) { return (n + PG_LDS - 1) / PG_LDS; }
__device__ __forceinline__ void pg_fill(const int64_t* cu, int64_t n, int64_t step, int64_t* s) {
  for (int64_t i = threadIdx.x; i * step < n; i += PG_NT) s[i] = cu[i * step];
}
// The last i in [0, n) with cu[i] <= x, or 0: by halves in LDS, then between two kept
// offsets in memory. Ends for any contents of cu, with an index inside [0, n).
__device__ __forceinline__ int64_t pg_find(const int64_t* cu, int64_t n, int64_t step,
                                           const int64_t* s, int64_t x) {
  int64_t lo = 0, hi = (n + step - 1) / step;
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) / 2;
    if (s[mid] <= x) lo = mid;
    else hi = mid;
  }
  lo *= step;
  hi = min(lo + step, n);
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) / 2;
    if (cu[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// ---- block tables. A workgroup fills the columns [PG_COLS y, PG_COLS (y + 1)) of row x.
// Where its own pages start in the free list is a sum over the rows before it, and whether
// anything is handed out depends on all rows: every workgroup adds up the rows itself (8
// bytes each, from the L2), which saves the launch of a scan. Bound by latency: the
// offsets, the lengths and the free list are three dependent loads.
constexpr int PG_COLS = 4096;

struct PgRow {
  int64_t first, need, shared;  // first row of its group, pages, pages shared with it
  bool ok;
};
__device__ __forceinline__ PgRow pg_row(const BlockTableArgs& a, int64_t b, int64_t g) {
  PgRow r;
  const int64_t kv = a.kv_len[b];
  r.ok = kv >= 0 && kv <= a.max_blocks * a.bs;
  r.need = r.ok ? (kv + a.bs - 1) / a.bs : 0;
  r.first = b;
  r.shared = 0;
  if (a.cu_group) {
    const int64_t f = a.cu_group[g], end = a.cu_group[g + 1];
    if (f < 0 || f > b || b >= end) {  // the offsets do not hold b
      r.ok = false;
    } else {
      const int64_t p = a.prefix_len[g];
      r.first = f;
      r.ok = r.ok && p >= 0 && p <= a.kv_len[f];  // the first row holds the whole prefix
      if (f != b && r.ok) r.shared = min(p / a.bs, r.need);
    }
  }
  return r;
}

__global__ void __launch_bounds__(PG_NT) block_tables_kernel(BlockTableArgs a) {
  __shared__ int64_t sCu[PG_LDS];
  __shared__ uint64_t sRed[PG_NT / kWave];
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x;
  const int64_t step = a.cu_group ? pg_step(a.groups) : 1;
  if (a.cu_group) pg_fill(a.cu_group, a.groups, step, sCu);
  __syncthreads();
  auto group_of = [&](int64_t b) -> int64_t {
    return a.cu_group ? pg_find(a.cu_group, a.groups, step, sCu, b) : 0;
  };
  const PgRow me = pg_row(a, row, group_of(row));
  // own pages of the rows before `row`, before its group's first row, and of all rows
  int64_t before = 0, before_first = 0, total = 0;
  int bad = 0;
  for (int64_t b = tid; b < a.batch; b += PG_NT) {
    const PgRow r = pg_row(a, b, group_of(b));
    bad |= !r.ok;
    const int64_t mine = r.need - r.shared;
    total += mine;
    if (b < row) before += mine;
    if (b < me.first) before_first += mine;
  }
  if (a.cu_group) {  // offsets from 0 up to the batch
    if (tid == 0) bad |= a.cu_group[0] != 0 || a.cu_group[a.groups] != a.batch;
    for (int64_t g = tid; g < a.groups; g += PG_NT) bad |= a.cu_group[g] > a.cu_group[g + 1];
  }
  total = pg_block_sum(total, sRed);
  before = pg_block_sum(before, sRed);
  before_first = pg_block_sum(before_first, sRed);
  bad = __syncthreads_or(bad) || total > a.num_free;
  if (blockIdx.x == 0 && blockIdx.y == 0 && tid == 0) {
    if (a.used) *a.used = bad ? 0 : total;
    if (bad && a.error) *a.error = 1;
  }
  int32_t* const out = a.table + row * a.max_blocks;
  const int64_t end = min(a.max_blocks, ((int64_t)blockIdx.y + 1) * PG_COLS);
  for (int64_t c = (int64_t)blockIdx.y * PG_COLS + tid; c < end; c += PG_NT) {
    int32_t v = -1;
    if (!bad && c < me.need)  // the first row's own pages start at its column 0
      v = a.free_blocks[c < me.shared ? before_first + c : before + c - me.shared];
    out[c] = v;
  }
}

// ---- positions and slots of the packed new tokens: a thread per token, its row found
// in the offsets. Two dependent loads after the search (row, page), 16 bytes written.
template <typename I>  // uint32_t where positions fit 32 bits (a short division), or uint64_t
__global__ void __launch_bounds__(PG_NT) paged_slots_kernel(PagedSlotArgs a) {
  __shared__ int64_t sCu[PG_LDS];
  const int64_t step = pg_step(a.batch);
  pg_fill(a.cu_q, a.batch, step, sCu);
  __syncthreads();
  const int64_t t = (int64_t)blockIdx.x * PG_NT + threadIdx.x;
  if (t >= a.tokens) return;
  const int64_t b = pg_find(a.cu_q, a.batch, step, sCu, t);
  const int64_t q0 = a.cu_q[b], q1 = a.cu_q[b + 1], kv = a.kv_len[b];
  int64_t pos = 0, slot = a.padding_slot;
  if (t >= q0 && t < q1) {
    const int64_t p = kv - (q1 - t);  // >= kv - q_b
    int bad = kv > a.max_blocks * a.bs || kv < q1 - q0 || q0 < 0;
    if (!bad) {
      const I pg = (I)p / (I)a.bs;
      const int32_t page = a.table[b * a.max_blocks + (int64_t)pg];
      bad = page < 0;
      if (!bad) {
        pos = p;
        slot = (int64_t)page * a.bs + (int64_t)((I)p - pg * (I)a.bs);
      }
    }
    if (bad && a.error) *a.error = 1;
  } else if (a.error && t < a.cu_q[a.batch]) {
    *a.error = 1;  // offsets that leave a token out
  }
  a.positions[t] = pos;
  a.slots[t] = slot;
}

// ---- append by slot: blockIdx.y is (layer, side); a thread moves PA_UN 16-byte units,
// all loads in flight before the first store. Bound by HBM.
constexpr int PA_UN = 4;
__global__ void __launch_bounds__(PG_NT) append_slots_kernel(AppendSlotArgs a) {
  const uint8_t* const src = a.staged + (int64_t)blockIdx.y * a.tokens * a.row_bytes;
  uint8_t* const dst = a.pool + (int64_t)(blockIdx.y / 2) * a.layer_bytes +
                       (int64_t)(blockIdx.y % 2) * a.side_bytes;
  const uint32_t upr = (uint32_t)(a.row_bytes / 16);
  const int64_t units = a.tokens * upr;
  const int64_t u0 = (int64_t)blockIdx.x * (PG_NT * PA_UN) + threadIdx.x;
  uint4 v[PA_UN];
  int64_t to[PA_UN];
#pragma unroll
  for (int i = 0; i < PA_UN; ++i) {
    const int64_t u = u0 + i * PG_NT;
    to[i] = -1;
    if (u >= units) continue;
    const int64_t t = units <= 0x7FFFFFFF ? (int64_t)((uint32_t)u / upr) : u / upr;
    const int64_t slot = a.slots[t];
    v[i] = *reinterpret_cast<const uint4*>(src + u * 16);
    if (slot >= 0 && slot < a.num_slots) to[i] = slot * a.row_bytes + (u - t * upr) * 16;
    else if (slot >= 0 && a.error) *a.error = 1;
  }
#pragma unroll
  for (int i = 0; i < PA_UN; ++i)
    if (to[i] >= 0) *reinterpret_cast<uint4*>(dst + to[i]) = v[i];
}

// ---------------------------------------------------------------- launches
hipError_t launch_block_tables(const BlockTableArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)a.batch, (unsigned)((a.max_blocks + PG_COLS - 1) / PG_COLS));
  hipLaunchKernelGGL(block_tables_kernel, grid, dim3(PG_NT), 0, s, a);
  return hipGetLastError();
}

hipError_t launch_paged_slots(const PagedSlotArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)((a.tokens + PG_NT - 1) / PG_NT));
  if (a.max_blocks * a.bs <= 0xFFFFFFFFll)
    hipLaunchKernelGGL((paged_slots_kernel<uint32_t>), grid, dim3(PG_NT), 0, s, a);
  else
    hipLaunchKernelGGL((paged_slots_kernel<uint64_t>), grid, dim3(PG_NT), 0, s, a);
  return hipGetLastError();
}

hipError_t launch_append_slots(const AppendSlotArgs& a, hipStream_t s) {
  const int64_t units = a.tokens * (a.row_bytes / 16);
  const dim3 grid((unsigned)((units + PG_NT * PA_UN - 1) / (PG_NT * PA_UN)), (unsigned)(2 * a.layers));
  hipLaunchKernelGGL(append_slots_kernel, grid, dim3(PG_NT), 0, s, a);
  return hipGetLastError();
}

}  // namespace sdx
