// Layout of a batch in the paged cache, from its lengths, on the device: block tables
// of rows whose groups share a prefix's pages, the slots of the step's new tokens, and
// the append of those tokens' K/V by slot. The slot formula block_table[b, pos / bs] * bs
// + pos % bs is the proposer's (vllm_draft_spec/proposer.py:295-314); the pool is the one
// of the paged append (proposer.py:18-22).
#include "sdx_launch.hpp"

#include <type_traits>

namespace sdx {

constexpr int PG_NT = 256;
constexpr int PG_LDS = 1024;  // offsets kept in LDS for a search

// Every `step`-th of n + 1 ascending offsets in LDS, step the smallest that fits.
__device__ __forceinline__ int64_t pg_step(int64_t n) { return (n + PG_LDS - 1) / PG_LDS; }
__device__ __forceinline__ void pg_fill(const int64_t* cu, int64_t n, int64_t step, int64_t* s) {
  for (int64_t i = threadIdx.x; i * step < n; i += PG_NT) s[i] = cu[i * step];
}
// The last i in [0, n) with cu[i] <= x, or 0: by halves in LDS, then between two kept
// offsets in memory. Ends for any contents of cu, with an index inside [0, n). N searches at
// once, whose steps wait for LDS together.
template <int N>
__device__ __forceinline__ void pg_find(const int64_t* cu, int64_t n, int64_t step, const int64_t* s,
                                        const int64_t (&x)[N], int64_t (&at)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) at[i] = 0;
  for (int len = (int)((n + step - 1) / step); len > 1; len -= len / 2) {  // uniform
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (s[at[i] + len / 2] <= x[i]) at[i] += len / 2;
  }
  if (step == 1) return;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    int64_t lo = at[i] * step, hi = min(lo + step, n);
    while (hi - lo > 1) {
      const int64_t mid = (lo + hi) / 2;
      if (cu[mid] <= x[i]) lo = mid;
      else hi = mid;
    }
    at[i] = lo;
  }
}

// ---- block tables. A workgroup fills the columns [PG_COLS y, PG_COLS (y + 1)) of a few
// consecutive rows, one up to PG_GRID rows. Where their own pages start in the free list is a
// sum over the rows before them, and whether anything is handed out depends on all rows: every
// workgroup adds up the rows itself (8 bytes each, from the L2), which saves the launch of a
// scan. Bound by latency: a row's length, its group's first row's length and the free list are
// three dependent loads, PG_UN rows of them in flight per thread, and the adding up grows with
// the rows; the offsets and prefixes lie in LDS up to 1,024 groups. In a graph, rows in
// groups of 6 to 8 with tables of 44 columns: 32 rows 4.2 us, 786 9.8 (10.4 with tables of 3 MB),
// 4,096 50 (83 with a workgroup for every row), 131,072 2,050 (92,000), 2^20 21,500.
constexpr int PG_COLS = 4096;
constexpr int PG_UN = 4;
constexpr int PG_GRID = 2048;  // workgroups that the chip holds at once: more would add up again

// I: uint32_t where the table's lengths fit 32 bits (a short division; a length or a prefix
// that does not makes its row, or its group's first, bad, and that leaves every table empty),
// or uint64_t.
struct PgRow {
  int64_t first;          // first row of its group
  int32_t need, shared;   // pages, pages shared with it
  bool ok;
};
template <typename I>
__device__ __forceinline__ PgRow pg_row(const BlockTableArgs& a, int64_t b, int64_t kv, int64_t f,
                                        int64_t end, int64_t p, int64_t kv_first) {
  PgRow r;
  const I bs = (I)a.bs;
  r.ok = kv >= 0 && kv <= a.max_blocks * a.bs;
  r.need = r.ok ? (int32_t)(((I)kv + bs - 1) / bs) : 0;
  r.first = b;
  r.shared = 0;
  if (a.cu_group) {
    if (f < 0 || f > b || b >= end) {  // the offsets do not hold b
      r.ok = false;
    } else {
      r.first = f;
      r.ok = r.ok && p >= 0 && p <= kv_first;  // the first row holds the whole prefix
      if (f != b && r.ok) r.shared = min((int32_t)((I)p / bs), r.need);
    }
  }
  return r;
}

// MANY: several rows a workgroup; the code for it costs a single one's 0.2 us of 4.
template <typename I, bool MANY>
__global__ void __launch_bounds__(PG_NT) block_tables_kernel(BlockTableArgs a) {
  constexpr int NW = PG_NT / kWave;
  __shared__ int64_t sCu[PG_LDS + 1], sPrefix[PG_LDS];
  __shared__ uint64_t sSum[NW][3];
  const int tid = threadIdx.x;
  const int64_t row = MANY ? (int64_t)blockIdx.x * a.rows : blockIdx.x;
  const bool grouped = a.cu_group;
  const int64_t step = grouped ? pg_step(a.groups) : 1;
  int bad = 0;
  if (grouped) {  // offsets from 0 up to the batch
    pg_fill(a.cu_group, a.groups, step, sCu);
    if (step == 1) {
      pg_fill(a.prefix_len, a.groups, 1, sPrefix);
      if (tid == 0) sCu[a.groups] = a.cu_group[a.groups];
    }
    if (tid == 0) bad |= a.cu_group[0] != 0 || a.cu_group[a.groups] != a.batch;
    for (int64_t g = tid; g < a.groups; g += PG_NT) bad |= a.cu_group[g] > a.cu_group[g + 1];
  }
  __syncthreads();
  // the rows of a thread at a time, in the order in which what follows from a load is loaded;
  // offsets that are no row are refused by pg_row
  int64_t sum[3] = {0, 0, 0};  // own pages of all rows, of those before `row`, before its group's first
  PgRow me;
  auto rows = [&](auto last, int64_t b0, bool first) {
    constexpr int N = last + 1;  // the first of them is `row` where `first`
    int64_t b[N], kv[N], kf[N], f[N], end[N], p[N], g[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      b[i] = first && i == 0 ? row : min(b0 + (int64_t)(i - (first ? 1 : 0)) * PG_NT, a.batch - 1);
      kv[i] = a.kv_len[b[i]];
      kf[i] = f[i] = end[i] = p[i] = 0;
    }
    if (grouped) {
      pg_find<N>(a.cu_group, a.groups, step, sCu, b, g);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        f[i] = step == 1 ? sCu[g[i]] : a.cu_group[g[i]];
        end[i] = step == 1 ? sCu[g[i] + 1] : a.cu_group[g[i] + 1];
        p[i] = step == 1 ? sPrefix[g[i]] : a.prefix_len[g[i]];
        kf[i] = a.kv_len[max((int64_t)0, min(f[i], a.batch - 1))];
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const PgRow r = pg_row<I>(a, b[i], kv[i], f[i], end[i], p[i], kf[i]);
      if (first && i == 0) {
        me = r;
      } else if (b0 + (int64_t)(i - (first ? 1 : 0)) * PG_NT < a.batch) {
        bad |= !r.ok;
        const int64_t own = r.need - r.shared;
        sum[0] += own;
        if (b[i] < row) sum[1] += own;
        if (b[i] < me.first) sum[2] += own;
      }
    }
  };
  if (a.batch <= PG_NT) {
    rows(std::integral_constant<int, 1>(), tid, true);
  } else {
    rows(std::integral_constant<int, PG_UN>(), tid, true);
    for (int64_t b0 = tid + PG_UN * PG_NT; b0 - tid < a.batch; b0 += PG_UN * PG_NT)
      rows(std::integral_constant<int, PG_UN - 1>(), b0, false);
  }
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    const uint64_t w = wave_sum_u64((uint64_t)sum[i]);
    if ((tid & (kWave - 1)) == 0) sSum[tid / kWave][i] = w;
  }
  bad = __syncthreads_or(bad);
  int64_t total = 0, before = 0, before_first = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    total += sSum[w][0];
    before += sSum[w][1];
    before_first += sSum[w][2];
  }
  bad |= total > a.num_free;
  if (blockIdx.x == 0 && blockIdx.y == 0 && tid == 0) {
    if (a.used) *a.used = bad ? 0 : total;
    if (bad && a.error) *a.error = 1;
  }
  const int64_t end = min(a.max_blocks, ((int64_t)blockIdx.y + 1) * PG_COLS);
  for (int64_t r = row;;) {  // uniform
    int32_t* const out = a.table + r * a.max_blocks;
    for (int64_t c0 = (int64_t)blockIdx.y * PG_COLS + tid; c0 < end; c0 += PG_UN * PG_NT) {
      int32_t v[PG_UN];
#pragma unroll
      for (int i = 0; i < PG_UN; ++i) {
        const int64_t c = c0 + i * PG_NT;
        v[i] = -1;
        if (!bad && c < me.need)  // the first row's own pages start at its column 0
          v[i] = a.free_blocks[c < me.shared ? before_first + c : before + c - me.shared];
      }
#pragma unroll
      for (int i = 0; i < PG_UN; ++i)
        if (c0 + i * PG_NT < end) out[c0 + i * PG_NT] = v[i];
    }
    if (!MANY || ++r == min(row + a.rows, a.batch)) break;
    // the next row: behind this one's pages; its group's first row is this group's, or itself
    before += me.need - me.shared;
    int64_t f = 0, ge = 0, p = 0, kf = 0;
    if (grouped) {
      const int64_t x[1] = {r};
      int64_t g[1];
      pg_find<1>(a.cu_group, a.groups, step, sCu, x, g);
      f = step == 1 ? sCu[g[0]] : a.cu_group[g[0]];
      ge = step == 1 ? sCu[g[0] + 1] : a.cu_group[g[0] + 1];
      p = step == 1 ? sPrefix[g[0]] : a.prefix_len[g[0]];
      kf = a.kv_len[max((int64_t)0, min(f, a.batch - 1))];
    }
    me = pg_row<I>(a, r, a.kv_len[r], f, ge, p, kf);
    if (me.first == r) before_first = before;
  }
}

// ---- positions and slots of the packed new tokens: a thread per token, its row found
// in the offsets. Two dependent loads after the search (row, page), 16 bytes written. In a
// graph 2.5 us for a step of 64 rows of up to 9 tokens, 4.2 for 243,000 tokens of 40 rows.
template <typename I>  // uint32_t where positions fit 32 bits (a short division), or uint64_t
__global__ void __launch_bounds__(PG_NT) paged_slots_kernel(PagedSlotArgs a) {
  __shared__ int64_t sCu[PG_LDS];
  const int64_t step = pg_step(a.batch);
  pg_fill(a.cu_q, a.batch, step, sCu);
  __syncthreads();
  const int64_t t = (int64_t)blockIdx.x * PG_NT + threadIdx.x;
  if (t >= a.tokens) return;
  const int64_t x[1] = {t};
  int64_t at[1];
  pg_find<1>(a.cu_q, a.batch, step, sCu, x, at);
  const int64_t b = at[0];
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
// all loads in flight before the first store. Bound by HBM: 64 layers of
// 320 tokens of 2 KB 40.8 us, 4.0 TB/s, 8 layers of 4,099 58.3, 4.5 TB/s; a copy of 1 GiB
// reaches 5.1.

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
hipError_t launch_block_tables(const BlockTableArgs& b, hipStream_t s) {
  BlockTableArgs a = b;
  a.rows = (a.batch + PG_GRID - 1) / PG_GRID;
  const dim3 grid((unsigned)((a.batch + a.rows - 1) / a.rows),
                  (unsigned)((a.max_blocks + PG_COLS - 1) / PG_COLS));
  if ((a.max_blocks + 1) * a.bs > 0xFFFFFFFFll)
    hipLaunchKernelGGL((block_tables_kernel<uint64_t, true>), grid, dim3(PG_NT), 0, s, a);
  else if (a.rows > 1)
    hipLaunchKernelGGL((block_tables_kernel<uint32_t, true>), grid, dim3(PG_NT), 0, s, a);
  else
    hipLaunchKernelGGL((block_tables_kernel<uint32_t, false>), grid, dim3(PG_NT), 0, s, a);
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
