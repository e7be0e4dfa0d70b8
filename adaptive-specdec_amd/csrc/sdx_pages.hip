// Pages of the paged cache after a step: the accepted nodes of a tree moved together behind
// their row, rows that go on from other rows, the pages that no row holds, and copies of pages.
// Nothing is counted up and down between calls: a page is free when no table holds it. The pool
// is the one of the paged append (vllm_draft_spec/proposer.py:18-22); without a counterpart in
// the reference, which leaves tables to a host-side manager and drafts chains.
#include <algorithm>

#include "sdx_launch.hpp"

namespace sdx {

constexpr int PGS_NT = 256;
constexpr int PGS_UN = 4;  // 16-byte loads in flight per thread

__device__ __forceinline__ uint8_t* pgs_side(uint8_t* pool, int64_t layer_bytes, int64_t side_bytes,
                                             int64_t ls) {
  return pool + ls / 2 * layer_bytes + ls % 2 * side_bytes;
}

// Work on n items in every (layer, side): groups of LS sides go to the XCDs in turn (workgroup % 8),
// so that an XCD's translations are those of its own sides. 64 rows of up to 64 nodes in 64 layers
// of 8 heads of 128 are compacted in 14.8 us, without it in 17.6; when the pages of 48 groups of 8 beams
// were freed, forked and copied in 39 us (now 40), they took 55 without it. The workgroup's item, and
// its first side.
__device__ __forceinline__ int64_t pgs_item(int64_t n, int LS, int& ls0) {
  const uint32_t k = blockIdx.x / 8, g = k / (uint32_t)n;
  ls0 = (int)(g * 8 + blockIdx.x % 8) * LS;
  return k - g * (uint32_t)n;
}
// Launches over n items, each of at most 2^23 workgroups (a grid's threads have to stay under 2^32):
// run(grid, first item, items).
template <typename F>
static hipError_t pgs_launch(int64_t n, int32_t layers, int LS, F run) {
  const int64_t groups = ((2 * (int64_t)layers + LS - 1) / LS + 7) / 8 * 8;  // 2^16 at most
  const int64_t each = ((int64_t)1 << 23) / groups;
  for (int64_t first = 0; first < n; first += each) {
    const int64_t count = std::min(each, n - first);
    run(dim3((unsigned)(count * groups)), first, count);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

// ---- compact: row b's tokens start + path[i] to start + i for i < keep, ascending. A thread
// moves a 16-byte column of them: path ascends from 0 or more, so path[i] >= i and no token is
// overwritten before the same thread has read it. A workgroup does CP_LS (layer, side) pairs of
// a row; the slots are worked out once and lie in LDS, and tokens that stay are left out. Bound by
// HBM: what moves is read once and written once, past the L2 (through it, the write-back at the
// kernel's end makes 14.8 us 24.1). 69 MB in 14.8 us are 4.7 TB/s, a copy's rate is 5.2.
// 3 rows of 28 layers: 4.1 us, an empty launch 3.6.
constexpr int CP_PATH = TREE_MAX_NODES;
constexpr int CP_LS = 2;  // 1 or 4: 15.1 us

__global__ void __launch_bounds__(PGS_NT) compact_paged_kernel(CompactArgs a) {
  __shared__ int64_t sFrom[CP_PATH], sTo[CP_PATH];
  __shared__ int sN;
  const int tid = threadIdx.x;
  int ls0;
  const int64_t b = a.first + pgs_item(a.count, CP_LS, ls0);
  if (ls0 >= 2 * a.layers) return;  // uniform
  const int64_t keep = a.keep[b], start = a.start[b];
  const int64_t* const path = a.path + b * a.max_path;
  const int32_t* const table = a.table + b * a.max_blocks;
  int bad = keep < 0 || keep > a.max_path || start < 0 || start > a.max_blocks * a.bs;
  const bool tell = a.kept && ls0 == 0 && tid == 0;
  if (!bad && keep == 0) {  // uniform
    if (tell) a.kept[b] = 0;
    return;
  }
  int stay = 0;  // (the row's first tokens stay: path ascends)
  if (!bad) {
    auto slot = [&](int64_t pos) -> int64_t {
      if (pos >= a.max_blocks * a.bs) return -1;
      const int64_t page = table[pos / a.bs];
      return page < 0 || page >= a.num_blocks ? -1 : page * a.bs + pos % a.bs;
    };
    for (int64_t i = tid; i < keep; i += PGS_NT) {
      const int64_t p = path[i], before = i > 0 ? path[i - 1] : -1;
      bad |= p <= before || p > a.max_blocks * a.bs;
      if (bad) break;
      const int64_t from = slot(start + p), to = slot(start + i);
      bad |= from < 0 || to < 0;
      sFrom[i] = from * a.row_bytes;
      sTo[i] = to * a.row_bytes;
      stay += p == i;
    }
  }
  if (tid == 0) sN = 0;
  bad = __syncthreads_or(bad);
  if (tell) a.kept[b] = bad ? 0 : keep;
  if (bad) {  // uniform
    if (tid == 0 && a.error) *a.error = 1;
    return;
  }
  if (stay) atomicAdd(&sN, stay);
  __syncthreads();
  const int i0 = sN;
  const uint32_t upr = (uint32_t)(a.row_bytes / 16);
  const int sides = min(CP_LS, 2 * a.layers - ls0);
  for (uint32_t u = tid; u < sides * upr; u += PGS_NT) {
    const uint32_t ls = u / upr;
    uint8_t* const at = pgs_side(a.pool, a.layer_bytes, a.side_bytes, ls0 + ls) + (int64_t)(u - ls * upr) * 16;
    for (int64_t i = i0; i < keep; i += PGS_UN) {
      uint4 v[PGS_UN];
#pragma unroll
      for (int k = 0; k < PGS_UN; ++k)
        if (i + k < keep) v[k] = *reinterpret_cast<const uint4*>(at + sFrom[i + k]);
#pragma unroll
      for (int k = 0; k < PGS_UN; ++k)
        if (i + k < keep) store_nt(at + sTo[i + k], v[k]);
    }
  }
}

// ---- the pages that no table holds. FREE_RANGE pages' bits fit a workgroup's LDS; `parts`
// workgroups go through a share of the tables each and leave their bits, the second kernel
// joins them and lists the pages whose bit is clear, by ascending id. Bound by the latency of a
// few dependent loads and of two launches.
constexpr int FP_NT = 512;
constexpr int FP_SEG = 8192;  // pages that a workgroup of the second kernel lists
// Words that all workgroups of the list read (a square of the pages), beyond which a kernel that counts
// is cheaper. 320 entries, without it and with it: 2^18 pages 13.9 and 10.5 us, 2^20 30.4 and 11.0, 2^24 787
// and 35; 115,200 entries and 2^15 pages 15.3 and 13.0; 2^17 pages of 320 entries (at the rule) 10.7 without.
constexpr int64_t FP_COUNT = 1 << 16;

// The bits of pages base .. in sBits, from the workgroup's share of the tables.
__device__ __forceinline__ void fp_mark(const FreePagesArgs& a, int64_t base, int words, uint32_t* sBits) {
  const int tid = threadIdx.x;
  for (int w = tid; w < words; w += FP_NT) sBits[w] = 0;
  __syncthreads();
  const uint32_t n = (uint32_t)(a.batch * a.max_blocks), each = (n + a.parts - 1) / a.parts;
  const uint32_t e0 = min(n, blockIdx.y * each), e1 = min(n, e0 + each), mb = (uint32_t)a.max_blocks;
  int bad = 0;
  for (uint32_t e = e0 + tid; e < e1; e += FP_NT) {
    const int32_t page = a.table[e];
    bool held = page >= 0;
    if (a.kv_len) {
      const uint32_t b = e / mb;
      const int64_t kv = a.kv_len[b];
      held = (int64_t)(e - b * mb) * a.bs < kv;
      bad |= kv < 0 || kv > a.max_blocks * a.bs;
    }
    if (!held) continue;
    const int64_t x = (int64_t)page - base;
    if (page < 0 || page >= a.num_blocks) bad = 1;
    else if (x >= 0 && x < words * 32) atomicOr(&sBits[x / 32], 1u << (x % 32));
  }
  if (bad && a.error) *a.error = 1;
  __syncthreads();
}

__global__ void __launch_bounds__(FP_NT) free_pages_mark_kernel(FreePagesArgs a) {
  __shared__ uint32_t sBits[FREE_RANGE / 32];
  const int tid = threadIdx.x;
  const int64_t base = (int64_t)blockIdx.x * FREE_RANGE;
  const int words = (int)((min((int64_t)FREE_RANGE, a.num_blocks - base) + 31) / 32);
  fp_mark(a, base, words, sBits);
  uint32_t* const out = a.bits + (int64_t)blockIdx.y * a.words + base / 32;
  for (int w = tid; w < words; w += FP_NT) out[w] = sBits[w];
}

// Many pages: the parts are joined once, in the place of the first, and every segment's free pages
// counted, a workgroup each; a workgroup of the list then adds up counts and not all pages.
constexpr int FP_SW = FP_SEG / 32;  // words of a segment
__device__ __forceinline__ uint32_t fp_free(const FreePagesArgs& a, int64_t w) {  // word w's free pages
  uint32_t held = 0;
#pragma unroll 8
  for (int p = 0; p < a.parts; ++p) held |= a.bits[p * a.words + w];
  const int64_t left = a.num_blocks - w * 32;
  return ~held & (left >= 32 ? 0xFFFFFFFFu : (1u << left) - 1u);
}
__global__ void __launch_bounds__(FP_SW) free_pages_count_kernel(FreePagesArgs a) {
  constexpr int NW = FP_SW / kWave;
  __shared__ uint32_t sSum[NW];
  const int tid = threadIdx.x;
  const int64_t w = (int64_t)blockIdx.x * FP_SW + tid;
  const uint32_t mine = w < a.words ? fp_free(a, w) : 0u;
  if (w < a.words) a.bits[w] = ~mine;
  const uint32_t n = (uint32_t)wave_sum_u64(__popc(mine));
  if (tid % kWave == 0) sSum[tid / kWave] = n;
  __syncthreads();
  if (tid == 0) {
    uint32_t sum = 0;
#pragma unroll
    for (int k = 0; k < NW; ++k) sum += sSum[k];
    a.counts[blockIdx.x] = sum;
  }
}

// Few pages and few entries: one workgroup, a word per thread, does both.
__global__ void __launch_bounds__(FP_NT) free_pages_small_kernel(FreePagesArgs a) {
  constexpr int NW = FP_NT / kWave;
  __shared__ uint32_t sBits[FP_NT], sAt[FP_NT], sWave[NW];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wv = tid / kWave;
  fp_mark(a, 0, (int)a.words, sBits);
  const int left = (int)a.num_blocks - tid * 32;
  const uint32_t mine = tid < a.words ? ~sBits[tid] & (left >= 32 ? 0xFFFFFFFFu : (1u << left) - 1u) : 0u;
  const uint32_t n = (uint32_t)__popc(mine), inc = wave_incl_scan_u32(n, lane);
  if (lane == kWave - 1) sWave[wv] = inc;
  __syncthreads();
  uint32_t at = inc - n, total = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    if (w < wv) at += sWave[w];
    total += sWave[w];
  }
  sBits[tid] = mine;
  sAt[tid] = at;
  __syncthreads();
  if (tid == 0) *a.num_free = total;
  for (int x = tid; x < a.num_blocks; x += FP_NT) {
    const uint32_t bits = sBits[x / 32], bit = 1u << (x % 32);
    if (bits & bit) a.free_blocks[sAt[x / 32] + __popc(bits & (bit - 1))] = x;
    if (x >= (int)total) a.free_blocks[x] = -1;
  }
}

template <bool COUNTED>
__global__ void __launch_bounds__(FP_NT) free_pages_list_kernel(FreePagesArgs a) {
  constexpr int SW = FP_SW, NW = FP_NT / kWave;
  static_assert(SW <= FP_NT, "a word per thread");
  __shared__ uint32_t sFree[SW], sAt[SW], sWave[NW];
  __shared__ uint64_t sSum[NW][2];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wv = tid / kWave;
  const int64_t w0 = (int64_t)blockIdx.x * SW;
  uint64_t before = 0, total = 0;
  if constexpr (COUNTED) {
    for (int64_t k = tid; k < gridDim.x; k += FP_NT) {
      const uint32_t n = a.counts[k];
      total += n;
      if (k < blockIdx.x) before += n;
    }
  } else {
    for (int64_t w = tid; w < a.words; w += FP_NT) {
      const uint32_t n = (uint32_t)__popc(fp_free(a, w));
      total += n;
      if (w < w0) before += n;
    }
  }
  const uint32_t mine = tid < SW && w0 + tid < a.words ? fp_free(a, w0 + tid) : 0u;
  const uint32_t n = (uint32_t)__popc(mine);
  const uint32_t inc = wave_incl_scan_u32(n, lane);
  total = wave_sum_u64(total);
  before = wave_sum_u64(before);
  if (lane == kWave - 1) {
    sWave[wv] = inc;
    sSum[wv][0] = total, sSum[wv][1] = before;
  }
  __syncthreads();
  uint32_t at = inc - n;
  total = before = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    if (w < wv) at += sWave[w];
    total += sSum[w][0], before += sSum[w][1];
  }
  if (tid < SW) sFree[tid] = mine, sAt[tid] = at;
  __syncthreads();
  if (blockIdx.x == 0 && tid == 0) *a.num_free = (int64_t)total;
  const int64_t end = min(a.num_blocks, (w0 + SW) * 32);
  for (int64_t x = w0 * 32 + tid; x < end; x += FP_NT) {
    const int i = (int)(x - w0 * 32);
    const uint32_t bits = sFree[i / 32], bit = 1u << (i % 32);
    if (bits & bit) a.free_blocks[before + sAt[i / 32] + __popc(bits & (bit - 1))] = (int32_t)x;
    if (x >= (int64_t)total) a.free_blocks[x] = -1;
  }
}

// ---- tables of rows that go on from others. Row i goes on from row p = parent[i] of the old
// table: it shares p's whole pages; p's last page, filled in part, goes to one row alone, the
// first that goes on in it while none holds it whole, and the others get copies.
struct FkRow {
  int64_t p, len, whole, part;  // parent (-1: none), its tokens, whole pages, tokens behind them
  bool ok;
};
__device__ __forceinline__ FkRow fk_row(const ForkArgs& a, int64_t i) {
  FkRow r{a.parent[i], 0, 0, 0, true};
  if (r.p < 0) {
    r.ok = r.p == -1;
    return r;
  }
  if (r.p >= a.old_batch) {
    r.ok = false;
    return r;
  }
  r.len = a.kv_len[r.p];
  r.ok = r.len >= 0 && r.len <= a.max_blocks * a.bs;
  if (r.ok) {
    r.whole = r.len / a.bs;
    r.part = r.len - r.whole * a.bs;
  }
  return r;
}

// What a wave works out for new row i: how many pages it gets, with FK_COPY if it copies its first,
// or FK_BAD.
constexpr int FK_UN = 4;  // rows of a lane at a time
constexpr int32_t FK_COPY = 1 << 30, FK_BAD = (int32_t)0x80000000;
__device__ __forceinline__ int32_t fk_own(const ForkArgs& a, int64_t i, int lane) {
  const FkRow r = fk_row(a, i);
  const int64_t room = a.room[i];
  bool ok = r.ok && room >= r.len && room <= a.max_blocks * a.bs;
  bool copy = false;
  if (ok && r.part > 0) {  // uniform
    const int32_t page = a.table[r.p * a.max_blocks + r.whole];
    ok = page >= 0;
    int other = 0;
    for (int64_t j0 = lane; ok && j0 < a.batch; j0 += FK_UN * kWave) {  // three loads, one behind another
      int64_t p[FK_UN], len[FK_UN];
      int32_t g[FK_UN];
      bool holds[FK_UN];
#pragma unroll
      for (int k = 0; k < FK_UN; ++k) p[k] = a.parent[min(j0 + k * kWave, a.batch - 1)];
#pragma unroll
      for (int k = 0; k < FK_UN; ++k) {
        holds[k] = p[k] >= 0 && p[k] < a.old_batch && j0 + k * kWave < a.batch && j0 + k * kWave != i;
        len[k] = a.kv_len[holds[k] ? p[k] : r.p];
      }
#pragma unroll
      for (int k = 0; k < FK_UN; ++k) {
        // the row's page in this column: whole if its tokens pass the page, else filled in part
        holds[k] &= len[k] <= a.max_blocks * a.bs && (len[k] >= (r.whole + 1) * a.bs ||
                                                      (len[k] > r.whole * a.bs && j0 + k * kWave < i));
        g[k] = a.table[(holds[k] ? p[k] : r.p) * a.max_blocks + r.whole];
      }
#pragma unroll
      for (int k = 0; k < FK_UN; ++k) other |= holds[k] && g[k] == page;
    }
    copy = __any(other);
  }
  int hole = 0;
  for (int64_t c = lane; ok && c < r.whole; c += kWave) hole |= a.table[r.p * a.max_blocks + c] < 0;
  ok = ok && !__any(hole);
  const int64_t kept = r.whole + (r.part > 0 && !copy), need = ok ? (room + a.bs - 1) / a.bs : 0;
  return ok ? (int32_t)(need - kept) | (copy ? FK_COPY : 0) : FK_BAD;
}

// Free pages are taken in front of the first entry that is no page (free_page_list leaves -1 behind
// its last one). All rows together take batch * max_blocks at most, so a wave per new row looks at
// max_blocks of them, whatever the pool has: row i's first that is no page, as an index of its
// share, or FK_NONE. 1 us of a call: 16 rows of 60 pages 5.2 us without it and 6.1, 384 rows 7.8 and 8.9.
constexpr int32_t FK_NONE = 0x7FFFFFFF;
__device__ __forceinline__ int64_t fk_have(const ForkArgs& a) {
  return a.num_free ? min(*a.num_free, a.max_free) : a.max_free;
}
struct FkGap {
  int64_t first, most, have;
  int32_t g[FK_UN];  // the share's first entries
};
// asked for ahead of what the row takes: none of these loads waits for another
__device__ __forceinline__ FkGap fk_ask(const ForkArgs& a, int64_t i, int lane) {
  FkGap r;
  r.first = i * a.max_blocks;
  r.most = min(a.max_free - r.first, a.max_blocks);
  r.have = fk_have(a);
#pragma unroll
  for (int k = 0; k < FK_UN; ++k)
    r.g[k] = r.most > 0 ? a.free_blocks[r.first + min((int64_t)k * kWave + lane, r.most - 1)] : 0;
  return r;
}
__device__ __forceinline__ int32_t fk_gap(const ForkArgs& a, FkGap& r, int lane) {
  const int64_t n = min(r.have - r.first, r.most);
  for (int64_t c0 = 0; c0 < n;) {  // uniform
#pragma unroll
    for (int k = 0; k < FK_UN; ++k) {
      const uint64_t none = __ballot(c0 + k * kWave + lane < n && r.g[k] < 0);
      if (none) return (int32_t)(c0 + k * kWave) + __ffsll((unsigned long long)none) - 1;
    }
    c0 += FK_UN * kWave;
    if (c0 >= n) break;
#pragma unroll
    for (int k = 0; k < FK_UN; ++k) r.g[k] = a.free_blocks[r.first + min(c0 + k * kWave + lane, n - 1)];
  }
  return FK_NONE;
}

// New row i's table and copy, by `step` threads, of which this is thread t: x from fk_own, `before`
// the pages of the rows in front of it, all the rows' pages.
__device__ __forceinline__ void fk_put(const ForkArgs& a, int64_t i, int32_t x, uint64_t before, uint64_t total,
                                       bool bad, int t, int step) {
  bad |= (int64_t)total > fk_have(a);
  const FkRow r = fk_row(a, i);
  const bool copy = x & FK_COPY;
  const int64_t kept = r.whole + (r.part > 0 && !copy), end = kept + (x & (FK_COPY - 1));
  if (t == 0) {
    if (i == 0) {
      *a.used = bad ? 0 : (int64_t)total;
      if (bad && a.error) *a.error = 1;
    }
    const bool c = !bad && copy;
    a.copies[i] = c ? a.table[r.p * a.max_blocks + r.whole] : -1;
    a.copies[a.batch + i] = c ? a.free_blocks[before] : -1;
    a.copies[2 * a.batch + i] = c ? (int32_t)r.part : 0;
  }
  int32_t* const out = a.out + i * a.max_blocks;
  for (int64_t c = t; c < a.max_blocks; c += step) {
    int32_t v = -1;
    if (!bad && c < end) v = c < kept ? a.table[r.p * a.max_blocks + c] : a.free_blocks[before + c - kept];
    out[c] = v;
  }
}

// Few rows: one workgroup, a wave per row, in place of two launches. 16 rows of 60 pages: 6.1 us and
// 7.4, 4 rows 4.8 and 7.1, 16 rows of 512 pages 8.3 and 8.6, of 1,024 11.1 and 10.1.
constexpr int FK_SMALL = 16;
constexpr int64_t FK_SMALL_BLOCKS = 512;
__global__ void __launch_bounds__(FK_SMALL * kWave) fork_small_kernel(ForkArgs a) {
  __shared__ int32_t sOwn[FK_SMALL], sGap[FK_SMALL];
  const int lane = threadIdx.x & (kWave - 1), i = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  if (i < a.batch) {  // uniform per wave
    FkGap ask = fk_ask(a, i, lane);
    const int32_t x = fk_own(a, i, lane), gap = fk_gap(a, ask, lane);
    if (lane == 0) sOwn[i] = x, sGap[i] = gap;
  }
  __syncthreads();
  const int32_t x = lane < a.batch ? sOwn[lane] : 0, gap = lane < a.batch ? sGap[lane] : FK_NONE;
  const uint32_t n = (uint32_t)x & (FK_COPY - 1), inc = wave_incl_scan_u32(n, lane);
  const uint32_t total = rdlane(inc, kWave - 1);
  const bool bad = __any(x < 0 || (gap != FK_NONE && lane * a.max_blocks + gap < (int64_t)total));
  if (i < a.batch)
    fk_put(a, i, (int32_t)rdlane((uint32_t)x, i), rdlane(inc - n, i), total, bad, lane, kWave);
}

// Many rows: a wave per new row, then a workgroup per row, which sums what those in front of it take.
__global__ void __launch_bounds__(PGS_NT) fork_rows_kernel(ForkArgs a) {
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t i = (int64_t)blockIdx.x * (PGS_NT / kWave) + threadIdx.x / kWave;
  if (i >= a.batch) return;  // uniform per wave
  FkGap ask = fk_ask(a, i, lane);
  const int32_t x = fk_own(a, i, lane), gap = fk_gap(a, ask, lane);
  if (lane == 0) a.own[i] = x, a.gap[i] = gap;
}

__global__ void __launch_bounds__(PGS_NT) fork_tables_kernel(ForkArgs a) {
  constexpr int NW = PGS_NT / kWave;
  __shared__ uint64_t sSum[NW][2];
  const int tid = threadIdx.x;
  const int64_t i = blockIdx.x;
  uint64_t total = 0, before = 0;
  int64_t none = INT64_MAX;  // first entry that is no page
  int bad = 0;
  for (int64_t j = tid; j < a.batch; j += PGS_NT) {
    const int32_t x = a.own[j], gap = a.gap[j];
    bad |= x < 0;
    if (gap != FK_NONE) none = min(none, j * a.max_blocks + gap);
    const uint64_t n = (uint32_t)x & (FK_COPY - 1);
    total += n;
    if (j < i) before += n;
  }
  total = wave_sum_u64(total);
  before = wave_sum_u64(before);
  if ((tid & (kWave - 1)) == 0) sSum[tid / kWave][0] = total, sSum[tid / kWave][1] = before;
  bad = __syncthreads_or(bad);
  total = before = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) total += sSum[w][0], before += sSum[w][1];
  bad |= __syncthreads_or(none < (int64_t)total);
  fk_put(a, i, a.own[i], before, total, bad != 0, tid, PGS_NT);
}

// ---- copies of pages: entry e's first tokens[e] tokens from page to page, in every layer and
// side. They lie one behind another on both sides. Bound by HBM, stored past the L2 as above:
// 139 copies of 1,149 tokens from 727, in 36 layers of 4 heads of 128, take 25 us (138 MB, 5.5
// TB/s); beams freed, forked and copied through it took 63 us, not 39.
constexpr int CY_LS = 1;  // 2: 42 us in place of 39
__global__ void __launch_bounds__(PGS_NT) copy_pages_kernel(CopyPagesArgs a) {
  int ls0;
  const int64_t e = a.first + pgs_item(a.count, CY_LS, ls0);
  if (ls0 >= 2 * a.layers) return;  // uniform
  const int32_t from = a.copies[e], to = a.copies[a.n + e], tokens = a.copies[2 * a.n + e];
  if (from < 0 || to < 0 || tokens == 0) return;  // uniform
  if (from >= a.num_blocks || to >= a.num_blocks || tokens < 0 || tokens > a.bs) {
    if (threadIdx.x == 0 && a.error) *a.error = 1;
    return;
  }
  const int64_t page = a.bs * a.row_bytes;
  const uint32_t upr = (uint32_t)(tokens * (a.row_bytes / 16));
  const int sides = min(CY_LS, 2 * a.layers - ls0);
  for (uint32_t u0 = threadIdx.x; u0 < sides * upr; u0 += PGS_NT * PGS_UN) {
    uint4 v[PGS_UN];
    uint8_t* dst[PGS_UN];
#pragma unroll
    for (int k = 0; k < PGS_UN; ++k) {
      const uint32_t u = u0 + k * PGS_NT;
      dst[k] = nullptr;
      if (u >= sides * upr) continue;
      const uint32_t ls = u / upr;
      uint8_t* const at = pgs_side(a.pool, a.layer_bytes, a.side_bytes, ls0 + ls) + (int64_t)(u - ls * upr) * 16;
      v[k] = *reinterpret_cast<const uint4*>(at + from * page);
      dst[k] = at + to * page;
    }
#pragma unroll
    for (int k = 0; k < PGS_UN; ++k)
      if (dst[k]) store_nt(dst[k], v[k]);
  }
}

// ---------------------------------------------------------------- launches
hipError_t launch_compact_paged(const CompactArgs& a, hipStream_t s) {
  return pgs_launch(a.batch, a.layers, CP_LS, [&](dim3 grid, int64_t first, int64_t count) {
    CompactArgs b = a;
    b.first = first, b.count = count;
    hipLaunchKernelGGL(compact_paged_kernel, grid, dim3(PGS_NT), 0, s, b);
  });
}

// a workgroup for every 1,024 entries, as far as their bits stay under 16 MB
int free_pages_parts(int64_t entries, int64_t words) {
  return (int)std::max<int64_t>(1, std::min<int64_t>({64, entries / 1024, (1 << 22) / words}));
}

int64_t free_pages_segments(int64_t num_blocks) { return (num_blocks + FP_SEG - 1) / FP_SEG; }

hipError_t launch_free_pages(const FreePagesArgs& a, hipStream_t s) {
  // One part (under 2,048 entries) and a word per thread: in one kernel 912 entries and 900 pages take
  // 3.2 us, in two 4.9; at the end of the rule, 16,384 pages, 7.3 and 7.5.
  if (a.parts == 1 && a.num_blocks <= FP_NT * 32) {
    hipLaunchKernelGGL(free_pages_small_kernel, dim3(1), dim3(FP_NT), 0, s, a);
    return hipGetLastError();
  }
  const unsigned ranges = (unsigned)((a.num_blocks + FREE_RANGE - 1) / FREE_RANGE);
  hipLaunchKernelGGL(free_pages_mark_kernel, dim3(ranges, (unsigned)a.parts), dim3(FP_NT), 0, s, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int64_t segments = free_pages_segments(a.num_blocks);
  if (a.parts * a.words * segments <= FP_COUNT) {
    hipLaunchKernelGGL(free_pages_list_kernel<false>, dim3((unsigned)segments), dim3(FP_NT), 0, s, a);
    return hipGetLastError();
  }
  hipLaunchKernelGGL(free_pages_count_kernel, dim3((unsigned)segments), dim3(FP_SW), 0, s, a);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  FreePagesArgs b = a;
  b.parts = 1;
  hipLaunchKernelGGL(free_pages_list_kernel<true>, dim3((unsigned)segments), dim3(FP_NT), 0, s, b);
  return hipGetLastError();
}

hipError_t launch_fork_tables(const ForkArgs& a, hipStream_t s) {
  if (a.batch <= FK_SMALL && a.max_blocks <= FK_SMALL_BLOCKS) {
    hipLaunchKernelGGL(fork_small_kernel, dim3(1), dim3(FK_SMALL * kWave), 0, s, a);
    return hipGetLastError();
  }
  constexpr int rows = PGS_NT / kWave;
  hipLaunchKernelGGL(fork_rows_kernel, dim3((unsigned)((a.batch + rows - 1) / rows)), dim3(PGS_NT), 0, s, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(fork_tables_kernel, dim3((unsigned)a.batch), dim3(PGS_NT), 0, s, a);
  return hipGetLastError();
}

hipError_t launch_copy_pages(const CopyPagesArgs& a, hipStream_t s) {
  return pgs_launch(a.n, a.layers, CY_LS, [&](dim3 grid, int64_t first, int64_t count) {
    CopyPagesArgs b = a;
    b.first = first, b.count = count;
    hipLaunchKernelGGL(copy_pages_kernel, grid, dim3(PGS_NT), 0, s, b);
  });
}

}  // namespace sdx
