// Attention of a batch whose rows share prefixes over the paged cache, one layer: the
// multi-query attention of sdx_attn.hip (bench/bench_engine.py:170-174, the mask of
// specdec/kvcache.py:138-162) for groups of rows that hold a prefix's keys once.
//
// out_t = sum_s p_s v_s / sum_s p_s,  p_s = 2^(scale log2(e) q_t k_s - m), over the keys
// s < P of the group's first row and P <= s of the row itself, s <= kv_len - q_b + j.
// The two ranges are segments with their own running maximum and sum: a group's prefix
// against all of the group's queries, a row's own keys against the row's.
//
// A segment's query rows (tokens x the query heads of a KV head) against its keys are cut
// into units: a tile of 128 query rows, a chunk of keys, a KV head. The four waves of a
// workgroup hold 32 query rows each and share 64-key tiles in LDS, which all of them load.
// Few rows leave waves without any: such units are bound by the read of the keys, full ones by
// the matrix instructions and the exponentials. (A form for up to 32 rows, in which every wave
// held them all and took 32 keys of each 128 by itself, was measured beside it: 8 rows behind
// 65,536 keys 79.7 us, now 71.0; 128 rows of up to 8,192 own keys, 2.08 GB, 426, now 414; 4 rows
// behind 2,000 keys 21.8 and 21.9; 2 rows of one KV head behind 12,000 keys 23.3, now 24.5.)
// S^T = K Q^T with v_mfma_f32_32x32x16: lane l then holds 16 keys' scores of
// query l % 32, so maxima and sums stay in the lane (one exchange with lane l ^ 32), and
// the weights, rounded to 16 bits, are the second operand of O^T = V^T P^T as they lie:
// its 16 keys are contracted in the order in which the scores hold them. V is read from
// its rows in LDS by the transposing 64-bit reads. The rounding of the weights is the second
// product's price: matrix instructions take 16-bit operands, two halves of each weight would double
// them. The running maximum moves only when a score passes it by 2^8 (weights up to 2^8 lose
// nothing), which spares rescaling O.
//
// A plan kernel of one workgroup lists the units from the lengths. A fixed grid takes them
// from eight queues, one for each XCD's share, so that the units of one chunk of keys read
// it from one L2: the groups' long ones first, then the rows'. A unit leaves (O, max, sum)
// in fp32, a third kernel joins them; a row without a prefix whose keys fit one unit is
// written directly.
//
// Measured, 32 query heads on 8 KV heads of 128, bf16, whole calls: a prefix of 16,384 under
// 128 rows of up to 9 tokens with up to 1,024 own keys 261 us, 710 TFLOP/s; 64 rows behind 4,096
// keys 70; 4 rows of one token behind 2,000 keys 20 (plan 6 to 8, units 8, join 4); 128 rows of up
// to 8,192 own keys behind a prefix of 16, 2.08 GB, 414, 5.0 TB/s, with one token each 5.8. A unit's
// keys do not stop where its query tile's view does: a prompt of 16,384 tokens takes 4.92 ms, 447
// TFLOP/s of the products that its mask leaves, about half of those done; and one row inside its
// prefix has the tiles of all groups masked (64 rows' step of 72 us beside a prompt of 4,096 tokens
// of 340: 392 us, 440 where that row shares the prompt). A tile takes 3,900 clocks of the two
// workgroups of a CU: QK 680, mask and softmax 910, PV 800, what is left the staging and its
// waits; 64 matrix instructions a SIMD are 2,048 of them, so the exponentials and the staging
// bound it. Tried: PV of the tile before among the exponentials (spills, 246 -> 283 us without
// own keys), staging between the products and the softmax (the same), the next unit asked for
// early (2 to 5% slower), units of rows among the groups' from the start (64 rows 73 -> 71, the
// longest 306 -> 330).
#include <algorithm>
#include <type_traits>

#include "sdx_attn_tile.hpp"

namespace sdx {

constexpr int PA_GRID = 512;      // two workgroups on each of 256 CUs
constexpr uint32_t PA_ASK = 0xFFFFFFFFu;
constexpr int PA_QUEUE = 32;      // words between the queues' heads
constexpr int PA_ZERO = 8 * PA_QUEUE;  // word of the head where a row of zeros lies
// ---- the batch's shape

// the call's lengths and offsets, in memory or copied to LDS
struct PaShape {
  const int64_t *cu_q, *kv_len, *cu_group, *prefix_len;
};
struct PaGroup {
  int64_t first, rows, prefix;  // rows of the batch, and their shared keys (0 in a group of one)
  int64_t t0, nt;               // tokens
  bool ok;
};
__device__ __forceinline__ PaGroup pa_group(const PrefixAttnArgs& a, const PaShape& c, int64_t g) {
  PaGroup r;
  const int64_t f = c.cu_group[g], e = c.cu_group[g + 1], p = c.prefix_len[g];
  r.first = f;
  r.rows = e - f;
  r.ok = f >= 0 && e >= f && e <= a.batch && p >= 0 && p <= a.max_blocks * a.bs;
  r.prefix = r.ok && r.rows > 1 ? p : 0;
  r.t0 = r.nt = 0;
  if (r.ok) {
    const int64_t t0 = c.cu_q[f], t1 = c.cu_q[e];
    r.ok = t0 >= 0 && t1 >= t0 && t1 <= a.tokens;
    if (r.ok) r.t0 = t0, r.nt = t1 - t0;
  }
  return r;
}
struct PaRow {
  int64_t t0, nt, kv, prefix, group;
  bool ok;
};
__device__ __forceinline__ PaRow pa_row(const PrefixAttnArgs& a, const PaShape& c, int64_t b) {
  PaRow r;
  r.group = pa_find(c.cu_group, a.groups, b);
  const PaGroup gr = pa_group(a, c, r.group);
  const int64_t t0 = c.cu_q[b], t1 = c.cu_q[b + 1];
  r.kv = c.kv_len[b];
  r.t0 = t0;
  r.nt = t1 - t0;
  r.prefix = gr.prefix;
  r.ok = gr.ok && b >= gr.first && b < gr.first + gr.rows && t0 >= gr.t0 && t1 >= t0 &&
         t1 <= gr.t0 + gr.nt && r.kv >= r.nt && r.kv <= a.max_blocks * a.bs;
  return r;
}

// A segment's size: tiles of query rows, 64-key tiles.
struct PaSeg {
  int32_t qt, kt;
};
__device__ __forceinline__ PaSeg pa_seg(const PrefixAttnArgs& a, int64_t nt, int64_t keys) {
  PaSeg s;
  const int64_t m = nt * a.group;
  s.qt = keys > 0 ? (int32_t)((m + PA_ROWS - 1) / PA_ROWS) : 0;
  s.kt = s.qt > 0 ? (int32_t)((keys + PA_TILE - 1) / PA_TILE) : 0;
  return s;
}

// ---- plan: one workgroup lists the units, resets the queues and notes the parts of every
// token for the join. Work is counted in 64-key tiles.
constexpr int PL_NT = 512;
constexpr int PL_CAND = 32;      // chunk sizes weighed for the groups
constexpr int PA_UNIT = 8;       // what a unit costs beside its tiles, the write of its part first
                                 // (4 or 16: within 3% of it)
constexpr int PL_OWN = 8;        // entries that a thread writes by itself

// f(x, k) for k < n of every lane's x (words): a lane's first few by itself, the rest by the
// wave. All lanes of the wave call it.
template <int W, class F>
__device__ __forceinline__ void pl_each(const int32_t (&x)[W], int32_t n, F f) {
  for (int k = 0; k < min(n, PL_OWN); ++k) f(x, k);
  uint64_t big = __ballot(n > PL_OWN);
  while (big) {  // uniform
    const int src = __ffsll((unsigned long long)big) - 1;
    big &= big - 1;
    int32_t y[W];
#pragma unroll
    for (int i = 0; i < W; ++i) y[i] = __shfl(x[i], src, kWave);
    const int32_t m = __shfl(n, src, kWave);
    for (int k = PL_OWN + (threadIdx.x & (kWave - 1)); k < m; k += kWave) f(y, k);
  }
}

// tiles per chunk of a segment of kt tiles for equal chunks of about c tiles
__device__ __forceinline__ int32_t pl_chunk(int32_t kt, int32_t c) {
  const int32_t n = (kt + c - 1) / c;
  return (kt + n - 1) / n;
}

// What the workgroup sums up over its threads, one wave's record after another in LDS.
struct PlSum {
  uint64_t cost;
  uint32_t most, most_row, flags;  // flags: 1 an error, 2 a token before the prefix's end
};

// The plan's steps are short and depend on each other, so its time is that of its rounds of
// loads (one, where the batch fits LDS) and barriers (four). 4 rows 6 to 8 us, 128 rows 9 to 10,
// of them 2 the launch's own.
__global__ void __launch_bounds__(PL_NT) prefix_attn_plan_kernel(PrefixAttnArgs a) {
  constexpr int NW = PL_NT / kWave;
  __shared__ PlSum sSum[NW];
  __shared__ uint64_t sScan[2][NW];
  __shared__ uint32_t sUnits[PL_CAND];
  __shared__ int64_t sQ[PL_NT + 1], sKv[PL_NT], sGroup[PL_NT + 1], sPrefix[PL_NT];
  __shared__ int2 sSeg[PL_NT];
  __shared__ int32_t sGroupItem[PL_NT][8], sRowItem[PL_NT][8];  // and the first entry of each
  __shared__ uint32_t sGroupAt[PL_NT], sRowAt[PL_NT];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wv = tid / kWave;
  const int32_t half = a.parts / 2;
  // one round of loads where the batch fits: everything after it reads LDS
  PaShape c{a.cu_q, a.kv_len, a.cu_group, a.prefix_len};
  const bool rows_fit = a.batch <= PL_NT, groups_fit = a.groups <= PL_NT;
  if (rows_fit) {
    c.cu_q = sQ;
    c.kv_len = sKv;
    sQ[tid] = a.cu_q[min((int64_t)tid, a.batch)];
    if (tid == 0) sQ[PL_NT] = a.cu_q[a.batch];
    sKv[tid] = a.kv_len[min((int64_t)tid, a.batch - 1)];
  }
  if (groups_fit) {
    c.cu_group = sGroup;
    c.prefix_len = sPrefix;
    sGroup[tid] = a.cu_group[min((int64_t)tid, a.groups)];
    if (tid == 0) sGroup[PL_NT] = a.cu_group[a.groups];
    sPrefix[tid] = a.prefix_len[min((int64_t)tid, a.groups - 1)];
  }
  int2* const seg = groups_fit ? sSeg : a.group_seg;  // query tiles, key tiles
  if (tid < 8) a.head[PA_QUEUE * tid] = PA_GRID / 8;
  if (tid < 64) a.head[PA_ZERO + tid] = 0;
  if (tid < PL_CAND) sUnits[tid] = 0;
  for (int64_t t = tid; t < a.tokens; t += PL_NT) a.token_parts[t] = 0;
  __syncthreads();

  // sizes
  PlSum sum = {};
  if (tid == 0 && (c.cu_group[0] != 0 || c.cu_group[a.groups] != a.batch)) sum.flags = 1;
  PaGroup group0 = {};
  PaRow row0 = {};
  for (int64_t g = tid; g < a.groups; g += PL_NT) {
    const PaGroup r = pa_group(a, c, g);
    if (g == tid) group0 = r;
    const PaSeg s = pa_seg(a, r.nt, r.prefix);
    if (!r.ok) sum.flags |= 1;
    sum.cost += (uint64_t)s.qt * s.kt;
    sum.most = max(sum.most, (uint32_t)s.kt);
    seg[g] = make_int2(s.qt, s.kt);
  }
  for (int64_t b = tid; b < a.batch; b += PL_NT) {
    const PaRow r = pa_row(a, c, b);
    if (b == tid) row0 = r;
    if (!r.ok) {
      sum.flags |= 1;
      continue;
    }
    const PaSeg s = pa_seg(a, r.nt, max((int64_t)0, r.kv - r.prefix));
    if (r.nt > 0 && r.kv - r.nt < r.prefix - 1) sum.flags |= 2;
    sum.cost += (uint64_t)s.qt * s.kt;
    sum.most_row = max(sum.most_row, (uint32_t)s.kt);
  }
  sum.cost = wave_sum_u64(sum.cost);
  sum.most = wave_max_u32(sum.most);
  sum.most_row = wave_max_u32(sum.most_row);
  sum.flags = (__any(sum.flags & 1) ? 1 : 0) | (__any(sum.flags & 2) ? 2 : 0);
  if (lane == 0) sSum[wv] = sum;
  __syncthreads();
  sum = sSum[0];
#pragma unroll
  for (int w = 1; w < NW; ++w) {
    sum.cost += sSum[w].cost;
    sum.most = max(sum.most, sSum[w].most);
    sum.most_row = max(sum.most_row, sSum[w].most_row);
    sum.flags |= sSum[w].flags;
  }

  // chunks of the groups: of the sizes most / 1, most / 2, ... the one whose units, dealt to
  // the grid round by round, are done first. A candidate for each pair of lanes; of many
  // groups every wave takes some.
  const int cand = lane % PL_CAND;
  // 1 .. 16, then to 224 in growing steps; no chunk below two tiles (one: the same times)
  auto cut = [](int i) { return i < 16 ? i + 1 : (16 + (i & 3) * 4) << ((i - 16) >> 2); };
  auto size = [&](int i) { return max(2, (int)((sum.most + cut(i) - 1) / cut(i))); };
  int32_t cg;
  {
    const int32_t mine = size(cand);
    const bool few = a.groups <= 32;
    uint32_t n = 0;
    for (int64_t g = few ? lane / PL_CAND : tid / PL_CAND; g < a.groups; g += few ? 2 : PL_NT / PL_CAND) {
      const int2 s = seg[g];
      if (s.y <= 0) continue;
      n += (uint32_t)s.x * ((s.y + mine - 1) / mine);
    }
    n *= (uint32_t)a.hkv;
    if (few) {
      n += (uint32_t)__shfl_xor((int)n, 32, kWave);
    } else {  // uniform
      atomicAdd(&sUnits[cand], n);
      __syncthreads();
      n = sUnits[cand];
    }
    const uint32_t rounds = (n + PA_GRID - 1) / PA_GRID;
    // in eighths of a tile: the rounds, and the join's read of the parts
    const uint64_t t = (uint64_t)rounds * (mine + PA_UNIT) * 8 + cut(cand);
    uint32_t best = cut(cand) <= half ? (uint32_t)min(t, (uint64_t)0x3FFFFFF) << 5 | cand : 0xFFFFFFFFu;
    best = ~wave_max_u32(~best);
    cg = size((int)(best & (PL_CAND - 1)));
  }
  // chunks of the rows: several per workgroup, which level out, but not below 8 tiles (of a
  // part's cost) where the grid is full without
  const uint64_t each = (sum.cost * a.hkv + PA_GRID - 1) / PA_GRID;
  const uint64_t k6 = max(max(min(each, (uint64_t)8), each / 6), (uint64_t)2);
  const int32_t cr = (int32_t)min(max(k6, (uint64_t)(sum.most_row + half - 1) / half), (uint64_t)0x3FFFFFFF);

  // entries: of the groups (the query tiles of a chunk follow each other), then of the rows
  uint32_t ngroup = 0, nrow = 0;  // of the threads' items so far
  auto group_item = [&](int64_t g, int32_t (&x)[7]) -> uint32_t {
    if (g >= a.groups) return 0;
    const PaGroup r = g == tid ? group0 : pa_group(a, c, g);
    const PaSeg s = pa_seg(a, r.nt, r.prefix);
    if (s.qt == 0) {
      a.group_seg[g].x = 0;
      return 0;
    }
    const int32_t k = pl_chunk(s.kt, cg), n = (s.kt + k - 1) / k;
    x[0] = (int32_t)r.first, x[1] = (int32_t)r.prefix, x[2] = (int32_t)r.t0, x[3] = s.qt, x[4] = k;
    x[5] = (int32_t)(r.nt * a.group);
    a.group_seg[g].x = n;
    return (uint32_t)s.qt * n;
  };
  int32_t row_t0 = 0, row_nt = 0, row_parts = 0;
  auto row_item = [&](int64_t b, int32_t (&x)[9]) -> uint32_t {
    row_nt = row_parts = 0;
    if (b >= a.batch) return 0;
    const PaRow r = b == tid ? row0 : pa_row(a, c, b);
    if (!r.ok) return 0;
    const PaSeg s = pa_seg(a, r.nt, max((int64_t)0, r.kv - r.prefix));
    row_t0 = (int32_t)r.t0, row_nt = (int32_t)r.nt;
    if (s.qt == 0) return 0;
    const int32_t k = pl_chunk(s.kt, cr), n = (s.kt + k - 1) / k;
    x[0] = (int32_t)b, x[1] = (int32_t)r.prefix, x[2] = (int32_t)r.t0, x[3] = s.qt, x[4] = k;
    x[5] = (int32_t)r.nt, x[6] = (int32_t)r.kv, x[7] = r.prefix == 0 && n == 1;
    row_parts = n;
    return (uint32_t)s.qt * n;
  };
  auto put_group = [&](const int32_t (&z)[7], int32_t k) {
    const int32_t ch = (int32_t)((uint32_t)k / (uint32_t)z[3]), qt = k - ch * z[3];
    PrefixAttnUnit u;
    u.table = z[0];
    u.key0 = ch * z[4] * PA_TILE;
    u.n = min(z[4] * PA_TILE, z[1] - u.key0);
    u.t0 = z[2];
    u.r0 = qt * PA_ROWS;
    u.m = min(PA_ROWS, z[5] - u.r0);
    u.base = 0x7FFFFFFF;
    u.part = ch | PA_GROUP;
    a.entries[z[6] + k] = u;
  };
  auto put_row = [&](const int32_t (&z)[9], int32_t k) {
    const int32_t ch = (int32_t)((uint32_t)k / (uint32_t)z[3]), qt = k - ch * z[3];
    PrefixAttnUnit u;
    u.table = z[0];
    u.key0 = z[1] + ch * z[4] * PA_TILE;
    u.n = min(z[4] * PA_TILE, z[6] - u.key0);
    u.t0 = z[2];
    u.r0 = qt * PA_ROWS;
    u.m = min(PA_ROWS, z[5] * a.group - u.r0);
    u.base = z[6] - z[5];
    u.part = (a.parts / 2 + ch) | (z[7] ? PA_DIRECT : 0);
    a.entries[z[8] + k] = u;
  };
  auto note_tokens = [&](int64_t b) {  // after the groups' parts are known
    if (row_nt > 0) {
      const PaRow& r = row0;
      const int64_t g = b == tid ? r.group : pa_find(c.cu_group, a.groups, b);
      const int64_t prefix = b == tid ? r.prefix : pa_group(a, c, g).prefix;
      const int32_t np = prefix > 0 ? a.group_seg[g].x : 0;
      row_parts = np == 0 && row_parts == 1 ? 0 : np | row_parts << 16;  // one part: written directly
    }
    const int32_t v[2] = {row_t0, row_parts};
    pl_each(v, row_parts ? row_nt : 0,
            [&](const int32_t (&z)[2], int32_t k) { a.token_parts[z[0] + k] = (uint32_t)z[1]; });
  };
  // one scan of both counts, for as many blocks of PL_NT items as the larger of them has
  auto scan = [&](uint32_t x, uint32_t y, uint32_t* ex, uint32_t* ey, int par) {
    const uint64_t v = (uint64_t)x | (uint64_t)y << 32, inc = wave_incl_scan_u64(v, lane);
    if (lane == kWave - 1) sScan[par][wv] = inc;
    __syncthreads();
    uint64_t before = inc - v, total = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      if (w < wv) before += sScan[par][w];
      total += sScan[par][w];
    }
    *ex = (uint32_t)before, *ey = (uint32_t)(before >> 32);
    return total;
  };
  if (rows_fit && groups_fit) {
    int32_t x[7] = {}, y[9] = {};
    const uint32_t n = group_item(tid, x), m = row_item(tid, y);
    uint32_t ex, ey;
    const uint64_t total = scan(n, m, &ex, &ey, 0);
    ngroup = (uint32_t)total, nrow = (uint32_t)(total >> 32);
    if ((int64_t)ngroup + nrow <= a.max_entries) {  // uniform
      // an entry per thread, which finds its item by its place: 2,300 clocks with 4 rows or 12
      // groups; every item's by the thread that has it and its wave took 3,450 and 7,600
      x[6] = (int32_t)ex;
      y[8] = (int32_t)(ngroup + ey);
      sGroupAt[tid] = ex;
      sRowAt[tid] = ey;
#pragma unroll
      for (int i = 0; i < 7; ++i) sGroupItem[tid][i] = x[i];
#pragma unroll
      for (int i = 0; i < 8; ++i) sRowItem[tid][i] = y[i];
      __syncthreads();
      auto find = [&](const uint32_t* at, int len, uint32_t e) {  // the last that starts at e or before
        int i = 0;
        for (; len > 1; len -= len / 2)
          if (at[i + len / 2] <= e) i += len / 2;
        return i;
      };
      for (uint32_t e = tid; e < ngroup + nrow; e += PL_NT) {
        if (e < ngroup) {
          const int i = find(sGroupAt, (int)a.groups, e);
          int32_t z[7];
#pragma unroll
          for (int j = 0; j < 7; ++j) z[j] = sGroupItem[i][j];
          put_group(z, (int32_t)(e - sGroupAt[i]));
        } else {
          const int i = find(sRowAt, (int)a.batch, e - ngroup);
          int32_t z[9];
#pragma unroll
          for (int j = 0; j < 8; ++j) z[j] = sRowItem[i][j];
          z[8] = (int32_t)(ngroup + sRowAt[i]);
          put_row(z, (int32_t)(e - ngroup - sRowAt[i]));
        }
      }
      note_tokens(tid);
    }
  } else {
    int par = 0;
    for (int64_t i = 0; i < a.groups; i += PL_NT, par ^= 1) {  // uniform
      int32_t x[7] = {};
      const uint32_t n = group_item(i + tid, x);
      uint32_t ex, ey;
      const uint32_t total = (uint32_t)scan(n, 0, &ex, &ey, par);
      x[6] = (int32_t)(ngroup + ex);
      ngroup += total;
      if (ngroup > a.max_entries) break;
      pl_each(x, (int32_t)n, put_group);
    }
    __syncthreads();  // group_seg holds the groups' parts
    for (int64_t i = 0; i < a.batch && (int64_t)ngroup + nrow <= a.max_entries; i += PL_NT, par ^= 1) {
      int32_t y[9] = {};
      const uint32_t n = row_item(i + tid, y);
      uint32_t ex, ey;
      const uint32_t total = (uint32_t)scan(n, 0, &ex, &ey, par);
      y[8] = (int32_t)(ngroup + nrow + ex);
      nrow += total;
      if ((int64_t)ngroup + nrow > a.max_entries) break;
      pl_each(y, (int32_t)n, put_row);
      note_tokens(i + tid);
    }
  }
  // more entries than there is room for: rows that share tokens, offsets out of order
  const bool none = (int64_t)ngroup + nrow > a.max_entries;
  if (tid == 0) {
    a.head[1] = none ? 0 : (int32_t)(ngroup * a.hkv);
    a.head[2] = none ? 0 : (int32_t)(nrow * a.hkv);
    a.head[3] = (sum.flags & 2) != 0;
    if ((none || (sum.flags & 1)) && a.error) *a.error = 1;
  }
  if (none) {  // uniform: nothing is computed, nothing is joined
    __syncthreads();
    for (int64_t t = tid; t < a.tokens; t += PL_NT) a.token_parts[t] = 0;
  }
}

struct PaUnit {
  int64_t table, key0, t0, base;
  int32_t n, r0, m, kvh, part;
  bool group, direct;
};
// Unit u: of the groups first (KV head slowest), then of the rows (KV head fastest).
__device__ __forceinline__ PaUnit pa_unit(const PrefixAttnArgs& a, uint32_t u, uint32_t ng) {
  uint32_t e;
  PaUnit r;
  if (u < ng) {
    const uint32_t entries = ng / (uint32_t)a.hkv;
    e = u % entries;
    r.kvh = (int32_t)(u / entries);
  } else {
    e = ng / (uint32_t)a.hkv + (u - ng) / (uint32_t)a.hkv;
    r.kvh = (int32_t)((u - ng) % (uint32_t)a.hkv);
  }
  const PrefixAttnUnit x = a.entries[e];
  r.table = x.table, r.key0 = x.key0, r.t0 = x.t0, r.base = x.base;
  r.n = x.n, r.r0 = x.r0, r.m = x.m;
  r.part = x.part & PA_PART;
  r.group = x.part & PA_GROUP;
  r.direct = x.part & PA_DIRECT;
  return r;
}

// ---- a unit's arithmetic

// Scores of keys past the lane's lim: keys t0 + 32 nb + 8 (i / 4) + 4 (l / 32) + i % 4 of the
// chunk in s[nb][i].
template <int NB>
__device__ __forceinline__ void pa_mask(pa_f16 (&s)[NB], int t0, int lim, int hi) {
  const int left = lim - t0 - 4 * hi;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (32 * nb + 8 * (i / 4) + i % 4 > left) s[nb][i] = -INFINITY;
}
// row of the pool of the key at position pos of table row `table`, or PA_NOSLOT
__device__ __forceinline__ uint32_t pa_slot(const PrefixAttnArgs& a, int32_t page, uint32_t pos) {
  return page >= 0 && page < a.num_blocks ? (uint32_t)page * (uint32_t)a.bs + pos % (uint32_t)a.bs
                                          : PA_NOSLOT;
}
// Those elements of keys from .. of the chunk.
template <int D, int FMT>
__device__ __forceinline__ void pa_add_odd(PaState<D>& st, const PrefixAttnArgs& a, const PaUnit& u,
                                           const int32_t* table, const uint8_t* vp, uint32_t row_bytes,
                                           int from, int lim, int hi) {
  constexpr uint32_t E = FMT == SDX_BF16 ? 0x7F80u : 0x7C00u;
#pragma nounroll
  for (int t = from; t < u.n; ++t) {
    const uint32_t pos = (uint32_t)u.key0 + t, s = pa_slot(a, table[pos / (uint32_t)a.bs], pos);
    if (s == PA_NOSLOT) continue;
    const uint16_t* const row = reinterpret_cast<const uint16_t*>(vp + (uint64_t)s * row_bytes);
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const ushort4 x = *reinterpret_cast<const ushort4*>(row + 32 * db + 8 * e + 4 * hi);
        const uint16_t y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (t <= lim && (y[i] & E) == E) st.o[db][4 * e + i] += pa_odd<FMT>(y[i]);
        __builtin_amdgcn_sched_barrier(0);  // few registers, the speed of this is no concern
      }
  }
}

// lim of query row i of a unit: the last key it sees, of the chunk (-1: none)
__device__ __forceinline__ int pa_lim(const PrefixAttnArgs& a, const PaUnit& u, bool masked, int i) {
  if (i >= u.m) return -1;
  const int64_t j = (u.r0 + i) / a.group;
  int64_t lim;
  if (!u.group) {
    lim = u.base + j;
  } else if (!masked) {
    return u.n - 1;
  } else {  // the token's own row
    const int64_t t = u.t0 + j, b = pa_find(a.cu_q, a.batch, t);
    lim = a.kv_len[b] - (a.cu_q[b + 1] - t);
  }
  return (int)max((int64_t)-1, min(lim - u.key0, (int64_t)u.n - 1));
}

// Results of query row `i` (lane l % 32's): O / l to out, or the part.
template <int D, int FMT>
__device__ __forceinline__ void pa_store4(const PrefixAttnArgs& a, const PaUnit& u, int64_t qrow, int d,
                                          float4 v) {
  if (u.direct) {
    uint2 w = make_uint2(pa_pack<FMT>(v.x, v.y), pa_pack<FMT>(v.z, v.w));
    *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(a.out) + qrow * D + d) = w;
  } else {
    *reinterpret_cast<float4*>(a.part_o + ((int64_t)u.part * a.tokens * a.hq + qrow) * D + d) = v;
  }
}
__device__ __forceinline__ int64_t pa_qrow(const PrefixAttnArgs& a, const PaUnit& u, int i) {
  const int r = u.r0 + i;
  return (u.t0 + r / a.group) * a.hq + u.kvh * a.group + r % a.group;
}

__device__ __forceinline__ uint32_t pa_take(const PrefixAttnArgs& a, uint32_t q) {
  return (uint32_t)__hip_atomic_fetch_add(a.head + PA_QUEUE * q, 1, __ATOMIC_RELAXED,
                                          __HIP_MEMORY_SCOPE_AGENT);
}

template <int D, int FMT>
__global__ void __launch_bounds__(PA_NT) __attribute__((amdgpu_waves_per_eu(2, 2)))
prefix_attn_kernel(PrefixAttnArgs a) {
  constexpr int NC = D / 8;            // 16-byte chunks of a row
  constexpr int RB = 2 * D;            // bytes of a row
  __shared__ __align__(256) uint8_t sMem[2 * 2 * PA_TILE * RB];  // two tiles of K and V
  __shared__ uint32_t sSlot[PA_RING * PA_TILE];
  __shared__ uint32_t sUnit;
  __shared__ int sOdd;  // V of the unit has elements that pa_add_odd adds
  // the wave's index and the unit are made scalar: what follows from them takes no vector
  // registers, of which a wave of two per SIMD has 256
  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  const int w = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int hi = lane / 32, l31 = lane & 31;
  const uint32_t row_bytes = (uint32_t)a.hkv * RB;
  // addresses of the lane's operands in LDS tiles
  const uint32_t ka = l31 * RB + ((hi ^ pa_swz_k<D>(l31)) << 4);
  const int vr = 4 * hi + ((lane & 15) >> 2), vd = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
  const uint32_t va = vr * RB + (((vd >> 3) ^ pa_swz_v<D>(vr)) << 4) + (vd & 7) * 2;
  const bool masked = a.head[3];
  // queue q: its eighth of the groups' units, then of the rows'. An XCD's workgroups have one
  // of its queue each to begin with, then empty it, then the others'; queues that the first
  // round empties are not asked (512 atomics to one line take as long as a small call)
  const uint32_t ng = a.head[1], nr = a.head[2];
  uint32_t at = blockIdx.x / 8;
  for (int queue = 0; queue < 8;) {  // uniform
    const uint32_t q = (blockIdx.x + queue) % 8;
    const uint32_t g0 = (uint32_t)((uint64_t)ng * q / 8), g1 = (uint32_t)((uint64_t)ng * (q + 1) / 8);
    const uint32_t b0 = (uint32_t)((uint64_t)nr * q / 8), b1 = (uint32_t)((uint64_t)nr * (q + 1) / 8);
    const uint32_t n = g1 - g0 + b1 - b0;
    if (at == PA_ASK) {
      if (n <= PA_GRID / 8) {
        ++queue;
        continue;
      }
      if (tid == 0) sUnit = pa_take(a, q);
      __syncthreads();
      at = __builtin_amdgcn_readfirstlane(sUnit);
      __syncthreads();
    }
    if (at >= n) {
      ++queue;
      at = PA_ASK;
      continue;
    }
    const PaUnit u = pa_unit(a, at < g1 - g0 ? g0 + at : ng + b0 + at - (g1 - g0), ng);
    at = PA_ASK;
    const int32_t* const table = a.block_table + u.table * a.max_blocks;
    const uint8_t* const kp = reinterpret_cast<const uint8_t*>(a.k_pool + u.kvh * D);
    const uint8_t* const vp = reinterpret_cast<const uint8_t*>(a.v_pool + u.kvh * D);
    // read in place of a key past the chunk, or without a page: its weight is 0, and its V
    // must not be NaN
    const uint8_t* const zero = reinterpret_cast<const uint8_t*>(a.head + PA_ZERO);
    const uint32_t pos0 = (uint32_t)u.key0;
    int bad = 0;
    PaState<D> st;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) st.o[db][i] = 0.0f;
    st.m = -INFINITY;
    st.l = 0.0f;
    const int r0 = PA_WROWS * w;  // the wave's rows
    const bool active = r0 < u.m;
    const int lim = pa_lim(a, u, masked, r0 + l31);
    // keys that every query row of the unit sees
    const int seen = u.group ? (masked ? 0 : u.n)
                             : (int)max((int64_t)0, min((int64_t)u.n, u.base + u.r0 / a.group + 1 - u.key0));
    pa_u4 qa[D / 16];
    {
      const uint16_t* src = a.q + (r0 + l31 < u.m ? pa_qrow(a, u, r0 + l31) * D : 0);
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        qa[ks] = *reinterpret_cast<const pa_u4*>(src + 16 * ks + 8 * hi);
        if (r0 + l31 >= u.m) qa[ks] = (pa_u4){0, 0, 0, 0};
      }
    }

    constexpr int H = NC / 4, TPR = PA_NT / NC;  // passes, rows per pass
    const int ntile = (u.n + PA_TILE - 1) / PA_TILE;
    const int lr = tid / NC, lc = tid % NC;
    // slots of the chunk's tiles, four tiles at a time, one by each wave: page ids are loaded
    // four tiles before they are needed here, eight before their keys
    auto page_of = [&](int tile) {
      const int t = tile * PA_TILE + lane;
      return t < u.n ? table[(pos0 + t) / (uint32_t)a.bs] : 0;
    };
    auto put_slot = [&](int tile, int32_t page) {
      const int t = tile * PA_TILE + lane;
      uint32_t s = PA_NOSLOT;
      if (t < u.n) {
        s = pa_slot(a, page, pos0 + t);
        bad |= s == PA_NOSLOT;
      }
      sSlot[(tile % PA_RING) * PA_TILE + lane] = s;
    };
    pa_u4 kk[H], vv[H];
    auto gather = [&](int tile) {
#pragma unroll
      for (int h = 0; h < H; ++h) {
        const uint32_t s = sSlot[(tile % PA_RING) * PA_TILE + lr + TPR * h];
        const uint64_t off = (uint64_t)s * row_bytes;
        kk[h] = *reinterpret_cast<const pa_u4*>((s == PA_NOSLOT ? zero : kp + off) + lc * 16);
        vv[h] = *reinterpret_cast<const pa_u4*>((s == PA_NOSLOT ? zero : vp + off) + lc * 16);
      }
    };
    static_assert(TPR % 16 == 0, "a pass's rows are swizzled alike");
    const uint32_t kw = lr * RB + ((lc ^ pa_swz_k<D>(lr)) << 4);
    const uint32_t vw = lr * RB + ((lc ^ pa_swz_v<D>(lr)) << 4);
    auto stage = [&](auto buf, int tile) {
      uint8_t* const k = sMem + buf * (2 * PA_TILE * RB);
      if ((tile + 1) * PA_TILE > seen && pa_finite_only<FMT, H>(vv)) sOdd = 1;
#pragma unroll
      for (int h = 0; h < H; ++h) {
        *reinterpret_cast<pa_u4*>(k + kw + TPR * h * RB) = kk[h];
        *reinterpret_cast<pa_u4*>(k + vw + (PA_TILE + TPR * h) * RB) = vv[h];
      }
    };
    put_slot(w, page_of(w));
    int32_t page = page_of(4 + w);
    if (tid == 0) sOdd = 0;
    __syncthreads();
    typedef std::integral_constant<int, 0> even;
    typedef std::integral_constant<int, 1> odd;
    gather(0);
    stage(even(), 0);
    gather(1);
    __syncthreads();
    auto tile = [&](int t, auto buf, auto next) {
      if (buf == 0 && t % 4 == 0) {  // uniform
        put_slot(t + 4 + w, page);
        page = page_of(t + 8 + w);
      }
      if (active) {
        const uint8_t* const k = sMem + buf * (2 * PA_TILE * RB);
        __builtin_amdgcn_s_setprio(1);
        pa_f16 s[2] = {};
        pa_u4 x[2][2];  // operands of a step, read a step ahead
        auto read = [&](int ks) {
#pragma unroll
          for (int n = 0; n < 2; ++n)
            x[ks & 1][n] = *reinterpret_cast<const pa_u4*>(k + (ka ^ (ks << 5)) + n * 32 * RB);
        };
        read(0);
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          if (ks + 1 < D / 16) read(ks + 1);
#pragma unroll
          for (int n = 0; n < 2; ++n) s[n] = pa_mfma<FMT>(x[ks & 1][n], qa[ks], s[n]);
        }
        // in this order: two steps' reads, then a step's products and the reads after next
        __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
          if (ks + 2 < D / 16) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        }
        __builtin_amdgcn_s_setprio(0);
        if ((t + 1) * PA_TILE > seen) pa_mask<2>(s, t * PA_TILE, lim, hi);  // uniform
        pa_softmax<D, FMT, 2>(st, s, a.scale_log2);
        __builtin_amdgcn_s_setprio(1);
        pa_pv<D, FMT, 2>(st, s, k + PA_TILE * RB, va);
        __builtin_amdgcn_s_setprio(0);
      }
      stage(next, t + 1);  // past the last tile: rows of zeros
      __builtin_amdgcn_sched_barrier(0);  // the registers are free before they are loaded
      gather(t + 2);
      __syncthreads();
    };
    for (int t = 0;; t += 2) {
      tile(t, even(), odd());
      if (t + 1 >= ntile) break;
      tile(t + 1, odd(), even());
      if (t + 2 >= ntile) break;
    }
    if (__builtin_amdgcn_readfirstlane(sOdd))
      pa_add_odd<D, FMT>(st, a, u, table, vp, row_bytes, seen / PA_TILE * PA_TILE, lim, hi);
    st.l = pa_sum_halves(st.l);
    const int i = r0 + l31;
    if (active && i < u.m) {
      const int64_t qrow = pa_qrow(a, u, i);
      const float f = u.direct ? (st.l > 0.0f || st.l != st.l ? 1.0f / st.l : 0.0f) : 1.0f;
#pragma unroll
      for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          pa_store4<D, FMT>(a, u, qrow, 32 * db + 8 * e + 4 * hi,
                            make_float4(st.o[db][4 * e] * f, st.o[db][4 * e + 1] * f,
                                        st.o[db][4 * e + 2] * f, st.o[db][4 * e + 3] * f));
      if (!u.direct && hi == 0)
        a.part_ml[(int64_t)u.part * a.tokens * a.hq + qrow] = make_float2(st.m, st.l);
    }
    if (bad && a.error) *a.error = 1;
  }
}

// Join of a query row's parts: out = sum_c w_c O_c, w_c = 2^(m_c - m) / sum 2^(m_c - m) l_c. A
// workgroup has HG heads of a token; 256 / (D / 4 HG) slices of D / 4 threads share a row's
// parts, each with a running maximum of its own, and are joined in LDS.
template <int D, int FMT, int HG>
__global__ void __launch_bounds__(PA_NT) prefix_attn_join_kernel(PrefixAttnArgs a) {
  constexpr int DL = D / 4, SL = PA_NT / DL / HG, UN = 4;
  __shared__ float4 sO[SL][HG][DL];
  __shared__ float2 sML[SL][HG];
  const uint32_t blocks = (uint32_t)(a.hq + HG - 1) / HG;
  const int64_t t = blockIdx.x / blocks;
  const uint32_t info = a.token_parts[t];
  if (info == 0) return;  // uniform
  const int tid = threadIdx.x, d4 = tid % DL, hh = tid / DL % HG, sl = tid / DL / HG;
  const int h = (int)(blockIdx.x % blocks) * HG + hh;
  const int np = info & 0xFFFF, n = np + (info >> 16), gap = a.parts / 2 - np;
  const int64_t stride = a.tokens * a.hq, qrow = t * a.hq + min(h, a.hq - 1);
  float m = -INFINITY, l = 0.0f;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int i0 = sl; i0 < n; i0 += SL * UN) {
    float2 ml[UN];
    float4 v[UN];
#pragma unroll
    for (int k = 0; k < UN; ++k) {  // part i lies at i, from np on at i + gap
      const int i = min(i0 + k * SL, n - 1);
      const int64_t p = (i + (i < np ? 0 : gap)) * stride + qrow;
      ml[k] = a.part_ml[p];
      v[k] = *reinterpret_cast<const float4*>(a.part_o + p * D + d4 * 4);
    }
    float mn = m;
#pragma unroll
    for (int k = 0; k < UN; ++k) mn = fmaxf(mn, ml[k].x);
    const float s = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
    l *= s;
    o = make_float4(o.x * s, o.y * s, o.z * s, o.w * s);
    m = mn;
#pragma unroll
    for (int k = 0; k < UN; ++k) {
      const bool none = i0 + k * SL >= n || ml[k].x == -INFINITY;  // no part: not a 0 times its O
      const float f = none ? 0.0f : __builtin_amdgcn_exp2f(ml[k].x - m);
      if (none) v[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      l += f * ml[k].y;  // 0 times the NaN sum of a part whose scores are all NaN is NaN, and so is out
      o.x += f * v[k].x;
      o.y += f * v[k].y;
      o.z += f * v[k].z;
      o.w += f * v[k].w;
    }
  }
  if constexpr (SL > 1) {
    sO[sl][hh][d4] = o;
    if (d4 == 0) sML[sl][hh] = make_float2(m, l);
    __syncthreads();
    if (sl > 0) return;
    float mn = m;
#pragma unroll
    for (int k = 1; k < SL; ++k) mn = fmaxf(mn, sML[k][hh].x);
    float s = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
    l *= s;
    o = make_float4(o.x * s, o.y * s, o.z * s, o.w * s);
#pragma unroll
    for (int k = 1; k < SL; ++k) {
      const float2 ml = sML[k][hh];
      const float4 v = sO[k][hh][d4];
      s = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - mn);
      l += s * ml.y;
      o.x += s * v.x;
      o.y += s * v.y;
      o.z += s * v.z;
      o.w += s * v.w;
    }
  }
  if (h >= a.hq) return;
  const float f = l > 0.0f || l != l ? 1.0f / l : 0.0f;
  *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(a.out) + qrow * D + d4 * 4) =
      make_uint2(pa_pack<FMT>(o.x * f, o.y * f), pa_pack<FMT>(o.z * f, o.w * f));
}

// Parts per query row: half for the prefix, half for the row's own keys. As many as the
// grid could fill from one row, in at most PA_ROOM bytes (but two).
constexpr int64_t PA_ROOM = (int64_t)192 << 20;
// That keeps two outputs in fp32 also where every row is written directly: 1.1 GB for 32,768 tokens
// of 32 heads of 128.
int prefix_attn_parts(int64_t tokens, int32_t hq, int32_t hkv, int32_t d) {
  const int64_t one = tokens * hq * (d + 2) * 4;
  const int64_t want = std::min<int64_t>(512, 2 * ((PA_GRID + hkv - 1) / hkv));
  return (int)std::max<int64_t>(2, std::min<int64_t>(want, PA_ROOM / std::max<int64_t>(1, one)) / 2 * 2);
}
// A segment that has tokens has a query tile of 128 rows for every 128 of its tokens' rows and one
// more; rows and groups without tokens, which may be most of them, have none.
int64_t prefix_attn_entries(int64_t tokens, int64_t batch, int64_t groups, int32_t group, int32_t parts) {
  return (2 * (tokens * group / PA_ROWS) + std::min(batch, tokens) + std::min(groups, tokens)) *
         (parts / 2);
}

template <int D, int FMT, int HG>
static void launch_join(const PrefixAttnArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((prefix_attn_join_kernel<D, FMT, HG>),
                     dim3((unsigned)(a.tokens * ((a.hq + HG - 1) / HG))), dim3(PA_NT), 0, s, a);
}

template <int D, int FMT>
static hipError_t launch_prefix_attn_t(const PrefixAttnArgs& a, hipStream_t s) {
  hipLaunchKernelGGL(prefix_attn_plan_kernel, dim3(1), dim3(PL_NT), 0, s, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((prefix_attn_kernel<D, FMT>), dim3(PA_GRID), dim3(PA_NT), 0, s, a);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  // few query rows have many parts: slices of a workgroup share them. Whole calls with 1, 2 and 4
  // heads a workgroup: 128 rows 21.7, - and 22.6 us, 6,400 rows 77.9, 74.2 and 74.6, 21,000 rows
  // 321, - and 307
  const int64_t rows = a.tokens * a.hq;
  if (rows <= 2048) launch_join<D, FMT, 1>(a, s);
  else if (rows <= 8192) launch_join<D, FMT, 2>(a, s);
  else launch_join<D, FMT, 4>(a, s);
  return hipGetLastError();
}

hipError_t launch_prefix_attn(int dtype, int d, const PrefixAttnArgs& a, hipStream_t s) {
  if (dtype == SDX_BF16)
    return d == 64 ? launch_prefix_attn_t<64, SDX_BF16>(a, s) : launch_prefix_attn_t<128, SDX_BF16>(a, s);
  return d == 64 ? launch_prefix_attn_t<64, SDX_F16>(a, s) : launch_prefix_attn_t<128, SDX_F16>(a, s);
}

}  // namespace sdx
