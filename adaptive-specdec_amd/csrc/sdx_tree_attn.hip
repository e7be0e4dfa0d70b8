// Attention of trees of drafted tokens over the paged cache, one layer: the verify attention of
// sdx_attn.hip (bench/bench_engine.py:170-174, the mask of specdec/kvcache.py:138-162) where a
// row's new tokens are the nodes of a tree. Node i of row b sees the row's cache, the
// kv_len - n keys in front of its nodes, and the nodes that its mask has a bit for:
//
//   out_i = sum_s p_s v_s / sum_s p_s,  p_s = 2^(scale log2(e) q_i k_s - m)
//
// An item is a tile of 256 query rows (nodes x the query heads of a KV head) of a row against
// all of its keys, in tiles of 64 that never hold cache and nodes both: cache tiles are bare but
// for the last one's end, a node tile takes one 64-bit word of each query row's mask. The items'
// tiles lie one behind another on a line, TA_COST more in front of each for what an item costs
// beside them, and every workgroup takes an equal stretch of it: no plan kernel, no queue, no
// counter, and the work is even whatever the rows' lengths are. Each workgroup works out the
// line from the lengths by itself (8 bytes a row, a scan). A stretch's first and last item may
// be parts, so there is room for two parts a workgroup, which leave (O, max, sum) in fp32 for a
// second kernel to join; whole items are written directly.
//
// Tiles go to LDS without a register in between, half of LDS ahead; 256 query rows a workgroup,
// since a second tile of a row's queries would read its keys from HBM once more; two waves per
// SIMD, 32 query rows each, of which one has matrix products while the other has exponentials.
//
// Measured, in graphs:
//   32 trees of up to 64 nodes, contexts of up to 8,192, 32 heads on 8 of 128, bf16: 250 us, 3.4
//     TB/s and 680 TFLOP/s (large copies and products reach 5.2 and 1,254: 165 us by the bytes,
//     135 by the products). Without its loads the kernel takes 200, the loads alone 206: they
//     share each CU's issue and LDS, and tiles are waited for at the barriers
//   24 trees of up to 33, contexts of up to 1,531, 14 heads on 2 of 64, fp16: 23.6 us (3.3 by the bytes)
//   1 tree of 26 behind 2,011 keys, 32 heads on 8 of 128: 17.4 us (1.7): two launches, loads that
//     wait for one another (lengths, pages, keys), instructions that are fetched once, the join
//   More than 256 query rows a KV head read its keys once for every 256: 32 trees behind 8,192 keys each
//     on 8 heads of 128, 64 nodes of 32 heads 348 us (219 by the bytes), 64 of 64 heads 657 (438 by the
//     products), 65 of 32 heads 519 (223 by the products)
#include <algorithm>
#include <type_traits>

#include "sdx_attn_tile.hpp"

namespace sdx {

constexpr int TA_GRID = TREE_ATTN_GRID;  // a workgroup on each of 256 CUs
constexpr int TA_NT = 512;               // two waves per SIMD
constexpr int TA_NW = TA_NT / kWave;
constexpr int TA_ROWS = TREE_ATTN_ROWS;  // query rows of an item, 32 per wave
constexpr int TA_RING = 2 * TA_NW;       // tiles of slots
static_assert(TA_ROWS == TA_NW * PA_WROWS, "every wave has rows of a full item");
// Tiles that an item costs beside its own. The cases above: 0 takes 255, 26.4 and 20.7 us, 4 takes
// 253, 23.9 and 17.1, 8 takes 257, 23.9 and 16.8.
constexpr uint32_t TA_COST = 4;
// Tiles of a stretch, at least: fewer parts of short items to join. The last case: 1 takes 17.3 us, 2
// takes 17.1, 4 takes 19.6; 9 trees of up to 70, 1,186 keys: 25.3, 21.9, 23.8.
constexpr uint32_t TA_LEAST = 2;

struct TaRow {
  int32_t t0, ctx;      // first node's token; keys in front of the nodes
  int32_t n, ct, kt;    // nodes; tiles of the cache, and with the nodes'
  int32_t qt;           // tiles of query rows
  bool ok, back;        // back: its offsets descend
  __device__ __forceinline__ uint32_t len() const { return (uint32_t)kt + TA_COST; }
};
__device__ __forceinline__ TaRow ta_row(const TreeAttnArgs& a, int64_t b) {
  TaRow r;
  const int64_t t0 = a.cu_q[b], t1 = a.cu_q[b + 1], kv = a.kv_len[b], n = t1 - t0;
  r.ok = t0 >= 0 && n >= 0 && t1 <= a.tokens && n <= min(a.words * 64, TREE_MAX_NODES) && kv >= n &&
         kv <= a.max_blocks * a.bs;  // 2^30 keys, 2^23 tokens at most
  r.back = n < 0;
  r.t0 = (int32_t)t0;
  r.n = r.ok ? (int32_t)n : 0;
  r.ctx = r.ok ? (int32_t)(kv - n) : 0;
  r.ct = (r.ctx + PA_TILE - 1) / PA_TILE;
  r.kt = r.ct + (r.n + PA_TILE - 1) / PA_TILE;
  r.qt = (r.n * a.group + TA_ROWS - 1) / TA_ROWS;
  return r;
}
__device__ __forceinline__ uint32_t ta_items(const TreeAttnArgs& a, const TaRow& r) {
  return (uint32_t)(r.qt * a.hkv);
}

// x / d for x < 2^30, with l = ceil(log2 d): mul = floor(2^(30 + l) / d) + 1 is off by at most d, and
// x d <= 2^(30 + l)
__device__ __forceinline__ uint32_t ta_div(uint32_t x, const TreeAttnDiv& d) {
  return (uint32_t)(((uint64_t)x * d.mul) >> d.shift);
}
static TreeAttnDiv ta_divide_by(int32_t d) {
  int l = 0;
  while ((int64_t)1 << l < d) ++l;
  return TreeAttnDiv{(uint32_t)(((uint64_t)1 << (30 + l)) / d + 1), 30 + l};
}

// a value that is the same in all lanes, as a scalar
__device__ __forceinline__ uint64_t ta_uniform(uint64_t x) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(x >> 32)) << 32 |
         (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)x);
}

struct TaScan {
  uint64_t line, lines;    // before this thread's, of all
  uint64_t item, items;
};
// sums over the workgroup's threads, in their order
__device__ __forceinline__ TaScan ta_scan(uint64_t line, uint64_t items, uint64_t* sLine, uint64_t* sItem) {
  const int lane = threadIdx.x & (kWave - 1), wv = threadIdx.x / kWave;
  const uint64_t li = wave_incl_scan_u64(line, lane);
  const uint64_t ii = wave_incl_scan_u64(items, lane);
  if (lane == kWave - 1) sLine[wv] = li, sItem[wv] = ii;
  __syncthreads();
  TaScan r{li - line, 0, ii - items, 0};
#pragma unroll
  for (int w = 0; w < TA_NW; ++w) {
    if (w < wv) r.line += sLine[w], r.item += sItem[w];
    r.lines += sLine[w], r.items += sItem[w];
  }
  __syncthreads();
  r.lines = ta_uniform(r.lines), r.items = ta_uniform(r.items);
  return r;
}

// S^T = K Q^T for a tile's 64 keys. ka: the lane's byte address in K's first row block.
template <int D, int FMT>
__device__ __forceinline__ void ta_qk(pa_f16 (&s)[2], const pa_u4 (&qa)[D / 16], const uint8_t* k, uint32_t ka) {
  constexpr int RB = 2 * D, N = D / 16, AHEAD = 2;
  pa_u4 x[AHEAD][2];  // operands of the steps to come
  auto read = [&](int ks) {
#pragma unroll
    for (int n = 0; n < 2; ++n)
      x[ks % AHEAD][n] = *reinterpret_cast<const pa_u4*>(k + (ka ^ (ks << 5)) + n * 32 * RB);
  };
#pragma unroll
  for (int ks = 0; ks < AHEAD; ++ks) read(ks);
#pragma unroll
  for (int ks = 0; ks < N; ++ks) {
#pragma unroll
    for (int n = 0; n < 2; ++n) s[n] = pa_mfma<FMT>(x[ks % AHEAD][n], qa[ks], s[n]);
    if (ks + AHEAD < N) read(ks + AHEAD);
  }
  // in this order: the first reads, then a step's products and the reads that follow them
  __builtin_amdgcn_sched_group_barrier(0x100, 2 * AHEAD, 0);
#pragma unroll
  for (int ks = 0; ks < N; ++ks) {
    __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
    if (ks + AHEAD < N) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
  }
}

// Scores of keys without their bit in m: key 32 nb + 8 (i / 4) + 4 hi + i % 4 in s[nb][i].
__device__ __forceinline__ void ta_mask(pa_f16 (&s)[2], uint64_t m, int hi) {
#pragma unroll
  for (int nb = 0; nb < 2; ++nb) {
    const uint32_t w = (uint32_t)(m >> (32 * nb)) >> (4 * hi);
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (!((w >> (8 * (i / 4) + i % 4)) & 1)) s[nb][i] = -INFINITY;
  }
}

// bits of the n nodes from 64 k on
__device__ __forceinline__ uint64_t ta_valid(int n, int k) {
  const int left = n - 64 * k;
  return left >= 64 ? ~0ull : (1ull << left) - 1;
}

// a stretch of an item
struct TaUnit {
  int32_t t0, ctx;
  int32_t n, ct, kvh, r0, m;  // r0, m: first query row, query rows
  int32_t lo, hi;             // tiles
  int32_t part;               // -1: whole, written directly
};
// token of query row i of the unit
__device__ __forceinline__ int64_t ta_token(const TreeAttnArgs& a, const TaUnit& u, int i) {
  return u.t0 + (int32_t)ta_div(u.r0 + i, a.by_group);
}
__device__ __forceinline__ int64_t ta_qrow(const TreeAttnArgs& a, const TaUnit& u, int i) {
  const uint32_t r = u.r0 + i, j = ta_div(r, a.by_group);
  return (int64_t)(u.t0 + j) * a.hq + u.kvh * a.group + (r - j * a.group);
}
// the word of query row i's mask for nodes 64 k ..
__device__ __forceinline__ uint64_t ta_word(const TreeAttnArgs& a, const TaUnit& u, int i, int k) {
  return i < u.m ? (uint64_t)a.mask[ta_token(a, u, i) * a.words + k] & ta_valid(u.n, k) : 0ull;
}

// V of nodes that some query rows do not see: infinities and NaN of theirs are 0 for the
// products (pa_finite_only) and are added here to the rows that see their node.
template <int D, int FMT>
__device__ __forceinline__ void ta_add_odd(PaState<D>& st, const TreeAttnArgs& a, const TaUnit& u,
                                           const int32_t* table, const uint8_t* vp, uint32_t row_bytes, int i,
                                           int hi) {
  constexpr uint32_t E = FMT == SDX_BF16 ? 0x7F80u : 0x7C00u;
#pragma nounroll
  for (int t = (max(u.lo, u.ct) - u.ct) * PA_TILE; t < min(u.n, (u.hi - u.ct) * PA_TILE); ++t) {
    const uint64_t w = ta_word(a, u, i, t / 64);
    const uint32_t pos = (uint32_t)u.ctx + t;
    const int32_t page = table[pos / (uint32_t)a.bs];
    if (page < 0 || page >= a.num_blocks) continue;
    const uint32_t s = (uint32_t)page * (uint32_t)a.bs + pos % (uint32_t)a.bs;
    const uint16_t* const row = reinterpret_cast<const uint16_t*>(vp + (uint64_t)s * row_bytes);
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const ushort4 x = *reinterpret_cast<const ushort4*>(row + 32 * db + 8 * e + 4 * hi);
        const uint16_t y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (((w >> (t % 64)) & 1) && (y[k] & E) == E) st.o[db][4 * e + k] += pa_odd<FMT>(y[k]);
        __builtin_amdgcn_sched_barrier(0);  // few registers, the speed of this is no concern
      }
  }
}

// 16 bytes of each lane from its own address to the 1 KB at LDS byte `to`, lane after lane, without
// a register in between. The compiler does not count it: ta_wait waits for it.
__device__ __forceinline__ void ta_load_lds(const uint8_t* from, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(from) : "memory", "m0");
}
__device__ __forceinline__ void ta_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

template <int D, int FMT>
__global__ void __launch_bounds__(TA_NT) __attribute__((amdgpu_waves_per_eu(2, 2)))
tree_attn_kernel(TreeAttnArgs a) {
  constexpr int NC = D / 8;            // 16-byte chunks of a row
  constexpr int RB = 2 * D;            // bytes of a row
  constexpr uint32_t KB = PA_TILE * RB, TB = 2 * KB;  // bytes of a tile's K, of its K and V
  constexpr int NB = D == 128 ? 4 : 8, PT = NB / 2;   // tiles in LDS, half of them in use
  __shared__ __align__(1024) uint8_t sMem[NB * TB];
  __shared__ uint32_t sSlot[TA_RING * PA_TILE];
  __shared__ uint64_t sLine[TA_NW], sItem[TA_NW], sAt[2];
  __shared__ int sOdd;  // V of the unit has elements that ta_add_odd adds
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

  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)sMem;

  // the line: its length, this workgroup's stretch, the row that the stretch starts in.
  // Neighbours on the line share an XCD (workgroup index % 8), whose L2 their keys go through.
  const uint32_t wg = blockIdx.x % 8 * (TA_GRID / 8) + blockIdx.x / 8;
  uint32_t total, step, pos = 0, from = 0;  // from: where row b starts
  uint32_t item0 = 0, items;
  int64_t b = 0;
  TaRow row = {};
  // for an output that is written whole: rows are refused, all of them are (offsets that descend may
  // name a token twice)
  bool refused = false, none = false;
  // Up to 64 rows, that is a row per lane, each wave does it by itself (a third of what the barriers
  // and the long code of any number of rows take, 2 us)
  bool quick = a.batch <= kWave;
  if (quick) {
    row = lane < a.batch ? ta_row(a, lane) : TaRow{0, 0, 0, 0, 0, 0, true, false};
    const uint32_t n = ta_items(a, row);
    const uint64_t tiles = (uint64_t)n * row.len();
    quick = !__any(tiles >> 25 != 0);
    if (quick) {  // uniform
      const uint32_t line = (uint32_t)tiles, li = wave_incl_scan_u32(line, lane), ii = wave_incl_scan_u32(n, lane);
      items = rdlane(ii, kWave - 1);
      const bool over = items > (uint64_t)a.max_items || (a.whole && __any(row.back));
      refused = __any(!row.ok), none = over;
      if ((refused || over) && a.error && blockIdx.x == 0) *a.error = 1;
      items = over ? 0 : items;
      total = over ? 0 : rdlane(li, kWave - 1);
      step = max(total / TA_GRID + (total % TA_GRID > 0), TA_LEAST);
      pos = wg * step;
      const uint64_t hit = __ballot(li - line <= pos && pos < li);
      if (hit && pos < total) {
        const int at = __ffsll((unsigned long long)hit) - 1;
        from = rdlane(li - line, at);
        item0 = rdlane(ii - n, at);
        b = at;
        row = TaRow{(int32_t)rdlane(row.t0, at), (int32_t)rdlane(row.ctx, at), (int32_t)rdlane(row.n, at),
                    (int32_t)rdlane(row.ct, at), (int32_t)rdlane(row.kt, at), (int32_t)rdlane(row.qt, at), true, false};
      } else {
        pos = total;
      }
    }
  }
  if (!quick) {
    const bool one = a.batch <= TA_NT;
    uint64_t line = 0, n = 0;
    int bad = 0, back = 0;
    for (int64_t i = tid; i < a.batch; i += TA_NT) {
      const TaRow r = ta_row(a, i);
      bad |= !r.ok;
      back |= r.back;
      line += (uint64_t)ta_items(a, r) * r.len();
      n += ta_items(a, r);
    }
    TaScan sc = ta_scan(line, n, sLine, sItem);
    // rows that share nodes (offsets out of order); a line of 2^32 tiles takes half a minute
    bool over = sc.items > (uint64_t)a.max_items || sc.lines >> 32;
    if (a.whole) {  // uniform
      refused = __syncthreads_or(bad);
      none = over = over || (refused && __syncthreads_or(back));
    }
    if ((bad || over) && a.error && blockIdx.x == 0) *a.error = 1;
    items = over ? 0 : (uint32_t)sc.items;
    total = over ? 0 : (uint32_t)sc.lines;
    step = max(total / TA_GRID + (total % TA_GRID > 0), TA_LEAST);
    pos = (uint32_t)min((uint64_t)wg * step, (uint64_t)total);
    uint64_t at = 0, it = 0;
    for (int64_t b0 = 0; at <= pos && pos < total; b0 += TA_NT) {  // uniform; ends where the line holds pos
      if (!one) {
        const TaRow r = b0 + tid < a.batch ? ta_row(a, b0 + tid) : TaRow{};
        n = b0 + tid < a.batch ? ta_items(a, r) : 0;
        line = n ? n * (uint64_t)r.len() : 0;
        sc = ta_scan(line, n, sLine, sItem);
      }
      if (at + sc.line <= pos && pos < at + sc.line + line) {
        sAt[0] = at + sc.line;
        sAt[1] = (uint64_t)(b0 + tid) << 32 | (it + sc.item);
      }
      at += sc.lines, it += sc.items;
    }
    __syncthreads();
    if (pos < total) {
      from = (uint32_t)ta_uniform(sAt[0]);
      const uint64_t x = ta_uniform(sAt[1]);
      item0 = (uint32_t)x;
      b = (int64_t)(x >> 32);
      row = ta_row(a, b);
    }
  }
  for (int64_t i = (int64_t)items + blockIdx.x * TA_NT + tid; i < a.max_items; i += TA_GRID * TA_NT)
    a.items[i].parts = 0;  // records of no item
  if (a.whole && blockIdx.x == 0 && tid == 0) *a.left = none ? 2 : refused;
  if (pos >= total) return;  // uniform
  const uint32_t end = min((uint64_t)total, (uint64_t)pos + step);

  uint32_t item = (pos - from) / row.len();
  while (pos < end) {  // uniform: the items of the stretch
    const uint32_t len = row.len(), p = from + item * len, e = min(end, p + len);
    const uint32_t mine = wg * step;
    const bool before = p + TA_COST < mine, behind = p + len - 1 >= mine + step;  // others have tiles of it
    TaUnit u;
    u.t0 = row.t0, u.ctx = row.ctx;
    u.n = row.n, u.ct = row.ct;
    u.kvh = (int32_t)(row.qt == 1 ? item : item / (uint32_t)row.qt);
    u.r0 = (int32_t)(item - u.kvh * row.qt) * TA_ROWS;
    u.m = min(TA_ROWS, row.n * a.group - u.r0);
    u.lo = (int32_t)(max(pos - p, TA_COST) - TA_COST);
    u.hi = (int32_t)(max(e - p, TA_COST) - TA_COST);
    u.part = before || behind ? (int32_t)(2 * wg + !before) : -1;
    if (!before && u.lo < u.hi && tid == 0)
      a.items[item0 + item] = TreeAttnItem{u.t0, u.kvh, u.r0, u.m, (int32_t)wg,
                                           behind ? (int32_t)((p + len - 1) / step - wg + 1) : 1, 0, 0};
    pos = e;
    const uint32_t row_end = from + ta_items(a, row) * len;
    if (u.lo < u.hi) {
      const int32_t* const table = a.block_table + b * a.max_blocks;
      const uint8_t* const kp = reinterpret_cast<const uint8_t*>(a.k_pool + u.kvh * D);
      const uint8_t* const vp = reinterpret_cast<const uint8_t*>(a.v_pool + u.kvh * D);
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
      const int ntile = u.hi - u.lo;
      // slots of the unit's tiles, eight tiles at a time, one by each wave: page ids are loaded
      // eight tiles before they are needed here
      auto key = [&](int tile) -> int32_t {  // position of the lane's key of a tile, -1: none
        const int t = u.lo + tile;
        if (t >= u.hi) return -1;
        const int x = (t < u.ct ? t : t - u.ct) * PA_TILE + lane;
        if (t < u.ct) return x < u.ctx ? x : -1;
        return x < u.n ? u.ctx + x : -1;
      };
      auto page_of = [&](int tile) {
        const int32_t x = key(tile);
        return x >= 0 ? table[ta_div(x, a.by_bs)] : 0;
      };
      auto put_slot = [&](int tile, int32_t page) {
        const int32_t x = key(tile);
        uint32_t s = PA_NOSLOT;
        if (x >= 0) {
          if (page >= 0 && page < a.num_blocks) s = (uint32_t)page * (uint32_t)a.bs + (x - ta_div(x, a.by_bs) * (uint32_t)a.bs);
          bad |= s == PA_NOSLOT;
        }
        sSlot[(tile % TA_RING) * PA_TILE + lane] = s;
      };
      // Tile t lies in LDS part t % NB. A wave's load fills 1 KB of it, RW rows; 16-byte chunk c of row
      // r lies in chunk c ^ swizzle(r), so the lanes ask for their chunks in that order. A key that is
      // none takes row 0 of the pool: its K is never seen, its V is 0 by `clean`.
      constexpr int RW = 1024 / RB, PW = PA_TILE / RW / TA_NW;  // loads of a wave for K, and for V
      const int lr = lane / NC, lc = lane % NC;
      auto slot = [&](int tile, int h) { return sSlot[(tile % TA_RING) * PA_TILE + (w * PW + h) * RW + lr]; };
      auto load = [&](int tile, int h, uint32_t sl) {
        const uint32_t at = lds0 + (uint32_t)(tile % NB) * TB + (w * PW + h) * 1024;
        const int r = (w * PW + h) * RW + lr;
        const uint64_t off = (uint64_t)(sl == PA_NOSLOT ? 0u : sl) * row_bytes;
        ta_load_lds(kp + off + ((lc ^ pa_swz_k<D>(r)) << 4), at);
        ta_load_lds(vp + off + ((lc ^ pa_swz_v<D>(r)) << 4), at + KB);
      };
      // V of the cache's last tile and of the nodes': rows of no key are 0, and so are elements that
      // ta_add_odd adds
      auto clean = [&](int tile) {
        const int g = u.lo + tile, last = g < u.ct ? u.ctx - g * PA_TILE : u.n - (g - u.ct) * PA_TILE;
        uint8_t* const v = sMem + (tile % NB) * TB + KB;
#pragma unroll
        for (int h = 0; h < PA_TILE * NC / TA_NT; ++h) {
          const int c = tid + h * TA_NT;
          pa_u4 x[1] = {*reinterpret_cast<const pa_u4*>(v + c * 16)};
          if (c / NC >= last) x[0] = (pa_u4){0, 0, 0, 0};
          if (g >= u.ct && pa_finite_only<FMT, 1>(x)) sOdd = 1;
          *reinterpret_cast<pa_u4*>(v + c * 16) = x[0];
        }
      };
      __syncthreads();  // the unit before is done with LDS
      // pages, then queries and masks: the keys wait for the pages alone
      const int32_t page0 = page_of(w);
      int32_t page = page_of(TA_NW + w);
      const int row_i = min(r0 + l31, u.m - 1);  // rows past the item's are computed like its last, and not stored
      pa_u4 qa[D / 16];
      {
        const uint16_t* const src = a.q + ta_qrow(a, u, row_i) * D + 8 * hi;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) qa[ks] = *reinterpret_cast<const pa_u4*>(src + 16 * ks);
      }
      const int64_t* const words = a.mask + ta_token(a, u, row_i) * a.words;
      uint64_t word = u.hi > u.ct ? words[max(u.lo, u.ct) - u.ct] : 0;
      put_slot(w, page0);
      if (tid == 0) sOdd = 0;
      __syncthreads();
      // PT tiles between two barriers, half of LDS. The loads of the other half lie between the
      // products and the exponentials of these: all at once they hold every wave up for a fifth of
      // the time, since a CU takes in 64 bytes a clock
      for (int t = 0; t < min(PT, ntile); ++t)
#pragma unroll
        for (int h = 0; h < PW; ++h) load(t, h, slot(t, h));
#pragma nounroll
      for (int t0 = 0; t0 < ntile; t0 += PT) {  // uniform
        ta_wait();        // this wave's part of the tiles is there
        __syncthreads();  // the tiles are whole, and nobody reads those before any more
        if (t0 % TA_NW == 0) {
          put_slot(t0 + TA_NW + w, page);
          page = page_of(t0 + 2 * TA_NW + w);
        }
        const int t1 = min(t0 + PT, ntile);
        if ((u.lo + t1) * PA_TILE > u.ctx) {
          for (int t = t0; t < t1; ++t)
            if ((u.lo + t + 1) * PA_TILE > u.ctx) clean(t);
          __syncthreads();
        }
#pragma nounroll
        for (int t = t0; t < t1; ++t) {
          const uint32_t at = (uint32_t)(t % NB) * TB;
          const bool more = t + PT < ntile;
          uint32_t sl[PW];
#pragma unroll
          for (int h = 0; h < PW; ++h) sl[h] = slot(t + PT, h);
          if (!active) {
#pragma unroll
            for (int h = 0; h < PW; ++h)
              if (more) load(t + PT, h, sl[h]);
            continue;
          }
          __builtin_amdgcn_s_setprio(1);
          pa_f16 s[2] = {};
          ta_qk<D, FMT>(s, qa, sMem, ka + at);
          __builtin_amdgcn_s_setprio(0);
          if (more) load(t + PT, 0, sl[0]);
          const int g = u.lo + t;
          if ((g + 1) * PA_TILE > u.ctx) {
            if (g < u.ct) {
              ta_mask(s, (1ull << (u.ctx - g * PA_TILE)) - 1, hi);
            } else {
              ta_mask(s, word & ta_valid(u.n, g - u.ct), hi);
              if (g + 1 < u.hi) word = words[g + 1 - u.ct];
            }
          }
          pa_softmax<D, FMT, 2>(st, s, a.scale_log2);
          if constexpr (PW > 1)
            if (more) load(t + PT, 1, sl[1]);
          __builtin_amdgcn_s_setprio(1);
          pa_pv<D, FMT, 2>(st, s, sMem, va + at + KB);
          __builtin_amdgcn_s_setprio(0);
        }
      }
      if (__builtin_amdgcn_readfirstlane(sOdd))
        ta_add_odd<D, FMT>(st, a, u, table, vp, row_bytes, r0 + l31, hi);
      st.l = pa_sum_halves(st.l);
      const int i = r0 + l31;
      if (active && i < u.m) {
        if (u.part < 0) {
          const float f = st.l > 0.0f || st.l != st.l ? 1.0f / st.l : 0.0f;
          uint16_t* const to = a.out + ta_qrow(a, u, i) * D + 4 * hi;
#pragma unroll
          for (int db = 0; db < D / 32; ++db)
#pragma unroll
            for (int e4 = 0; e4 < 4; ++e4)
              store_nt(to + 32 * db + 8 * e4,
                       make_uint2(pa_pack<FMT>(st.o[db][4 * e4] * f, st.o[db][4 * e4 + 1] * f),
                                  pa_pack<FMT>(st.o[db][4 * e4 + 2] * f, st.o[db][4 * e4 + 3] * f)));
        } else {
          float* const to = a.part_o + ((int64_t)u.part * TA_ROWS + i) * D + 4 * hi;
#pragma unroll
          for (int db = 0; db < D / 32; ++db)
#pragma unroll
            for (int e4 = 0; e4 < 4; ++e4)
              store_nt(to + 32 * db + 8 * e4, make_float4(st.o[db][4 * e4], st.o[db][4 * e4 + 1],
                                                          st.o[db][4 * e4 + 2], st.o[db][4 * e4 + 3]));
          if (hi == 0) a.part_ml[(int64_t)u.part * TA_ROWS + i] = make_float2(st.m, st.l);
        }
      }
      if (bad && a.error) *a.error = 1;
    }
    ++item;
    if (pos == row_end) {  // the next row that has nodes
      item = 0;
      from = pos;
      item0 += ta_items(a, row);
      while (++b < a.batch) {
        row = ta_row(a, b);
        if (row.n > 0) break;
      }
    }
  }
}

// Tokens t0 .. t1 - 1 of out become 0, by `parts` workgroups, of which this is one.
template <int D>
__device__ __forceinline__ void ta_zero(const TreeAttnArgs& a, int64_t t0, int64_t t1, uint32_t part, uint32_t parts) {
  const int64_t units = (int64_t)a.hq * (D / 8);  // of 16 bytes
  t0 = max(t0, (int64_t)0), t1 = min(t1, a.tokens);
  if (t0 >= t1) return;  // uniform
  for (int64_t u = t0 * units + part * PA_NT + threadIdx.x; u < t1 * units; u += parts * PA_NT)
    store_nt(a.out + u * 8, make_uint4(0, 0, 0, 0));
}
// What nothing is computed for: tokens in front of the rows and behind them, those of refused rows.
template <int D>
__device__ __forceinline__ void ta_rest(const TreeAttnArgs& a, uint32_t part, uint32_t parts) {
  const int32_t left = *a.left;
  ta_zero<D>(a, 0, left > 1 ? a.tokens : a.cu_q[0], part, parts);
  ta_zero<D>(a, a.cu_q[a.batch], a.tokens, part, parts);
  for (int64_t i = part; left == 1 && i < a.batch; i += parts)
    if (!ta_row(a, i).ok) ta_zero<D>(a, a.cu_q[i], a.cu_q[i + 1], 0, 1);
}

// Join of the items that are split: out = sum_c w_c O_c, w_c = 2^(m_c - m) / sum 2^(m_c - m) l_c.
// A workgroup has RB query rows of an item at a time; 256 / (D / 4 RB) slices of D / 4 threads
// share a row's parts, each with a running maximum of its own, and are joined in LDS. TA_REST
// workgroups behind those of the items write the rest of an output that is written whole: there they
// hold nobody up (one tree of 26: without them 17.1 us, with them 17.4, in the kernel before 17.9).
constexpr int TA_REST = 256;
template <int D, int FMT, int RB>
__global__ void __launch_bounds__(PA_NT) tree_attn_join_kernel(TreeAttnArgs a) {
  constexpr int DL = D / 4, SL = PA_NT / DL / RB, UN = SL > 1 ? 4 : 2;
  __shared__ float4 sO[SL][RB][DL];
  __shared__ float2 sML[SL][RB];
  if (blockIdx.x >= a.max_items) {  // uniform
    ta_rest<D>(a, (blockIdx.x - (uint32_t)a.max_items) * gridDim.y + blockIdx.y,
               (gridDim.x - (uint32_t)a.max_items) * gridDim.y);
    return;
  }
  const TreeAttnItem x = a.items[blockIdx.x];
  if (x.parts < 2) return;  // uniform: written directly, or no item
  const int tid = threadIdx.x, d4 = tid % DL, rr = tid / DL % RB, sl = tid / DL / RB;
  for (int i0 = blockIdx.y * RB; i0 < x.m; i0 += gridDim.y * RB) {  // uniform
    const int i = min(i0 + rr, x.m - 1);
    float m = -INFINITY, l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int c0 = sl; c0 < x.parts; c0 += SL * UN) {
      float2 ml[UN];
      float4 v[UN];
#pragma unroll
      for (int k = 0; k < UN; ++k) {
        const int c = min(c0 + k * SL, x.parts - 1);
        const int64_t p = (int64_t)(2 * (x.first + c) + (c == 0)) * TA_ROWS + i;
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
        const bool none = c0 + k * SL >= x.parts || ml[k].x == -INFINITY;  // not a 0 times its O
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
      __syncthreads();
      sO[sl][rr][d4] = o;
      if (d4 == 0) sML[sl][rr] = make_float2(m, l);
      __syncthreads();
      if (sl == 0) {
        float mn = m;
#pragma unroll
        for (int k = 1; k < SL; ++k) mn = fmaxf(mn, sML[k][rr].x);
        float s = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
        l *= s;
        o = make_float4(o.x * s, o.y * s, o.z * s, o.w * s);
#pragma unroll
        for (int k = 1; k < SL; ++k) {
          const float2 ml = sML[k][rr];
          const float4 v = sO[k][rr][d4];
          s = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - mn);
          l += s * ml.y;
          o.x += s * v.x;
          o.y += s * v.y;
          o.z += s * v.z;
          o.w += s * v.w;
        }
      }
    }
    if (sl == 0 && i0 + rr < x.m) {
      const float f = l > 0.0f || l != l ? 1.0f / l : 0.0f;
      const uint32_t r = x.r0 + i, j = r / (uint32_t)a.group;
      const int64_t qrow = (int64_t)(x.t0 + j) * a.hq + x.kvh * a.group + (r - j * a.group);
      store_nt(a.out + qrow * D + d4 * 4,
               make_uint2(pa_pack<FMT>(o.x * f, o.y * f), pa_pack<FMT>(o.z * f, o.w * f)));
    }
  }
}

// items of a call: tiles of 256 query rows, of every row that has nodes
int64_t tree_attn_items(int64_t tokens, int64_t batch, int32_t hkv, int32_t group) {
  return hkv * (tokens * group / TA_ROWS + std::min(batch, tokens));
}

template <int D, int FMT, int RB>
static void launch_join(const TreeAttnArgs& a, int64_t items, hipStream_t s) {
  const unsigned blocks = RB >= 8 ? TA_ROWS / RB / 2 : TA_ROWS / RB;
  const unsigned columns = (unsigned)items + (a.whole ? TA_REST / blocks : 0);
  hipLaunchKernelGGL((tree_attn_join_kernel<D, FMT, RB>), dim3(columns, blocks), dim3(PA_NT), 0, s, a);
}

template <int D, int FMT>
static hipError_t launch_tree_attn_t(const TreeAttnArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((tree_attn_kernel<D, FMT>), dim3(TA_GRID), dim3(TA_NT), 0, s, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int64_t items = a.max_items;
  // Few items have many parts: slices of a workgroup share them. The cases of the file's head, whose
  // bounds are 464, 84 and 8 items: one thread for all parts of its columns 253, 23.7 and 20.6 us, rows
  // in twos 267, 26.0 and 16.8, one by one 285, 31.0 and 17.2
  if (items <= 16) launch_join<D, FMT, 1>(a, items, s);
  else if (items <= 64) launch_join<D, FMT, 2>(a, items, s);
  else launch_join<D, FMT, PA_NT / (D / 4)>(a, items, s);
  return hipGetLastError();
}

hipError_t launch_tree_attn(int dtype, int d, const TreeAttnArgs& b, hipStream_t s) {
  TreeAttnArgs a = b;
  a.by_bs = ta_divide_by(a.bs);
  a.by_group = ta_divide_by(a.group);
  if (dtype == SDX_BF16)
    return d == 64 ? launch_tree_attn_t<64, SDX_BF16>(a, s) : launch_tree_attn_t<128, SDX_BF16>(a, s);
  return d == 64 ? launch_tree_attn_t<64, SDX_F16>(a, s) : launch_tree_attn_t<128, SDX_F16>(a, s);
}

}  // namespace sdx
