// Log probabilities of given tokens, the entropy of each row's distribution and its
// likeliest tokens, without the probabilities: what a caller of to_probs + gather_prob
// (specdec/sampling.py:34-67,93-95) needs for scores, in one read of the logits.
//
// With m = max x, d = (x - m) / T, z = sum e^d and w = sum d e^d:
//   log p(i) = d_i - ln z          entropy = ln z - w / z
// One pass: every thread keeps (m, z, w) of what it has read, in base 2 and shifted to its
// own running maximum (w of a sum shifted by s: 2^s (w + s z)), and joins with the others
// at the end. Sums are fp32; no decision depends on them. The shift is taken in x, before the
// product with log2(e) / T: one operation an element more than x c - m c fused, but the
// largest logit's term is exactly 1 and rows masked by their type's lowest value do not
// overflow.
//
// Likeliest tokens, by (value, lowest id): a thread also keeps its largest value and the
// first 16-byte vector that holds it, unique to the thread. Take the n-th best of any n or
// more of these heads as an edge: n elements reach it, so no element below it is listed, and
// a thread whose head is below it has none that is. The edge comes from 64 heads, the best
// of four threads each (by a wave, the largest n times); the few threads that reach it read their
// vectors again, and what reaches it there, n elements and a few, is sorted. Per element the
// list costs the maximum that the sums need anyway.
//
// Bound by the read of the logits and of the list's second look: 576 x 151,936 bf16 without a list
// 41 us and 175 MB fetched, 4.3 TB/s; with 20 alternatives 52 us (fp16 53, 288 rows of fp32 52) and
// 263 MB, 5.1 TB/s, since 16-byte vectors of a few threads lie in half of the row's lines; 1 to 5
// alternatives 47. A row is split over workgroups where rows are few, and a second kernel joins
// its parts: 5 x 50,257 fp32 6.5 us and 4.6, the launches' latency.
#include <algorithm>

#include "sdx_launch.hpp"

namespace sdx {

constexpr int LP_NT = 256;
constexpr int LP_CAP = 1024;  // collected elements; more are taken one by one
constexpr float LP_LOWEST = -3.402823466e+38f;
constexpr float LP_FAR = -200.0f;  // 2^LP_FAR is 0 in fp32

struct LpPart {  // of a row's part: sums in base 2, relative to m
  float m, z, w, pad;
};

template <int FMT>
constexpr int lp_vec() { return FMT == SDX_F32 ? 4 : 8; }  // elements of a 16-byte vector
// Vectors per thread in flight, 16 elements. 576 x 151,936 bf16 with 20 alternatives: 2 54 us,
// 4 58; 288 x 151,936 fp32: 2 59, 4 54.
template <int FMT>
constexpr int lp_un() { return 16 / lp_vec<FMT>(); }

// Ascending order as unsigned words; -0 and 0 are equal. A NaN is below everything.
__device__ __forceinline__ uint32_t lp_ord(float x) {
  if (x != x) return 1u;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float lp_unord(uint32_t o) {
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);
}

template <int FMT>
__device__ __forceinline__ float lp_elem(const void* row, int64_t i) {
  if constexpr (FMT == SDX_F32) return reinterpret_cast<const float*>(row)[i];
  else return decode16<FMT>(reinterpret_cast<const uint16_t*>(row)[i]);
}

// A row as whole 16-byte vectors, from `head` elements after its start, and its edges: those
// elements and the ones behind the last vector. A part is vectors v0 .. v1 - 1; part 0 has the
// edges too.
struct LpSpan {
  const uint8_t* row;
  const uint8_t* vec;  // vector 0, on a 16-byte boundary
  uint32_t V, head, edges, v0, v1;
};
template <int FMT>
__device__ __forceinline__ LpSpan lp_span(const LogprobArgs& a, int64_t r, int part) {
  constexpr int VEC = lp_vec<FMT>(), ES = 16 / VEC;
  LpSpan s;
  s.row = reinterpret_cast<const uint8_t*>(a.logits) + r * a.ld * ES;
  s.V = (uint32_t)a.V;
  s.head = min(s.V, (uint32_t)(-(uintptr_t)s.row & 15u) / ES);
  s.vec = s.row + s.head * ES;
  const uint32_t n = (s.V - s.head) / VEC;
  s.v0 = (uint32_t)((uint64_t)n * part / a.parts);
  s.v1 = (uint32_t)((uint64_t)n * (part + 1) / a.parts);
  s.edges = part == 0 ? s.V - n * VEC : 0;
  return s;
}
// Vector v, or another of the part behind its end: loads that no branch holds up. The part
// has a vector.
__device__ __forceinline__ uint4 lp_load(const LpSpan& s, uint32_t v) {
  return *reinterpret_cast<const uint4*>(s.vec + (uint64_t)min(v, s.v1 - 1) * 16);
}
template <int FMT>
__device__ __forceinline__ void lp_elems(uint4 raw, float (&x)[lp_vec<FMT>()]) {
  const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (FMT == SDX_F32) {
      x[i] = __uint_as_float(u[i]);
    } else {
      x[2 * i] = decode16<FMT>(u[i] & 0xFFFFu);
      x[2 * i + 1] = decode16<FMT>(u[i] >> 16);
    }
  }
}
// Id of edge e, and its element.
template <int FMT>
__device__ __forceinline__ uint32_t lp_edge_id(const LpSpan& s, uint32_t e) {
  return e < s.head ? e : s.V - s.edges + e;
}

// (m, z, w) moved to the larger maximum mn.
__device__ __forceinline__ void lp_shift(float& z, float& w, float m, float mn, float c) {
  const float s = fmaxf((m - mn) * c, LP_FAR);
  const float f = __builtin_amdgcn_exp2f(s);
  w = f * fmaf(s, z, w);
  z *= f;
}
__device__ __forceinline__ void lp_join(LpPart& a, const LpPart& b, float c) {
  const float mn = fmaxf(a.m, b.m);
  float zb = b.z, wb = b.w;
  lp_shift(a.z, a.w, a.m, mn, c);
  lp_shift(zb, wb, b.m, mn, c);
  a.m = mn;
  a.z += zb;
  a.w += wb;
}
__device__ __forceinline__ void lp_wave_join(LpPart& p, float c) {
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    LpPart q;
    q.m = __shfl_xor(p.m, o, kWave);
    q.z = __shfl_xor(p.z, o, kWave);
    q.w = __shfl_xor(p.w, o, kWave);
    lp_join(p, q, c);
  }
}

// Descending sort of the n keys in LDS, padded with zeros up to `size` (a power of two of
// at least n); all threads.
__device__ __forceinline__ void lp_sort(uint64_t* k, int n, int size) {
  for (int i = n + threadIdx.x; i < size; i += LP_NT) k[i] = 0;
  __syncthreads();
  for (int len = 2; len <= size; len <<= 1)
    for (int st = len >> 1; st > 0; st >>= 1) {
      for (int i = threadIdx.x; i < size / 2; i += LP_NT) {
        const int a = 2 * i - (i & (st - 1)), b = a + st;
        const uint64_t x = k[a], y = k[b];
        if (((a & len) == 0) == (x < y)) k[a] = y, k[b] = x;
      }
      __syncthreads();
    }
}
__device__ __forceinline__ int lp_pow2(int n) {
  return n <= 2 ? 2 : 1 << (32 - __clz(n - 1));
}

struct LpRow {  // a row's sums, and ln z
  float m, z, w, lnz;
};
__device__ __forceinline__ LpRow lp_row(const LpPart& p) { return LpRow{p.m, p.z, p.w, logf(p.z)}; }
// log p at logit x.
__device__ __forceinline__ float lp_logp(const LogprobArgs& a, const LpRow& p, float x) {
  return !(p.z > 0.0f) ? NAN : (x - p.m) / a.T - p.lnz;  // no finite maximum, or a NaN
}
// A row's results from its sums, by `lanes` threads from `tid` on.
template <int FMT>
__device__ __forceinline__ void lp_finish(const LogprobArgs& a, int64_t r, const void* row,
                                          const LpRow& p, int tid, int lanes) {
  for (int i = tid; i < a.n_ids; i += lanes) {
    const int64_t id = a.ids[r * a.n_ids + i];
    const bool in = id >= 0 && id < a.V;
    const float v = lp_logp(a, p, in ? lp_elem<FMT>(row, id) : 0.0f);
    a.logp[r * a.n_ids + i] = in || v != v ? v : -INFINITY;
  }
  if (tid == 0) a.entropy[r] = !(p.z > 0.0f) ? NAN : p.lnz - 0.6931471805599453f * (p.w / p.z);
}
// Entry i of a row's list from its key (value order << 32 | ~id).
__device__ __forceinline__ void lp_put(const LogprobArgs& a, int64_t r, int i, const LpRow& p,
                                       uint64_t key) {
  const uint32_t o = (uint32_t)(key >> 32);  // 0 and 1 only in a row with NaN
  a.top_ids[r * a.top_n + i] = o == 0u ? -1 : (int64_t)(uint32_t)~(uint32_t)key;
  a.top_logp[r * a.top_n + i] = o <= 1u ? NAN : lp_logp(a, p, lp_unord(o));
}
// The number of the first n of a wave's keys in LDS that are greater than `key`.
__device__ __forceinline__ int lp_rank(const uint64_t* keys, int n, uint64_t key) {
  int rank = 0;
  for (int t = 0; t < n; t += 4) {  // uniform; the keys are padded with zeros
#pragma unroll
    for (int i = 0; i < 4; ++i) rank += keys[t + i] > key;
  }
  return rank;
}
// Orders the writes and reads of a wave's own LDS.
__device__ __forceinline__ void lp_wave_sync() {
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_wave_barrier();
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
}
// The n-th best of a wave's 64 heads (value order << 32 | ~vector; 0: none), or 0 where there
// are fewer. s: 64 words of LDS.
__device__ __forceinline__ uint64_t lp_wave_nth(uint64_t head, int n, uint32_t* s) {
  const int lane = threadIdx.x & (kWave - 1);
  const uint32_t o = (uint32_t)(head >> 32);
  s[lane] = o;
  lp_wave_sync();
  int above = 0;
#pragma unroll
  for (int t = 0; t < kWave; t += 4) {
    const uint4 k = *reinterpret_cast<const uint4*>(s + t);
    above += (k.x > o) + (k.y > o) + (k.z > o) + (k.w > o);
  }
  // the smallest value with fewer than n above it
  const uint32_t nth = ~wave_max_u32(above < n ? ~o : 0u);
  if (nth == 0) return 0;
  const bool tied = o == nth;
  uint32_t v = tied ? (uint32_t)head : 0u, last = wave_max_u32(v);
  int left = n - (int)rdlane((uint32_t)above, __ffsll((unsigned long long)__ballot(tied)) - 1);
  // the left-th first vector of the tied ones; all of them where they are no more
  if (__popcll(__ballot(tied)) <= left) return (uint64_t)nth << 32 | ~wave_max_u32(tied ? ~v : 0u);
  for (; left > 1; --left) {  // uniform
    if (v == last) v = 0;  // vectors differ
    last = wave_max_u32(v);
  }
  return (uint64_t)nth << 32 | last;
}

// Part blockIdx.x % parts of row blockIdx.x / parts: elements [lo, hi). One part: the results; several: the
// part's record and its top_n keys, for logprob_join_kernel.
template <int FMT, bool TOP>
__global__ void __launch_bounds__(LP_NT) logprob_kernel(LogprobArgs a) {
  constexpr int VEC = lp_vec<FMT>(), LP_UN = lp_un<FMT>();
  __shared__ LpPart sPart[LP_NT / kWave];
  __shared__ __align__(16) uint64_t sKeys[TOP ? LP_CAP : 1];
  __shared__ uint64_t sHead[TOP ? LP_NT : 1], sEdge;
  __shared__ int sSel[TOP ? LP_NT : 1], sCount, sNsel;
  const int tid = threadIdx.x;
  const int64_t r = blockIdx.x / (uint32_t)a.parts;
  const int part = (int)(blockIdx.x % (uint32_t)a.parts);
  const LpSpan span = lp_span<FMT>(a, r, part);
  const uint32_t v0 = span.v0, v1 = span.v1;
  const float c = a.c;

  LpPart p{LP_LOWEST, 0.0f, 0.0f, 0.0f};
  // a NaN or an infinite maximum reaches z; -inf adds nothing to either sum
  auto add = [&](float x) {
    const float d = (x - p.m) * c, e = __builtin_amdgcn_exp2f(d);
    p.z += e;
    p.w = fmaf(fmaxf(d, LP_FAR), e, p.w);
  };
  uint32_t best = 0;  // order of the thread's largest value, and the vector it first came in
  uint32_t at = 0;
  for (uint32_t vb = v0; vb < v1; vb += LP_NT * LP_UN) {  // uniform
    uint4 raw[LP_UN];
#pragma unroll
    for (int u = 0; u < LP_UN; ++u) raw[u] = lp_load(span, vb + u * LP_NT + tid);
    float x[LP_UN][VEC];
#pragma unroll
    for (int u = 0; u < LP_UN; ++u) lp_elems<FMT>(raw[u], x[u]);
    if (vb + LP_NT * LP_UN > v1) {  // uniform: the last ones
#pragma unroll
      for (int u = 0; u < LP_UN; ++u)
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          if (vb + u * LP_NT + tid >= v1) x[u][i] = -INFINITY;
    }
    float top = LP_LOWEST;
#pragma unroll
    for (int u = 0; u < LP_UN; ++u) {
      float vm = x[u][0];
#pragma unroll
      for (int i = 1; i < VEC; ++i) vm = fmaxf(vm, x[u][i]);
      top = fmaxf(top, vm);
      if constexpr (TOP) {
        const uint32_t v = vb + u * LP_NT + tid, o = lp_ord(vm);
        if (o > best && v < v1) best = o, at = v;
      }
    }
    const float mn = fmaxf(p.m, top);
    lp_shift(p.z, p.w, p.m, mn, c);
    p.m = mn;
#pragma unroll
    for (int u = 0; u < LP_UN; ++u)
#pragma unroll
      for (int i = 0; i < VEC; ++i) add(x[u][i]);
  }
  const bool has_edge = (uint32_t)tid < span.edges;
  float edge_x = 0.0f;
  if (has_edge) {
    edge_x = lp_elem<FMT>(span.row, lp_edge_id<FMT>(span, tid));
    const float mn = fmaxf(p.m, edge_x);
    lp_shift(p.z, p.w, p.m, mn, c);
    p.m = mn;
    add(edge_x);
  }
  lp_wave_join(p, c);
  if ((tid & (kWave - 1)) == 0) sPart[tid / kWave] = p;
  const uint64_t head = best ? (uint64_t)best << 32 | (uint32_t)~at : 0;
  if constexpr (TOP) sHead[tid] = head;
  if (tid == 0) sCount = 0, sNsel = 0;
  __syncthreads();
  p = sPart[0];
#pragma unroll
  for (int w = 1; w < LP_NT / kWave; ++w) lp_join(p, sPart[w], c);

  const LpRow row_sums = lp_row(p);
  bool sorted = false;  // the list lies in sKeys in order
  if constexpr (TOP) {
    if (tid < kWave) {
      uint64_t h = head;
#pragma unroll
      for (int w = 1; w < LP_NT / kWave; ++w) {
        const uint64_t k = sHead[w * kWave + tid];
        h = k > h ? k : h;
      }
      // 0, fewer heads than n: everything is listed
      h = lp_wave_nth(h, a.top_n, reinterpret_cast<uint32_t*>(sKeys));
      if (tid == 0) sEdge = h;
    }
    __syncthreads();
    const uint64_t edge = sEdge;
    const uint32_t eo = (uint32_t)(edge >> 32), ev = ~(uint32_t)edge;
    if (best && head >= edge) sSel[atomicAdd(&sNsel, 1)] = tid;
    __syncthreads();
    // take(key) for the elements of those threads that reach the edge: their vectors spread
    // over the workgroup, several loads in flight; and for the row's edges that do. Of equal
    // values those behind the n-th head's vector are beaten by n heads.
    constexpr int SL = 8;  // lanes a thread's vectors are spread over
    const int nsel = sNsel;
    const uint32_t per = (v1 - v0 + LP_NT - 1) / LP_NT;
    auto visit = [&](auto take) {
      for (int i0 = tid / SL; i0 < nsel; i0 += LP_NT / SL)
        for (uint32_t j0 = tid % SL; j0 < per; j0 += SL * LP_UN) {
          uint4 raw[LP_UN];
          const uint32_t vs = v0 + j0 * LP_NT + sSel[i0];
#pragma unroll
          for (int u = 0; u < LP_UN; ++u) raw[u] = lp_load(span, vs + u * SL * LP_NT);
#pragma unroll
          for (int u = 0; u < LP_UN; ++u) {
            const uint32_t v = vs + u * SL * LP_NT;
            float y[VEC];
            lp_elems<FMT>(raw[u], y);
            const uint32_t least = edge == 0 || v <= ev ? max(eo, 1u) : eo + 1;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              const uint32_t o = lp_ord(y[e]);
              if (o >= least && v < v1)
                take((uint64_t)o << 32 | (uint32_t)~(span.head + v * VEC + e));
            }
          }
        }
      if (has_edge) {
        const uint32_t o = lp_ord(edge_x);
        if (o >= (edge == 0 || (uint32_t)tid < span.head ? max(eo, 1u) : eo + 1))
          take((uint64_t)o << 32 | (uint32_t)~lp_edge_id<FMT>(span, tid));
      }
    };
    visit([&](uint64_t k) {
      const int n = atomicAdd(&sCount, 1);
      if (n < LP_CAP) sKeys[n] = k;
    });
    __syncthreads();
    const int n = sCount;
    if (n <= kWave) {  // one wave ranks them
      if (tid < kWave) {
        const uint64_t k = tid < n ? sKeys[tid] : 0;
        lp_wave_sync();
        if (tid >= n) sKeys[tid] = 0;
        lp_wave_sync();
        const int i = lp_rank(sKeys, n, k);
        // the list is longer than a part with fewer elements: zeros follow
        if (k > 0 && i < a.top_n) {
          if (a.parts == 1) lp_put(a, r, i, row_sums, k);
          else a.part_keys[(r * a.parts + part) * a.top_n + i] = k;
        }
        if (tid >= n && tid < a.top_n) {
          if (a.parts == 1) lp_put(a, r, tid, row_sums, 0);
          else a.part_keys[(r * a.parts + part) * a.top_n + tid] = 0;
        }
      }
    } else if (n <= LP_CAP) {
      lp_sort(sKeys, n, lp_pow2(n));
      sorted = true;
    } else {  // many elements of few threads: the largest, then the largest below it, ...
      uint64_t last = ~0ull;
      for (int k = 0; k < a.top_n; ++k) {
        uint64_t b = 0;
        visit([&](uint64_t q) { b = q < last && q > b ? q : b; });
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
          const uint64_t q = __shfl_xor((unsigned long long)b, o, kWave);
          b = q > b ? q : b;
        }
        if ((tid & (kWave - 1)) == 0) sHead[tid / kWave] = b;
        __syncthreads();
        for (int w = 0; w < LP_NT / kWave; ++w) b = sHead[w] > b ? sHead[w] : b;
        if (tid == 0) sKeys[k] = b;
        last = b;
        __syncthreads();
      }
      sorted = true;
    }
    if (sorted)
      for (int i = tid; i < a.top_n; i += LP_NT) {
        if (a.parts == 1) lp_put(a, r, i, row_sums, sKeys[i]);
        else a.part_keys[(r * a.parts + part) * a.top_n + i] = sKeys[i];
      }
  }
  if (a.parts == 1) lp_finish<FMT>(a, r, span.row, row_sums, tid, LP_NT);
  else if (tid == 0) reinterpret_cast<LpPart*>(a.part)[r * a.parts + part] = p;
}

// A wave per row joins its parts: the sums across lanes, a lane a part, and the sorted lists.
// Of p lists' j-th best, p j >= n, the smallest, or, of p >= n lists, the n-th best of their
// first is reached by n keys: the few keys that reach it are ranked.
template <int FMT>
__global__ void __launch_bounds__(kWave) logprob_join_kernel(LogprobArgs a) {
  __shared__ __align__(16) uint64_t sKeys[LP_MAX_PARTS * LP_MAX_TOP], sList[kWave];
  const int lane = threadIdx.x;
  const int64_t r = blockIdx.x;
  const int n = a.parts * a.top_n;
  for (int i = lane; i < n; i += kWave) sKeys[i] = a.part_keys[r * n + i];
  LpPart p{LP_LOWEST, 0.0f, 0.0f, 0.0f};
  if (lane < a.parts) p = reinterpret_cast<const LpPart*>(a.part)[r * a.parts + lane];
  lp_wave_join(p, a.c);
  const void* const row = reinterpret_cast<const uint8_t*>(a.logits) +
                          r * a.ld * (FMT == SDX_F32 ? 4 : 2);
  const LpRow sums = lp_row(p);
  lp_finish<FMT>(a, r, row, sums, lane, kWave);
  if (a.top_n == 0) return;
  lp_wave_sync();  // the keys are in LDS
  const int depth = (a.top_n + a.parts - 1) / a.parts;
  const uint64_t mine = lane < a.parts ? sKeys[lane * a.top_n + depth - 1] : 0;
  uint64_t least;
  if (depth == 1) {  // the n-th best first key: its value, ties included
    least = lp_wave_nth(mine, a.top_n, reinterpret_cast<uint32_t*>(sList)) & ~0xFFFFFFFFull;
  } else {
    const uint32_t o = ~wave_max_u32(lane < a.parts ? ~(uint32_t)(mine >> 32) : 0u);
    least = (uint64_t)o << 32;
  }
  lp_wave_sync();
  int count = 0;
  for (int i0 = 0; i0 < n; i0 += kWave) {  // uniform
    const uint64_t k = i0 + lane < n ? sKeys[i0 + lane] : 0;
    const uint64_t in = __ballot(k > 0 && k >= least);
    const int at = count + __popcll(in & ((1ull << lane) - 1));
    if (k > 0 && k >= least && at < kWave) sList[at] = k;
    count += __popcll(in);
  }
  if (count <= kWave) {  // uniform
    lp_wave_sync();
    const uint64_t k = lane < count ? sList[lane] : 0;
    lp_wave_sync();
    if (lane >= count) sList[lane] = 0;
    lp_wave_sync();
    const int i = lp_rank(sList, count, k);
    if (k > 0 && i < a.top_n) lp_put(a, r, i, sums, k);
    if (lane >= count && lane < a.top_n) lp_put(a, r, lane, sums, 0);
    return;
  }
  // many equal values: the largest of the lists' first keys, n times
  int at = lane * a.top_n, left = lane < a.parts ? a.top_n : 0;
  uint64_t key = left > 0 ? sKeys[at] : 0, best = 0;
  for (int i = 0; i < a.top_n; ++i) {  // uniform
    const uint32_t o = wave_max_u32((uint32_t)(key >> 32));
    const uint32_t id = wave_max_u32((uint32_t)(key >> 32) == o ? (uint32_t)key : 0u);
    const uint64_t top = (uint64_t)o << 32 | id;
    if (lane == i) best = top;
    if (key == top && left > 0) {
      ++at;
      key = --left > 0 ? sKeys[at] : 0;
    }
  }
  if (lane < a.top_n) lp_put(a, r, lane, sums, best);
}

// Parts of a row: the fewest that give the shortest rounds of workgroups on the chip, a part
// counted by its elements and LP_OVER more for what follows them (2,048 or 32,768 for LP_OVER: the
// same within 2% at 1 to 1,000 rows).
constexpr int64_t LP_SLOTS = 2048, LP_LEAST = 2048, LP_OVER = 8192;
int logprob_parts(int64_t rows, int64_t V) {
  int best = 1;
  int64_t least = INT64_MAX;
  for (int p = 1; p <= LP_MAX_PARTS && (p == 1 || V / p >= LP_LEAST); ++p) {
    const int64_t t = (rows * p + LP_SLOTS - 1) / LP_SLOTS * (V / p + LP_OVER);
    if (t < least) least = t, best = p;
  }
  return best;
}

template <int FMT>
static hipError_t launch_logprob_t(const LogprobArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)(a.parts * a.rows));
  if (a.top_n > 0) hipLaunchKernelGGL((logprob_kernel<FMT, true>), grid, dim3(LP_NT), 0, s, a);
  else hipLaunchKernelGGL((logprob_kernel<FMT, false>), grid, dim3(LP_NT), 0, s, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.parts == 1) return e;
  hipLaunchKernelGGL((logprob_join_kernel<FMT>), dim3((unsigned)a.rows), dim3(kWave), 0, s, a);
  return hipGetLastError();
}

hipError_t launch_logprob(int dtype, const LogprobArgs& a, hipStream_t s) {
  if (dtype == SDX_F32) return launch_logprob_t<SDX_F32>(a, s);
  return dtype == SDX_BF16 ? launch_logprob_t<SDX_BF16>(a, s) : launch_logprob_t<SDX_F16>(a, s);
}

}  // namespace sdx
