// Log probabilities of given tokens, the entropy of each row's distribution and its
// likeliest tokens, without the probabilities: what a caller of to_probs + gather_prob
// (specdec/sampling.py:34-67,93-95) needs for scores, in one read of the logits.
//
// With m = max x, d = (x - m) / T, z = sum e^d and w = sum d e^d:
//   log p(i) = d_i - ln z          entropy = ln z - w / z
// One pass: every thread keeps (m, z, w) of what it has read, in base 2 and shifted to its
// own running maximum (w of a sum shifted by s: 2^s (w + s z)), and joins with the others
// at the end. Sums are fp32; no decision depends on them.
//
// Likeliest tokens, by (value, lowest id): a thread also keeps its largest value and the
// first 16-byte vector that holds it, unique to the thread. Every one of the n best
// elements lies in one of the n best threads by (largest value, first vector): an element
// outside them is beaten by one element of each. So the n threads' vectors are read again
// (1 / 12 of a row's part at n = 20), those elements collected that reach the n-th thread's
// (value, vector), and sorted. Per element the list costs the maximum that the sums need
// anyway.
//
// Bound by the read of the logits. A row is split over workgroups where rows are few, and a
// second kernel joins its parts.
#include <algorithm>

#include "sdx_launch.hpp"

namespace sdx {

constexpr int LP_NT = 256;
constexpr int LP_UN = 4;      // vectors per thread in flight
constexpr int LP_CAP = 1024;  // collected elements; more are taken one by one
constexpr float LP_LOWEST = -3.402823466e+38f;
constexpr float LP_FAR = -200.0f;  // 2^LP_FAR is 0 in fp32

struct LpPart {  // of a row's part: sums in base 2, relative to m
  float m, z, w, pad;
};

template <int FMT>
constexpr int lp_vec() { return FMT == SDX_F32 ? 4 : 8; }  // elements of a 16-byte vector

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

// The 16-byte vector of elements first .. first + VEC - 1, which all lie in the row.
template <int FMT>
__device__ __forceinline__ void lp_load(const void* row, int64_t first, float (&x)[lp_vec<FMT>()]) {
  if constexpr (FMT == SDX_F32) {
    const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(row) + first);
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  } else {
    const uint4 v = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(row) + first);
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = decode16<FMT>(u[i] & 0xFFFFu);
      x[2 * i + 1] = decode16<FMT>(u[i] >> 16);
    }
  }
}
// The same where it may reach past [lo, hi): those elements are not read, and are -inf.
template <int FMT>
__device__ __forceinline__ void lp_load_edge(const void* row, int64_t first, int64_t lo, int64_t hi,
                                             float (&x)[lp_vec<FMT>()]) {
  constexpr int VEC = lp_vec<FMT>();
  if (first >= lo && first + VEC <= hi) return lp_load<FMT>(row, first, x);
#pragma unroll
  for (int i = 0; i < VEC; ++i)
    x[i] = first + i >= lo && first + i < hi ? lp_elem<FMT>(row, first + i) : -INFINITY;
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

// A row's results from its sums and its sorted keys (value order << 32 | ~id).
template <int FMT>
__device__ __forceinline__ void lp_finish(const LogprobArgs& a, int64_t r, const void* row,
                                          const LpPart& p, const uint64_t* keys) {
  const float lnz = logf(p.z);
  const bool none = !(p.z > 0.0f);  // no finite maximum, or a NaN
  auto logp = [&](float x) { return none ? NAN : (x - p.m) / a.T - lnz; };
  for (int i = threadIdx.x; i < a.n_ids; i += LP_NT) {
    const int64_t id = a.ids[r * a.n_ids + i];
    a.logp[r * a.n_ids + i] =
        id >= 0 && id < a.V ? logp(lp_elem<FMT>(row, id)) : (none ? NAN : -INFINITY);
  }
  if (threadIdx.x == 0) a.entropy[r] = none ? NAN : lnz - 0.6931471805599453f * (p.w / p.z);
  for (int i = threadIdx.x; i < a.top_n; i += LP_NT) {
    const uint32_t o = (uint32_t)(keys[i] >> 32);  // 0 and 1 only in a row with NaN
    a.top_ids[r * a.top_n + i] = o == 0u ? -1 : (int64_t)(uint32_t)~(uint32_t)keys[i];
    a.top_logp[r * a.top_n + i] = o <= 1u ? NAN : logp(lp_unord(o));
  }
}

// Part blockIdx.x % parts of row blockIdx.x / parts: elements [lo, hi). One part: the results; several: the
// part's record and its top_n keys, for logprob_join_kernel.
template <int FMT, bool TOP>
__global__ void __launch_bounds__(LP_NT) logprob_kernel(LogprobArgs a) {
  constexpr int VEC = lp_vec<FMT>();
  __shared__ LpPart sPart[LP_NT / kWave];
  __shared__ uint64_t sKeys[TOP ? LP_CAP : 1];
  __shared__ uint64_t sHead[TOP ? LP_NT : 1];
  __shared__ int sSel[TOP ? LP_NT : 1], sCount;
  const int tid = threadIdx.x;
  const int64_t r = blockIdx.x / (uint32_t)a.parts;
  const int part = (int)(blockIdx.x % (uint32_t)a.parts);
  const void* const row = reinterpret_cast<const uint8_t*>(a.logits) +
                          r * a.ld * (FMT == SDX_F32 ? 4 : 2);
  // vectors of the row from the 16-byte boundary at or before it; this part's [v0, v1)
  const int off = (int)(((uintptr_t)row & 15u) / (FMT == SDX_F32 ? 4 : 2));
  const int64_t nvec = (a.V + off + VEC - 1) / VEC;
  const int64_t v0 = nvec * part / a.parts, v1 = nvec * (part + 1) / a.parts;
  const int64_t lo = max((int64_t)0, v0 * VEC - off), hi = min(a.V, v1 * VEC - off);
  const float c = a.c;

  LpPart p{LP_LOWEST, 0.0f, 0.0f, 0.0f};
  uint32_t best = 0;  // order of the thread's largest value, and the vector it first came in
  uint32_t at = 0;
  for (int64_t vb = v0; vb < v1; vb += LP_NT * LP_UN) {  // uniform
    float x[LP_UN][VEC];
    if (vb > v0 && vb + LP_NT * LP_UN < v1) {  // whole vectors throughout
#pragma unroll
      for (int u = 0; u < LP_UN; ++u)
        lp_load<FMT>(row, (vb + u * LP_NT + tid) * VEC - off, x[u]);
    } else {
#pragma unroll
      for (int u = 0; u < LP_UN; ++u)
        lp_load_edge<FMT>(row, (vb + u * LP_NT + tid) * VEC - off, lo, hi, x[u]);
    }
    float mn = p.m;
#pragma unroll
    for (int u = 0; u < LP_UN; ++u) {
      float vm = x[u][0];
#pragma unroll
      for (int i = 1; i < VEC; ++i) vm = fmaxf(vm, x[u][i]);
      mn = fmaxf(mn, vm);
      if constexpr (TOP) {
        const int64_t v = vb + u * LP_NT + tid;
        const uint32_t o = lp_ord(vm);
        if (o > best && v < v1) best = o, at = (uint32_t)v;
      }
    }
    lp_shift(p.z, p.w, p.m, mn, c);
    p.m = mn;
#pragma unroll
    for (int u = 0; u < LP_UN; ++u)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        // a NaN or an infinite maximum reaches z; -inf adds nothing to either sum
        const float d = (x[u][i] - mn) * c, e = __builtin_amdgcn_exp2f(d);
        p.z += e;
        p.w = fmaf(fmaxf(d, LP_FAR), e, p.w);
      }
  }
  lp_wave_join(p, c);
  if ((tid & (kWave - 1)) == 0) sPart[tid / kWave] = p;
  if constexpr (TOP) sHead[tid] = ((uint64_t)best << 32) | (uint32_t)~at;
  if (tid == 0) sCount = 0;
  __syncthreads();
  p = sPart[0];
#pragma unroll
  for (int w = 1; w < LP_NT / kWave; ++w) lp_join(p, sPart[w], c);

  if constexpr (TOP) {
    // the top_n best threads by (value, first vector); threads without a vector have 0
    const uint64_t mine = sHead[tid];
    int rank = 0;
    for (int t = 0; t < LP_NT; ++t) rank += sHead[t] > mine || (sHead[t] == mine && t < tid);
    if (rank < a.top_n) sSel[rank] = tid;
    __syncthreads();
    const int nsel = min(a.top_n, LP_NT);
    const uint64_t edge = sHead[sSel[nsel - 1]];
    const uint32_t eo = (uint32_t)(edge >> 32), ev = ~(uint32_t)edge;
    const int per = (int)((v1 - v0 + LP_NT - 1) / LP_NT);  // vectors of a thread
    // `take` gets every element (key) of the selected threads that can be in the list
    auto visit = [&](auto take) {
      for (int i = tid; i < nsel * per; i += LP_NT) {
        const int64_t v = v0 + (int64_t)(i / nsel) * LP_NT + sSel[i % nsel];
        if (v >= v1) continue;
        float y[VEC];
        lp_load_edge<FMT>(row, v * VEC - off, lo, hi, y);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const int64_t id = v * VEC - off + e;
          const uint32_t o = lp_ord(y[e]);
          if (id >= lo && id < hi && (o > eo || (o == eo && (eo == 0 || (uint32_t)v <= ev))))
            take(((uint64_t)o << 32) | (uint32_t)~(uint32_t)id);
        }
      }
    };
    visit([&](uint64_t k) {
      const int n = atomicAdd(&sCount, 1);
      if (n < LP_CAP) sKeys[n] = k;
    });
    __syncthreads();
    const int n = sCount;
    if (n <= LP_CAP) {
      lp_sort(sKeys, n, lp_pow2(max(n, a.top_n)));
    } else {  // many elements of few threads: the largest, then the largest below it, ...
      uint64_t last = ~0ull;
      __syncthreads();
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
    }
  }
  if (a.parts == 1) {
    lp_finish<FMT>(a, r, row, p, sKeys);
  } else {
    const int64_t to = r * a.parts + part;
    if (tid == 0) reinterpret_cast<LpPart*>(a.part)[to] = p;
    if constexpr (TOP)
      for (int i = tid; i < a.top_n; i += LP_NT) a.part_keys[to * a.top_n + i] = sKeys[i];
  }
}

// A workgroup per row joins its parts: the sums in a wave, the sorted lists by a sort of all.
template <int FMT>
__global__ void __launch_bounds__(LP_NT) logprob_join_kernel(LogprobArgs a) {
  __shared__ uint64_t sKeys[LP_MAX_PARTS * LP_MAX_TOP];
  __shared__ LpPart sPart;
  const int64_t r = blockIdx.x;
  const int tid = threadIdx.x, n = a.parts * a.top_n;
  for (int i = tid; i < n; i += LP_NT) sKeys[i] = a.part_keys[r * n + i];
  if (tid < kWave) {
    LpPart p{LP_LOWEST, 0.0f, 0.0f, 0.0f};
    if (tid < a.parts) p = reinterpret_cast<const LpPart*>(a.part)[r * a.parts + tid];
    lp_wave_join(p, a.c);
    if (tid == 0) sPart = p;
  }
  __syncthreads();
  if (a.top_n > 0) lp_sort(sKeys, n, lp_pow2(n));
  const void* const row = reinterpret_cast<const uint8_t*>(a.logits) +
                          r * a.ld * (FMT == SDX_F32 ? 4 : 2);
  lp_finish<FMT>(a, r, row, sPart, sKeys);
}

// Parts of a row: about LP_WGS workgroups in all, none of less than LP_LEAST elements.
constexpr int64_t LP_WGS = 2048, LP_LEAST = 4096;
int logprob_parts(int64_t rows, int64_t V) {
  const int64_t want = (LP_WGS + rows - 1) / rows;
  return (int)std::max<int64_t>(1, std::min<int64_t>({want, V / LP_LEAST, LP_MAX_PARTS}));
}

template <int FMT>
static hipError_t launch_logprob_t(const LogprobArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)(a.parts * a.rows));
  if (a.top_n > 0) hipLaunchKernelGGL((logprob_kernel<FMT, true>), grid, dim3(LP_NT), 0, s, a);
  else hipLaunchKernelGGL((logprob_kernel<FMT, false>), grid, dim3(LP_NT), 0, s, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.parts == 1) return e;
  hipLaunchKernelGGL((logprob_join_kernel<FMT>), dim3((unsigned)a.rows), dim3(LP_NT), 0, s, a);
  return hipGetLastError();
}

hipError_t launch_logprob(int dtype, const LogprobArgs& a, hipStream_t s) {
  if (dtype == SDX_F32) return launch_logprob_t<SDX_F32>(a, s);
  return dtype == SDX_BF16 ? launch_logprob_t<SDX_BF16>(a, s) : launch_logprob_t<SDX_F16>(a, s);
}

}  // namespace sdx
