// Logits as a server changes them before they are sampled: penalties for tokens that the row
// already holds, biases, grammar masks. Every row of logits is a position of a batch row: one
// (decoding), a chain's or a tree's nodes, whose own path's tokens count as written.
//
//   x = l > 0 ? l / r : l r   where the token is in the history or on the path
//   x = x - f c               c: how often it was written (history behind the prompt, and path)
//   x = x - p                 where c > 0
//   x = x + b                 b: the token's bias entries, added up in their order
//   -inf                      where the grammar refuses the token
//
// in fp32, rounded once to the logits' type; a logit that none of them concerns keeps its bits.
// The transforms of specdec/sampling.py:34-67 follow it (temperature, top-k, top-p).
//
// Bound by HBM: each logit is read and written once. A workgroup takes a slice of the
// vocabulary for a few consecutive rows. What a batch row holds of the slice is counted in LDS,
// a word per token and a bit for those that have one, from a scan of its history (8 bytes a
// token, from L2 for all slices but the first), once for all of the batch row's positions; a
// position's path is added to the words and taken off again. A row passes through registers in
// 16-byte units, whose logits are asked for before the words are built; eight tokens' bits say
// whether any of them is looked at by itself, the lanes' one after another, so that a few
// tokens a unit cost little. Rows that start anywhere: a row's units begin where its addresses
// are multiples of 16, and the words have room for a unit in front of the slice. Results are
// stored past the L2, whose write-back at a kernel's end is waited for.
//
// Measured, bf16, V = 151,936: 256 rows that decode, histories of up to 2,048 and 4 biases 44.2 us
// (159 MB, 3.6 TB/s); 8 trees of 32 nodes under grammars, histories of up to 8,192 34.6 us (122 MB,
// 3.5 TB/s). Without histories the same 256 rows take 26 us (6.0 TB/s), with 2,048 tokens each 38:
// their loads, counting and the tokens' own changes have a few us each. Not faster: histories and
// biases asked for a unit ahead (spilled registers), the tokens' changes in LDS by a thread per 32
// (another 16 KB, three workgroups a CU in place of four), atomics of several slots at once. 8 fp32 rows of 50,257: 6.8 us, of which an empty launch is 3.6.
#include <algorithm>

#include "sdx_launch.hpp"

namespace sdx {

constexpr int PN_NT = 256;
constexpr int PN_S = 8192;    // tokens of a slice of 16-bit logits
constexpr int PN_WGS = 1024;  // workgroups that the chip holds at once, by their LDS: 256 x 151,936 bf16 take
                              // 44.2 us, with half as many 65.9; twice as many slow trees by 14 %
constexpr int PN_UN = 8;      // history tokens in flight per thread
// a token's word: seen in the history, 1 + the index of its bias, times written
constexpr uint32_t PN_SEEN = 0x80000000u, PN_COUNT = (1u << 20) - 1;
static_assert(PN_HISTORY + TREE_MAX_NODES <= (int64_t)PN_COUNT && PN_MAX_BIAS < 2047, "fields of a word");

template <int DT>
struct PnType;
template <>
struct PnType<SDX_F32> {
  typedef uint32_t raw;
  static __device__ __forceinline__ float get(uint32_t x) { return __uint_as_float(x); }
  static __device__ __forceinline__ uint32_t put(float x) { return __float_as_uint(x); }
  static constexpr uint32_t kNegInf = 0xFF800000u;
};
template <>
struct PnType<SDX_BF16> {
  typedef uint16_t raw;
  static __device__ __forceinline__ float get(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }
  static __device__ __forceinline__ uint16_t put(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }
  static constexpr uint16_t kNegInf = 0xFF80u;
};
template <>
struct PnType<SDX_F16> {
  typedef uint16_t raw;
  static __device__ __forceinline__ float get(uint16_t x) { return (float)__builtin_bit_cast(_Float16, x); }
  static __device__ __forceinline__ uint16_t put(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }
  static constexpr uint16_t kNegInf = 0xFC00u;
};

// the last i in [0, n) with cu[i] <= x, or 0: the wave looks at 64 places at a time, so a batch
// takes two loads that depend on each other, not eight. Ends for any contents of cu.
__device__ __forceinline__ int64_t pn_find(const int64_t* cu, int64_t n, int64_t x) {
  int64_t lo = 0, len = n;
  while (len > 1) {  // uniform
    const int64_t step = (len + kWave - 1) / kWave, i = lo + (threadIdx.x & (kWave - 1)) * step;
    const uint64_t m = __ballot(i < lo + len && cu[min(i, n - 1)] <= x);
    const int64_t at = m ? (63 - __clzll((long long)m)) * step : 0;
    len = min(step, len - at);
    lo += at;
  }
  return lo;
}

// element k of a 16-byte unit
template <typename raw>
__device__ __forceinline__ raw pn_get(const uint4& v, int k) {
  constexpr int P = sizeof(raw) == 2 ? 2 : 1;  // elements of a dword
  const int d = k / P;
  const uint32_t lo = d & 1 ? v.y : v.x, up = d & 1 ? v.w : v.z;
  return (raw)((d & 2 ? up : lo) >> (P == 2 ? 16 * (k & 1) : 0));
}
template <typename raw>
__device__ __forceinline__ void pn_set(uint4& v, int k, raw y) {
  constexpr int P = sizeof(raw) == 2 ? 2 : 1;
  const int d = k / P;
  const uint32_t keep = P == 2 ? (k & 1 ? 0x0000FFFFu : 0xFFFF0000u) : 0u, at = (uint32_t)y << (P == 2 ? 16 * (k & 1) : 0);
  v.x = d == 0 ? (v.x & keep) | at : v.x;
  v.y = d == 1 ? (v.y & keep) | at : v.y;
  v.z = d == 2 ? (v.z & keep) | at : v.z;
  v.w = d == 3 ? (v.w & keep) | at : v.w;
}

// What a batch row asks of a logit.
struct PnRow {
  float rep, freq, pres;
};
template <int DT>
__device__ __forceinline__ typename PnType<DT>::raw pn_apply(typename PnType<DT>::raw l, uint32_t w, const PnRow& p,
                                                             const float* sBias) {
  typedef PnType<DT> Ty;
  if (w == 0) return l;
  float x = Ty::get(l);
  const uint32_t c = w & PN_COUNT, e = (w & ~PN_SEEN) >> 20;
  if ((w & PN_SEEN) || c > 0) x = x > 0.0f ? x / p.rep : x * p.rep;
  if (c > 0) {
    x -= p.freq * (float)c;
    x -= p.pres;
  }
  if (e > 0) x += sBias[e - 1];
  return Ty::put(x);
}

// S: tokens of a slice
template <int DT, int S>
__global__ void __launch_bounds__(PN_NT) __attribute__((amdgpu_waves_per_eu(4))) penalize_kernel(PenalizeArgs a) {
  typedef PnType<DT> Ty;
  typedef typename Ty::raw raw;
  constexpr int E = 16 / (int)sizeof(raw);   // elements of a unit
  constexpr int NV = S / E / PN_NT;          // units of a thread
  static_assert(S % (E * PN_NT) == 0, "whole units");
  __shared__ __align__(16) uint32_t sWord[S + E];       // of tokens vb ..
  __shared__ __align__(16) uint32_t sBit[S / 32 + 4];   // words that are not 0
  extern __shared__ float sBias[];                      // [biases], then their tokens
  uint16_t* const sBiasAt = reinterpret_cast<uint16_t*>(sBias + a.biases);
  const int tid = threadIdx.x;
  // the units of this workgroup: (slice, row) pairs, the rows of a slice one after another
  uint32_t u = blockIdx.x * a.each + min(blockIdx.x, a.more);
  const uint32_t u1 = u + a.each + (blockIdx.x < a.more);
  int64_t slice = u / (uint32_t)a.rows, r = u - (uint32_t)slice * (uint32_t)a.rows;
  // a row whose first token lies `mis` elements behind a multiple of 16 bytes has tokens
  // slice S - mis .. + S in the slice, inside [vb, vb + S + E) for every row
  const uint64_t nb = S + E;
  int64_t b = 0, have = -1;
  PnRow p = {};
  int64_t q0 = 0, q1 = 0;
  bool ok = false;
  const int V = (int)a.V;  // 2^30 at most
  auto first = [&](int64_t sl, int64_t row) -> int {  // (a.vec: its address is a multiple of 16)
    const uintptr_t at = (uintptr_t)((const raw*)a.logits + row * a.ld);
    return (int)(sl * S) - (a.vec ? (int)(at % 16 / sizeof(raw)) : 0);
  };
  uint4 x[NV], ahead[NV];  // a unit's logits, asked for a unit ahead
  auto load = [&](int64_t sl, int64_t row) {
    if (!a.vec) return;
    const raw* const src = (const raw*)a.logits + row * a.ld;
    const int v0 = first(sl, row);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int v = v0 + (tid + k * PN_NT) * E;
      if (v >= 0 && v + E <= V) ahead[k] = *reinterpret_cast<const uint4*>(src + v);
    }
  };
  load(slice, r);
  bool found = false;
  for (; u < u1; ++u) {  // uniform
#pragma unroll
    for (int k = 0; k < NV; ++k) x[k] = ahead[k];
    const int v0 = first(slice, r), vb = (int)(slice * S) - E;
    const raw* const src = (const raw*)a.logits + r * a.ld;
    raw* const dst = (raw*)a.out + r * a.out_ld;
    const uint32_t* const bits = a.allowed ? a.allowed + r * a.allowed_ld : nullptr;
    const bool last = r + 1 == a.rows;
    if (u + 1 < u1) load(last ? slice + 1 : slice, last ? 0 : r + 1);
    if (!a.cu_rows) {
      b = r;
    } else if (!found) {
      b = pn_find(a.cu_rows, a.batch, r);
      found = true;
    } else {
      while (b + 1 < a.batch && r >= (b == have ? q1 : a.cu_rows[b + 1])) ++b;
    }
    if (b != have) {  // uniform: what the batch row holds of the slice
      have = b;
      q0 = a.cu_rows ? a.cu_rows[b] : b;
      q1 = a.cu_rows ? a.cu_rows[b + 1] : b + 1;
      const int64_t len = a.history ? a.history_len[b] : 0;
      const int64_t prompt = a.history && a.prompt_len ? a.prompt_len[b] : 0;
      ok = q0 >= 0 && q1 >= q0 && q1 <= a.rows && (!a.node_tokens || q1 - q0 <= TREE_MAX_NODES) && len >= 0 &&
           len <= a.max_history && prompt >= 0 && prompt <= len;
      if (!ok && tid == 0 && a.error) *a.error = 1;
      p.rep = a.repetition ? a.repetition[b] : 1.0f;
      p.freq = a.frequency ? a.frequency[b] : 0.0f;
      p.pres = a.presence ? a.presence[b] : 0.0f;
      // the first tokens are asked for before the words are cleared
      const uint8_t* const h = reinterpret_cast<const uint8_t*>(a.history + b * a.history_ld);
      const int n = ok ? (int)len : 0;
      uint2 y[PN_UN];  // tokens
      auto fetch = [&](int i0) {
#pragma unroll
        for (int k = 0; k < PN_UN; ++k)
          y[k] = *reinterpret_cast<const uint2*>(h + min((uint32_t)(tid + i0 + k * PN_NT) * 8u, (uint32_t)(n - 1) * 8u));
      };
      if (n > 0) fetch(0);
      uint32_t mine = 0;
      __syncthreads();  // the words are read no more
      for (int i = tid * 4; i < S + E; i += PN_NT * 4)
        *reinterpret_cast<uint4*>(&sWord[i]) = make_uint4(0, 0, 0, 0);
      for (int i = tid; i < S / 32 + 4; i += PN_NT) sBit[i] = 0;
      if (ok)
        for (int e = tid; e < a.biases; e += PN_NT) {
          const uint64_t z = (uint64_t)(a.bias_ids[b * a.biases + e] - vb);
          sBiasAt[e] = z < nb ? (uint16_t)z : 0xFFFFu;
          sBias[e] = a.bias[b * a.biases + e];
        }
      __syncthreads();
      if (ok) {
        for (int i0 = 0; i0 < n;) {  // uniform. A wave's instruction takes four clocks: few of them per token
#pragma unroll
          for (int k = 0; k < PN_UN; ++k) {
            const uint32_t t = y[k].x - (uint32_t)vb;
            if (t >= (uint32_t)nb || y[k].y != 0 || tid >= n - i0 - k * PN_NT) continue;
            if (tid < (int)prompt - i0 - k * PN_NT) atomicOr(&sWord[t], PN_SEEN);
            else atomicAdd(&sWord[t], 1u);
            atomicOr(&sBit[t / 32], 1u << (t % 32));
          }
          i0 += PN_UN * PN_NT;
          if (i0 < n) fetch(i0);
        }
        // bias entries of the slice, counted in the field of their index; whoever finds it at 0 sees
        // to the token
        for (int e = tid, k = 0; e < a.biases; e += PN_NT, ++k) {
          const uint32_t t = sBiasAt[e];
          if (t == 0xFFFFu) continue;
          if (((atomicAdd(&sWord[t], 1u << 20) & ~PN_SEEN) >> 20) == 0) mine |= 1u << k;
          atomicOr(&sBit[t / 32], 1u << (t % 32));
        }
      }
      __syncthreads();
      if (a.biases > 0) {  // uniform
        const int lane = tid & (kWave - 1);
        for (int e0 = 0, k = 0; e0 < a.biases; e0 += PN_NT, ++k) {  // uniform
          const int e = e0 + tid;
          const bool own = (mine >> k) & 1;
          const uint32_t t = own ? sBiasAt[e] : 0u, n = own ? (sWord[t] & ~PN_SEEN) >> 20 : 0u;
          uint64_t several = __ballot(n > 1);
          while (several) {  // uniform: the sum of a token's entries, in their order, by the wave
            const int who = __ffsll((unsigned long long)several) - 1;
            several &= several - 1;
            const uint32_t z = rdlane(t, who);
            float y = 0.0f;
            bool any = false;
            for (int f0 = 0; f0 < a.biases; f0 += kWave) {
              const int f = min(f0 + lane, a.biases - 1);
              const float x = sBias[f];
              uint64_t hit = __ballot(f0 + lane < a.biases && sBiasAt[f] == z);
              for (; hit; hit &= hit - 1) {
                const float v = __uint_as_float(rdlane(__float_as_uint(x), __ffsll((unsigned long long)hit) - 1));
                y = any ? y + v : v;
                any = true;
              }
            }
            if (lane == who) sBias[e] = y;
          }
          if (own) atomicAdd(&sWord[t], (uint32_t)(e + 1 - n) << 20);  // the field: n, now e + 1
        }
        __syncthreads();
      }
    }
    const bool row = ok && r >= q0 && r < q1;  // a position of the batch row
    // the path of the position: nodes j of the row, by the mask, or those up to its own. Bits
    // stay behind it, with words of 0
    auto path = [&](uint32_t add) {
      if (!row) return;
      const int i = (int)(r - q0), n = (int)(q1 - q0);
      for (int j = tid; j < n; j += PN_NT) {
        bool on = j <= i;
        if (a.tree_mask) on = j < a.mask_words * 64 && (a.tree_mask[r * a.mask_words + j / 64] >> (j % 64)) & 1;
        if (!on) continue;
        const uint64_t t = (uint64_t)(a.node_tokens[q0 + j] - vb);
        if (t >= nb) continue;
        atomicAdd(&sWord[t], add);
        if (add == 1u) atomicOr(&sBit[t / 32], 1u << (t % 32));
      }
    };
    if (a.node_tokens) {
      path(1u);
      __syncthreads();
    }
    auto single = [&](int v) {  // token v by itself
      raw y = row ? pn_apply<DT>(src[v], sWord[v - vb], p, sBias) : src[v];
      if (row && bits && !((bits[v / 32] >> (v % 32)) & 1)) y = Ty::kNegInf;
      dst[v] = y;
    };
    if (a.vec) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int v = v0 + (tid + k * PN_NT) * E;
        if (v >= 0 && v + E <= V) {
          if (row) {
            uint32_t may = (1u << E) - 1;
            if (bits) {
              const uint8_t* const at = reinterpret_cast<const uint8_t*>(bits) + v / 8;
              uint32_t m = *at;
              if ((v % 8) + E > 8) m |= (uint32_t)at[1] << 8;
              may &= m >> (v % 8);
            }
            const uint32_t t = (uint32_t)(v - vb);
            const uint64_t two = (uint64_t)sBit[t / 32 + 1] << 32 | sBit[t / 32];
            uint32_t todo = (uint32_t)(two >> (t % 32)) & may;
            while (todo) {
              const int i = __ffs(todo) - 1;
              todo &= todo - 1;
              pn_set<raw>(x[k], i, pn_apply<DT>(pn_get<raw>(x[k], i), sWord[t + i], p, sBias));
            }
            if (may != (1u << E) - 1) {
              uint32_t* const d = reinterpret_cast<uint32_t*>(&x[k]);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                if constexpr (E == 8) {
                  const uint32_t m = ((may >> (2 * i)) & 1 ? 0xFFFFu : 0u) | ((may >> (2 * i + 1)) & 1 ? 0xFFFF0000u : 0u);
                  d[i] = (d[i] & m) | (((uint32_t)Ty::kNegInf << 16 | Ty::kNegInf) & ~m);
                } else {
                  d[i] = (may >> i) & 1 ? d[i] : (uint32_t)Ty::kNegInf;
                }
              }
            }
          }
          store_nt(dst + v, x[k]);
        }
      }
      // the row's ends, where a unit is not whole
      const int head = v0 < 0 ? E + v0 : 0, tail = v0 + (V - v0) / E * E;
      if (v0 < 0 && tid < min(head, V)) single(tid);
      if (tail >= head && tail < v0 + S && tid < V - tail) single(tail + tid);
    } else {
      for (int v = v0 + tid; v < min(v0 + S, V); v += PN_NT) single(v);
    }
    if (a.node_tokens) {
      __syncthreads();
      path(~0u);
    }
    if (++r == a.rows) {  // the next slice, from its first row
      r = 0;
      ++slice;
      have = -1;
      found = false;
    }
  }
}

// ---------------------------------------------------------------- launches
template <int DT, int S>
static hipError_t launch_penalize_s(const PenalizeArgs& b, hipStream_t s) {
  PenalizeArgs a = b;
  const int64_t E = 16 / (DT == SDX_F32 ? 4 : 2), slices = (a.V + (a.vec ? E - 1 : 0) + S - 1) / S;
  // as many workgroups as the chip holds at once (units: under 2^32, sdx_penalize_logits sees to it)
  const uint32_t units = (uint32_t)(a.rows * slices);
  const dim3 grid(std::min<uint32_t>(units, S > PN_NT * 8 ? PN_WGS : 2 * PN_WGS));
  a.each = units / grid.x;
  a.more = units % grid.x;
  hipLaunchKernelGGL((penalize_kernel<DT, S>), grid, dim3(PN_NT), (unsigned)(6 * a.biases), s, a);
  return hipGetLastError();
}

template <int DT>
static hipError_t launch_penalize_t(const PenalizeArgs& a, hipStream_t s) {
  constexpr int few = PN_NT * 8, many = DT == SDX_F32 ? PN_S / 2 : PN_S;
  // Short slices spread few logits over more workgroups, long ones go through a history less often.
  // bf16 rows of 151,936, histories of 1,000: 8 rows take 6.0 us in short slices and 7.3 in long
  // ones, 16 rows 8.4 and 7.7, 100 rows 27.9 and 16.4. A vocabulary within one short slice takes it whatever
  // the rows (6,000 rows of 1,000: 35.7 and 39.3 us).
  if (a.V + 7 <= few || a.rows * ((a.V + PN_S - 1) / PN_S) < 256) return launch_penalize_s<DT, few>(a, s);
  return launch_penalize_s<DT, many>(a, s);
}

hipError_t launch_penalize(int dtype, const PenalizeArgs& a, hipStream_t s) {
  if (dtype == SDX_F32) return launch_penalize_t<SDX_F32>(a, s);
  return dtype == SDX_BF16 ? launch_penalize_t<SDX_BF16>(a, s) : launch_penalize_t<SDX_F16>(a, s);
}

}  // namespace sdx
