// Logits as a server changes them before they are sampled: penalties for tokens that the row
// already holds, biases, grammar masks. Every row of logits is a position of a batch row: one
// (decoding), a chain's or a tree's nodes, whose own path's tokens count as written.
//
//   x = l > 0 ? l / r : l r   where the token is in the history or on the path
//   x = x - f c               c: how often it was written (history behind the prompt, and path)
//   x = x - p                 where c > 0
//   x = x + b                 of the token's bias entries, in their order
//   -inf                      where the grammar refuses the token
//
// in fp32, rounded once to the logits' type; a logit that none of them concerns keeps its bits.
// The transforms of specdec/sampling.py:34-67 follow it (temperature, top-k, top-p).
//
// Bound by HBM: each logit is read and written once. A workgroup takes a slice of the
// vocabulary for a few consecutive rows. What a batch row holds of the slice is counted in LDS,
// a word per token, from a scan of its history (8 bytes a token, from L2 for all slices but the
// first), once for all of the batch row's positions; a position's path is added to the words
// and taken off again.
#include <algorithm>

#include "sdx_launch.hpp"

namespace sdx {

constexpr int PN_NT = 256;
// a token's word: seen in the history, has a bias, times on the path, times written before
constexpr uint32_t PN_SEEN = 0x80000000u, PN_BIAS = 0x40000000u, PN_PATH = 1u << 20;
constexpr uint32_t PN_COUNT = PN_PATH - 1;
static_assert(TREE_MAX_NODES < 1024 && PN_HISTORY <= (int64_t)PN_COUNT, "counts fit their bits");

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

// the last i in [0, n) with cu[i] <= x, or 0
__device__ __forceinline__ int64_t pn_find(const int64_t* cu, int64_t n, int64_t x) {
  int64_t lo = 0, hi = n;
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) / 2;
    if (cu[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

template <int DT, int S>
__global__ void __launch_bounds__(PN_NT) penalize_kernel(PenalizeArgs a) {
  typedef PnType<DT> Ty;
  typedef typename Ty::raw raw;
  constexpr int E = 16 / (int)sizeof(raw);   // elements of 16 bytes
  __shared__ __align__(16) uint32_t sWord[S];
  __shared__ float sBias[PN_MAX_BIAS];
  __shared__ uint16_t sBiasAt[PN_MAX_BIAS];
  __shared__ int sBiases;
  const int tid = threadIdx.x;
  const int64_t v0 = (int64_t)blockIdx.x * S;
  const int ns = (int)min((int64_t)S, a.V - v0);
  const int64_t r0 = (int64_t)blockIdx.y * a.rows_each, r1 = min(a.rows, r0 + a.rows_each);
  const raw* const in = (const raw*)a.logits + v0;
  raw* const out = (raw*)a.out + v0;
  int64_t b = a.cu_rows ? pn_find(a.cu_rows, a.batch, r0) : r0, have = -1;
  float rep = 1.0f, freq = 0.0f, pres = 0.0f;
  int64_t q0 = 0, q1 = 0;
  bool ok = false, held = false;  // (held: the words are not all zero)
  for (int64_t r = r0; r < r1; ++r) {
    if (a.cu_rows)
      while (b + 1 < a.batch && r >= a.cu_rows[b + 1]) ++b;
    else b = r;
    if (b != have) {  // uniform: what the batch row holds of the slice
      have = b;
      q0 = a.cu_rows ? a.cu_rows[b] : b;
      q1 = a.cu_rows ? a.cu_rows[b + 1] : b + 1;
      const int64_t len = a.history ? a.history_len[b] : 0;
      const int64_t prompt = a.history && a.prompt_len ? a.prompt_len[b] : 0;
      ok = q0 >= 0 && q1 >= q0 && q1 <= a.rows && (!a.node_tokens || q1 - q0 <= TREE_MAX_NODES) && len >= 0 &&
           len <= a.max_history && prompt >= 0 && prompt <= len;
      if (!ok && tid == 0 && a.error) *a.error = 1;
      rep = a.repetition ? a.repetition[b] : 1.0f;
      freq = a.frequency ? a.frequency[b] : 0.0f;
      pres = a.presence ? a.presence[b] : 0.0f;
      __syncthreads();  // the words are read no more
      for (int i = tid * 4; i < S; i += PN_NT * 4)
        *reinterpret_cast<uint4*>(&sWord[i]) = make_uint4(0, 0, 0, 0);
      if (tid == 0) sBiases = 0;
      __syncthreads();
      if (ok) {
        const int64_t* const h = a.history + b * a.history_ld;
        for (int64_t i = tid; i < len; i += PN_NT) {
          const uint64_t x = (uint64_t)(h[i] - v0);
          if (x >= (uint64_t)ns) continue;
          if (i < prompt) atomicOr(&sWord[x], PN_SEEN);
          else atomicAdd(&sWord[x], 1u);
        }
        if (a.biases > 0 && tid < kWave) {  // in order: the entries of one token add up in theirs
          int n = 0;
          for (int e0 = 0; e0 < a.biases; e0 += kWave) {
            const int e = e0 + tid;
            const uint64_t x = e < a.biases ? (uint64_t)(a.bias_ids[b * a.biases + e] - v0) : ~0ull;
            const bool mine = x < (uint64_t)ns;
            const uint64_t m = __ballot(mine);
            if (mine) {
              const int at = n + __popcll(m & ((1ull << tid) - 1));
              sBiasAt[at] = (uint16_t)x;
              sBias[at] = a.bias[b * a.biases + e];
              atomicOr(&sWord[x], PN_BIAS);
            }
            n += __popcll(m);
          }
          if (tid == 0) sBiases = n;
        }
      }
      __syncthreads();
    }
    const bool row = ok && r >= q0 && r < q1;  // a position of the batch row
    // the path of the position: nodes j of the row, by the mask, or those up to its own
    auto path = [&](uint32_t add) {
      if (!row || !a.node_tokens) return;
      const int i = (int)(r - q0), n = (int)(q1 - q0);
      for (int j = tid; j < n; j += PN_NT) {
        bool on = j <= i;
        if (a.tree_mask) on = j < a.mask_words * 64 && (a.tree_mask[r * a.mask_words + j / 64] >> (j % 64)) & 1;
        if (!on) continue;
        const uint64_t x = (uint64_t)(a.node_tokens[q0 + j] - v0);
        if (x < (uint64_t)ns) atomicAdd(&sWord[x], add);
      }
    };
    if (a.node_tokens) {
      path(PN_PATH);
      __syncthreads();
    }
    const uint32_t* const bits = a.allowed && row ? a.allowed + r * a.allowed_ld : nullptr;
    auto one = [&](raw l, int i) -> raw {  // token v0 + i
      const uint32_t w = row ? sWord[i] : 0u;
      raw y = l;
      if (w) {
        float x = Ty::get(l);
        const uint32_t c = (w & PN_COUNT) + ((w & ~(PN_SEEN | PN_BIAS)) / PN_PATH);
        if ((w & PN_SEEN) || c > 0) x = x > 0.0f ? x / rep : x * rep;
        if (c > 0) {
          x -= freq * (float)c;
          x -= pres;
        }
        if (w & PN_BIAS)
          for (int e = 0; e < sBiases; ++e)
            if (sBiasAt[e] == i) x += sBias[e];
        y = Ty::put(x);
      }
      return y;
    };
    const raw* const src = in + r * a.ld;
    raw* const dst = out + r * a.out_ld;
    if (a.vec) {  // rows of 16-byte units
      for (int i = tid * E; i < ns; i += PN_NT * E) {
        if (i + E <= ns) {
          union { uint4 v; raw x[E]; } u;
          u.v = *reinterpret_cast<const uint4*>(src + i);
          uint32_t ok8 = ~0u;
          if (bits) ok8 = bits[(v0 + i) / 32] >> ((v0 + i) % 32);
#pragma unroll
          for (int k = 0; k < E; ++k) {
            u.x[k] = one(u.x[k], i + k);
            if (!((ok8 >> k) & 1)) u.x[k] = Ty::kNegInf;
          }
          *reinterpret_cast<uint4*>(dst + i) = u.v;
        } else {
          for (int k = i; k < ns; ++k)
            dst[k] = bits && !((bits[(v0 + k) / 32] >> ((v0 + k) % 32)) & 1) ? Ty::kNegInf : one(src[k], k);
        }
      }
    } else {
      for (int i = tid; i < ns; i += PN_NT)
        dst[i] = bits && !((bits[(v0 + i) / 32] >> ((v0 + i) % 32)) & 1) ? Ty::kNegInf : one(src[i], i);
    }
    if (a.node_tokens) {
      __syncthreads();
      path(0u - PN_PATH);
    }
  }
}

// ---------------------------------------------------------------- launches
template <int DT>
static hipError_t launch_penalize_t(const PenalizeArgs& b, hipStream_t s) {
  PenalizeArgs a = b;
  constexpr int S = 8192;
  const int64_t slices = (a.V + S - 1) / S;
  a.rows_each = std::max<int64_t>(1, std::min<int64_t>(64, a.rows * slices / 1024));
  const dim3 grid((unsigned)slices, (unsigned)((a.rows + a.rows_each - 1) / a.rows_each));
  hipLaunchKernelGGL((penalize_kernel<DT, S>), grid, dim3(PN_NT), 0, s, a);
  return hipGetLastError();
}

hipError_t launch_penalize(int dtype, const PenalizeArgs& a, hipStream_t s) {
  if (dtype == SDX_F32) return launch_penalize_t<SDX_F32>(a, s);
  return dtype == SDX_BF16 ? launch_penalize_t<SDX_BF16>(a, s) : launch_penalize_t<SDX_F16>(a, s);
}

}  // namespace sdx
