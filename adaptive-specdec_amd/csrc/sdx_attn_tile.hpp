// Device code that the attention kernels over the paged cache share (sdx_prefix_attn.hip,
// sdx_tree_attn.hip): tiles of 64 keys against the 32 query rows of a wave.
//
// S^T = K Q^T with v_mfma_f32_32x32x16: lane l then holds 16 keys' scores of query l % 32, so
// maxima and sums stay in the lane (one exchange with lane l ^ 32), and the weights, rounded to
// 16 bits, are the second operand of O^T = V^T P^T as they lie.
#pragma once

#include "sdx_launch.hpp"

namespace sdx {

constexpr int PA_NT = 256;
constexpr int PA_TILE = 64;       // keys per tile
constexpr int PA_ROWS = 128;      // query rows of a workgroup
constexpr int PA_WROWS = 32;      // query rows per wave
constexpr uint32_t PA_NOSLOT = 0xFFFFFFFFu;
constexpr int PA_RING = 8;        // tiles of slots
constexpr float PA_SLACK = 8.0f;  // log2 by which a weight may pass its step of the maximum
// log2 of the weight that such a step gives the largest score. An fp16 weight below 2^-14 is rounded
// to a multiple of 2^-24, which adds up over many keys far below the largest: n keys lose up to
// n 2^-25 of the output with 1 as the largest weight, eight half steps of the type at 131,072, and
// n 2^-32 with 2^7 (2^15 with the slack, below the type's 65,504). bf16 has fp32's exponents.
template <int FMT>
constexpr float pa_lift() { return FMT == SDX_F16 ? 7.0f : 0.0f; }

typedef short pa_s4 __attribute__((ext_vector_type(4)));
typedef uint32_t pa_u4 __attribute__((ext_vector_type(4)));
typedef __bf16 pa_bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 pa_h8 __attribute__((ext_vector_type(8)));
typedef float pa_f16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) pa_s4 pa_lds_s4;

// v_mfma_f32_32x32x16: lane l holds A[l % 32][8 (l / 32) .. + 7], B[8 (l / 32) .. + 7][l % 32]
// and D[8 (i / 4) + 4 (l / 32) + i % 4][l % 32] in element i.
template <int FMT>
__device__ __forceinline__ pa_f16 pa_mfma(pa_u4 a, pa_u4 b, pa_f16 c) {
  if constexpr (FMT == SDX_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(pa_bf8, a),
                                                   __builtin_bit_cast(pa_bf8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(pa_h8, a),
                                                  __builtin_bit_cast(pa_h8, b), c, 0, 0, 0);
}
// two fp32 rounded to 16 bits (nearest even), x in the low half
template <int FMT>
__device__ __forceinline__ uint32_t pa_pack(float x, float y) {
  if constexpr (FMT == SDX_BF16) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, (b2){(__bf16)x, (__bf16)y});
  } else {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, (h2){(_Float16)x, (_Float16)y});
  }
}
// the values of lanes l and l ^ 32 in both
__device__ __forceinline__ float pa_max_halves(float x) {
  typedef uint32_t u2 __attribute__((ext_vector_type(2)));
  const u2 r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float pa_sum_halves(float x) {
  typedef uint32_t u2 __attribute__((ext_vector_type(2)));
  const u2 r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// the last i in [0, n) with cu[i] <= x, or 0
__device__ __forceinline__ int64_t pa_find(const int64_t* cu, int64_t n, int64_t x) {
  int64_t lo = 0, hi = n;
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) / 2;
    if (cu[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// The running state of a wave's 32 query rows: lane l holds row l % 32, and of O^T the
// dims 32 db + 8 (i / 4) + 4 (l / 32) + i % 4 in o[db][i]. l is of the lane's own keys.
template <int D>
struct PaState {
  pa_f16 o[D / 32];
  float m, l;
};

// Weights of NB x 32 scores, in s. st.m is the largest score in log2 so far, less the lift and up to
// the slack, which is tested with the weights' own argument: none passes 2^(lift + slack).
template <int D, int FMT, int NB>
__device__ __forceinline__ void pa_softmax(PaState<D>& st, pa_f16 (&s)[NB], float scale) {
  float mx = s[0][0];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[nb][i]);
  constexpr float LIFT = pa_lift<FMT>();
  mx = pa_max_halves(mx);
  if (__any(fmaf(mx, scale, -st.m) > LIFT + PA_SLACK)) {
    const float mn = fmaxf(st.m, mx * scale - LIFT);
    const float alpha = st.m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(st.m - mn);
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) st.o[db][i] *= alpha;
    st.l *= alpha;
    st.m = mn;
  }
  const float off = st.m == -INFINITY ? 0.0f : -st.m;  // no key seen yet: all weights 0
  float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[nb][i] = __builtin_amdgcn_exp2f(fmaf(s[nb][i], scale, off));
      sum[i % 4] += s[nb][i];
    }
  st.l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

// 16-byte chunk c of row r of a tile in LDS lies in chunk c ^ swizzle(r): the operand reads of
// a phase then fall into different banks of the 64. K rows are read 16 bytes a lane, 16 rows
// at a time; V rows 64 bytes of 4 rows at a time.
template <int D>
__device__ __forceinline__ int pa_swz_k(int r) { return r & (D / 8 - 1); }
template <int D>
__device__ __forceinline__ int pa_swz_v(int r) { return D == 128 ? 4 * (r & 3) : 4 * ((r >> 1) & 1); }

// O^T += V^T P^T for NB x 32 keys. va: the lane's byte address in V's first row block. The
// operands of AHEAD products are read ahead.
template <int D, int FMT, int NB, int AHEAD = 4>
__device__ __forceinline__ void pa_pv(PaState<D>& st, const pa_f16 (&s)[NB], const uint8_t* sV,
                                      uint32_t va) {
  constexpr int DB = D / 32, N = NB * 2 * DB;
  pa_u4 x[AHEAD];
  auto read = [&](int j) {  // product j: keys 16 (j / DB) .., dims 32 (j % DB) ..
    const uint8_t* const at = sV + (va ^ ((j % DB) << 6)) + 16 * (j / DB) * 2 * D;
    typedef uint32_t u2 __attribute__((ext_vector_type(2)));
    const u2 lo = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((pa_lds_s4*)at));
    const u2 up = __builtin_bit_cast(
        u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((pa_lds_s4*)(at + 8 * 2 * D)));
    x[j % AHEAD] = (pa_u4){lo[0], lo[1], up[0], up[1]};
  };
#pragma unroll
  for (int j = 0; j < AHEAD; ++j) read(j);
  pa_u4 p;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int k = j / DB;
    if (j % DB == 0) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        p[e] = pa_pack<FMT>(s[k / 2][8 * (k % 2) + 2 * e], s[k / 2][8 * (k % 2) + 2 * e + 1]);
    }
    st.o[j % DB] = pa_mfma<FMT>(x[j % AHEAD], p, st.o[j % DB]);
    if (j + AHEAD < N) read(j + AHEAD);
  }
  // reads (0x100) and products (0x008) in this order; the rest falls between them
  __builtin_amdgcn_sched_group_barrier(0x100, 2 * AHEAD, 0);
#pragma unroll
  for (int j = 0; j < N; ++j) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    if (j + AHEAD < N) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
  }
}

// V in tiles of which some query rows see a part: a weight of 0 times an infinity or a NaN would
// be a NaN, so such elements are 0 for the products, and are added behind the last tile to the
// rows that see their key. One comparison for the largest of a thread's elements costs nothing that
// shows (128 rows of up to 8,192 own keys 414 us with and without, 64 rows 70.9 and 70.8; 0.8 and
// 1.4% when it came in); one for each, or the sums in every tile, 3 to 9%.
template <int FMT, int H>
__device__ __forceinline__ bool pa_finite_only(pa_u4 (&v)[H]) {
  typedef uint16_t h2 __attribute__((ext_vector_type(2)));
  constexpr uint16_t E = FMT == SDX_BF16 ? 0x7F80u : 0x7C00u;
  h2 mx = {0, 0};  // of the elements without their signs
#pragma unroll
  for (int h = 0; h < H; ++h)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      mx = __builtin_elementwise_max(mx, __builtin_bit_cast(h2, v[h][i] & 0x7FFF7FFFu));
  const bool odd = max(mx.x, mx.y) >= E;
  if (__any(odd)) {
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[h][i] &= ((v[h][i] & E) == E ? 0u : 0xFFFFu) | ((v[h][i] >> 16 & E) == E ? 0u : 0xFFFF0000u);
  }
  return odd;
}
template <int FMT>
__device__ __forceinline__ float pa_odd(uint16_t x) {
  if constexpr (FMT == SDX_BF16)
    return __uint_as_float((uint32_t)x << 16);
  else
    return (float)__builtin_bit_cast(_Float16, x);
}

}  // namespace sdx
