// Norms of queries and keys per head and their rotation by position, in one pass.
//
//   x' = x / sqrt(mean_d x_d^2 + eps) * gain          (a row: one head of one token; or x' = x)
//   angle of pair p = position[axis(p)] * inv_freq[p]
//   y_i = x'_i cos - x'_j sin,  y_j = x'_j cos + x'_i sin
//
// with (i, j) = (p, p + pairs) or (2 p, 2 p + 1); dims past the pairs are only normed.  Everything between the load of a
// row and its store is in fp32, rounded once.
//
// The angle is the product in 64 bits: at position 2^20 a product in 32 is off by up to 0.06 rad.  That of a position and a
// frequency of 24 bits is exact up to 2^29; further out it is rounded, by up to 2^-53 of it (1.2e-4 rad at 2^40).  It is reduced to
// [-pi/4, pi/4] and a quadrant in 64 bits, so that sine and cosine are those of a small fp32 argument.  The angles of a token are
// the same for all its heads: a workgroup computes them once, into LDS.
#include <hip/hip_runtime.h>

#include "common.h"
#include "cortex_hip.h"

namespace cortex {
namespace {

constexpr int RP_ERR = 8;        // bit of *err: an axis outside the positions
constexpr int RP_ANGLES = 2048;  // (token, pair) angles of a workgroup, at most
constexpr int RP_MAX_DIM = 256;

struct RopeSide {  // the queries, or the keys
  const void* x;
  int64_t st, sh;
  void* y;
  int64_t yt, yh;
  const void* gain;
  int heads;
  int tokens;     // of a workgroup
  unsigned grid;  // workgroups
};

struct RopeArgs {
  RopeSide side[2];
  int64_t T;
  int dim, pairs, lanes;  // lanes of a row, a power of two
  const int64_t* positions;
  int64_t p_st, p_sa, n_axes;
  const float* inv_freq;
  const int32_t* axes;
  float eps;
  int gain_f32;
  int32_t* err;
};

// 16 bytes of a row, and as numbers.
template <class X>
__device__ __forceinline__ void numbers(const i32x4& w, float* f) {
#pragma unroll
  for (int j = 0; j < 16 / (int)sizeof(X); ++j) {
    if constexpr (sizeof(X) == 4)
      f[j] = __int_as_float(w[j]);
    else
      f[j] = __int_as_float((j & 1) ? (w[j >> 1] & 0xffff0000) : (w[j >> 1] << 16));
  }
}
__device__ __forceinline__ i32x4 packed(const float* f, float) {
  return __builtin_bit_cast(i32x4, f32x4{f[0], f[1], f[2], f[3]});
}
__device__ __forceinline__ i32x4 packed(const float* f, bf16) {
  bf16x8 v;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (bf16)f[e];
  return __builtin_bit_cast(i32x4, v);
}

// Cosine and sine of a 64-bit angle, each rounded from an fp32 argument of at most pi/4.
__device__ __forceinline__ float2 turn(double angle) {
  const double n = rint(angle * 0.63661977236758134308);  // quarter turns
  // pi/2 as the double next to it and the rest: n of each, the first product exact in the fma
  const double r = fma(-n, 6.123233995736766036e-17, fma(-n, 1.5707963267948965580, angle));
  float s, c;
  sincospif((float)(r * 0.31830988618379067154), &s, &c);  // (in half turns: no reduction of large arguments to carry)
  const int quadrant = (int)((int64_t)n & 3);
  const float a = (quadrant & 1) ? s : c, b = (quadrant & 1) ? c : s;
  return make_float2((quadrant == 1 || quadrant == 2) ? -a : a, (quadrant & 2) ? -b : b);
}

// Sum over the `lanes` lanes of a row (1 .. 16, within 16 lanes), in each of them.
__device__ __forceinline__ float row_sum(float v, int lanes) {
  if (lanes > 1) v += dpp_mov<0xB1>(v);   // the neighbour
  if (lanes > 2) v += dpp_mov<0x4E>(v);   // the other two of four
  if (lanes > 4) v += dpp_mov<0x141>(v);  // mirrored within eight
  if (lanes > 8) v += dpp_mov<0x140>(v);  // and within sixteen
  return v;
}

// A workgroup takes `tokens` tokens of the queries or of the keys, and all threads the same number of rounds.  A lane takes
// 16 values of a row in units of 16 bytes, those that turn with each other among them: of the 2 pairs dims that turn the
// units l, l + L, l + 2 L .. (L lanes for them), of the others likewise, so that neighbouring lanes have neighbouring
// units.  The first half of a lane's units turns with the second.
//
// Bound by HBM for many tokens: 16,801 tokens of 32 + 8 heads x 128 in bf16, 344 MB, 71 us, 4.8 TB/s (with eight values a lane,
// whose partners then come through LDS, and four rows at once instead of the next one ahead 168 us; non-temporal stores
// 66.5, but 31 instead of 17 us where only 32 bytes lie side by side).  4999 tokens of 12 + 12 heads x 64 in fp32, 62 MB, 16.6 us:
// the loads, angles and first rows of the one round of workgroups come first.  64 tokens of 32 + 8 heads x 128: 4.7 us, one
// token 3.2.
template <class X, bool NORM, bool INTER>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(RopeArgs a) {
  constexpr int CE = 16 / sizeof(X), NU = 16 / CE;  // values of a unit, units a lane
  __shared__ __attribute__((aligned(16))) float2 angles[RP_ANGLES];  // cosine, sine
  const int tid = threadIdx.x;
  const bool keys = blockIdx.x >= a.side[0].grid;
  const RopeSide& o = a.side[keys];
  const int64_t t0 = (int64_t)(blockIdx.x - (keys ? a.side[0].grid : 0u)) * o.tokens;
  const int count = (int)min((int64_t)o.tokens, a.T - t0);
  const int l = tid & (a.lanes - 1), turning = a.pairs >> 3;  // (256 is a multiple of lanes)
  const bool turned = l < turning;
  const int rest = (a.dim - 2 * a.pairs + 15) >> 4;  // lanes of the dims that do not turn
  const int d0 = turned ? CE * l : 2 * a.pairs + CE * (l - turning), d_step = CE * (turned ? turning : rest);
  // rows: token k, head r; `step` rows further are dk tokens and dr heads
  const int step = 256 / a.lanes, rows = count * o.heads;
  const int dk = step / o.heads, dr = step - dk * o.heads;
  int row = tid / a.lanes, k = row / o.heads, r = row - k * o.heads;
  const X* x = reinterpret_cast<const X*>(o.x) + (t0 + k) * o.st + r * o.sh + d0;
  X* y = reinterpret_cast<X*>(o.y) + (t0 + k) * o.yt + r * o.yh + d0;
  const int64_t x_step = dk * o.st + dr * o.sh, x_wrap = o.st - o.heads * o.sh;
  const int64_t y_step = dk * o.yt + dr * o.yh, y_wrap = o.yt - o.heads * o.yh;
  bool in[NU];
#pragma unroll
  for (int j = 0; j < NU; ++j) in[j] = l < turning + rest && d0 + j * d_step < a.dim;

  // the next row is loaded before this one is computed
  i32x4 w[2][NU];
  int ahead = row, rx = r;
  auto load = [&](i32x4 (&to)[NU]) {
    const bool there = ahead < rows;
#pragma unroll
    for (int j = 0; j < NU; ++j) {
      to[j] = (i32x4){0, 0, 0, 0};
      if (there && in[j]) to[j] = *reinterpret_cast<const i32x4*>(x + j * d_step);
    }
    const bool wrap = (rx += dr) >= o.heads;
    rx -= wrap ? o.heads : 0;
    x += x_step + (wrap ? x_wrap : 0);
    ahead += step;
  };
  load(w[0]);

  float gain[16];
  if constexpr (NORM) {
#pragma unroll
    for (int e = 0; e < 16; ++e) gain[e] = 1.0f;
    if (o.gain) {
#pragma unroll
      for (int j = 0; j < NU; ++j) {
        const int d = d0 + j * d_step;
        if (!in[j]) continue;
        if (a.gain_f32) {
#pragma unroll
          for (int e = 0; e < CE; e += 4)
            numbers<float>(*reinterpret_cast<const i32x4*>(reinterpret_cast<const float*>(o.gain) + d + e), gain + j * CE + e);
        } else {
          bf16 g[CE];
          __builtin_memcpy(g, __builtin_assume_aligned(reinterpret_cast<const bf16*>(o.gain) + d, 2 * CE), 2 * CE);
#pragma unroll
          for (int e = 0; e < CE; ++e) gain[j * CE + e] = to_f32(g[e]);
        }
      }
    }
  }
  for (int i = tid; i < count * a.pairs; i += 256) {
    const int t = i / a.pairs, p = i - t * a.pairs;
    const int axis = a.axes ? a.axes[p] : 0;
    const bool there = (uint64_t)(int64_t)axis < (uint64_t)a.n_axes;
    if (!there && a.err) atomicOr(a.err, RP_ERR);
    const int64_t at = there ? a.positions[(t0 + t) * a.p_st + axis * a.p_sa] : 0;
    angles[i] = turn((double)at * (double)a.inv_freq[p]);
  }
  __syncthreads();

  const float inv_dim = 1.0f / (float)a.dim;
  auto rotate = [&](const i32x4 (&from)[NU]) {
    const bool there = row < rows;
    float f[16];
#pragma unroll
    for (int j = 0; j < NU; ++j) numbers<X>(from[j], f + j * CE);
    if constexpr (NORM) {
      float sum = 0.0f;
#pragma unroll
      for (int e = 0; e < 16; ++e) sum += f[e] * f[e];
      const float inv = rsqrtf(row_sum(sum, a.lanes) * inv_dim + a.eps);
#pragma unroll
      for (int e = 0; e < 16; ++e) f[e] = f[e] * inv * gain[e];
    }
    if (turned && there) {
      const float2* at = angles + k * a.pairs;
      if constexpr (INTER) {
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          const float2 t = at[(d0 + (e / CE) * d_step + e % CE) >> 1];
          const float u = f[e], v = f[e + 1];
          f[e] = u * t.x - v * t.y;
          f[e + 1] = v * t.x + u * t.y;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float2 t = at[d0 + (e / CE) * d_step + e % CE];
          const float u = f[e], v = f[e + 8];
          f[e] = u * t.x - v * t.y;
          f[e + 8] = v * t.x + u * t.y;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < NU; ++j)
      if (there && in[j]) *reinterpret_cast<i32x4*>(y + j * d_step) = packed(f + j * CE, X());
    const bool wrap = (r += dr) >= o.heads;
    r -= wrap ? o.heads : 0;
    k += dk + (wrap ? 1 : 0);
    y += y_step + (wrap ? y_wrap : 0);
    row += step;
  };
  // (lanes of a row add up together: the rounds are the same for all threads)
  for (int done = 0; done < rows; done += 2 * step) {
    load(w[1]);
    rotate(w[0]);
    if (done + step >= rows) break;
    load(w[0]);
    rotate(w[1]);
  }
}

template <class X>
int launch(const RopeArgs& a, bool norm, bool interleaved, hipStream_t stream) {
  const dim3 grid(a.side[0].grid + a.side[1].grid), block(256);
  if (norm && interleaved)
    hipLaunchKernelGGL((qk_norm_rope_kernel<X, true, true>), grid, block, 0, stream, a);
  else if (norm)
    hipLaunchKernelGGL((qk_norm_rope_kernel<X, true, false>), grid, block, 0, stream, a);
  else if (interleaved)
    hipLaunchKernelGGL((qk_norm_rope_kernel<X, false, true>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((qk_norm_rope_kernel<X, false, false>), grid, block, 0, stream, a);
  CORTEX_CHECK_LAUNCH("qk_norm_rope_kernel");
  return OK;
}

}  // namespace
}  // namespace cortex

using namespace cortex;

extern "C" int cortex_qk_norm_rope(int64_t T, int64_t heads, int64_t kv_heads, int64_t dim, int dtype, const void* q,
                                   int64_t q_st, int64_t q_sh, const void* k, int64_t k_st, int64_t k_sh,
                                   const int64_t* positions, int64_t p_st, int64_t p_sa, int64_t n_axes, int64_t pairs,
                                   const float* inv_freq, const int32_t* axes, int interleaved, int norm, float eps,
                                   const void* q_gain, const void* k_gain, int gain_dtype, void* q_out, int64_t qo_st,
                                   int64_t qo_sh, void* k_out, int64_t ko_st, int64_t ko_sh, int32_t* err,
                                   hipStream_t stream) {
  const char* who = "cortex_qk_norm_rope";
  CORTEX_CHECK_ARG(T >= 0 && T <= 0x7fffffffLL && heads >= 0 && kv_heads >= 0 && heads + kv_heads <= 65535,
                   "%s: %lld tokens of %lld + %lld heads", who, (long long)T, (long long)heads, (long long)kv_heads);
  CORTEX_CHECK_ARG(dim >= 8 && dim <= RP_MAX_DIM && dim % 8 == 0, "%s: head dim %lld is not a multiple of 8 up to %d", who,
                   (long long)dim, RP_MAX_DIM);
  CORTEX_CHECK_ARG(pairs >= 0 && pairs % 8 == 0 && 2 * pairs <= dim,
                   "%s: %lld pairs are not a multiple of 8 up to half of the head dim %lld", who, (long long)pairs, (long long)dim);
  CORTEX_CHECK_ARG(dtype == DT_F32 || dtype == DT_BF16, "%s: rows of dtype %d (f32 or bf16)", who, dtype);
  CORTEX_CHECK_ARG(!(q_gain || k_gain) || (norm && (gain_dtype == DT_F32 || gain_dtype == DT_BF16)),
                   "%s: gains (f32 or bf16) belong to the norm", who);
  CORTEX_CHECK_ARG(!norm || eps >= 0.0f, "%s: negative eps", who);
  CORTEX_CHECK_ARG(n_axes >= 1, "%s: %lld axes", who, (long long)n_axes);
  if (T == 0 || heads + kv_heads == 0) return OK;
  CORTEX_CHECK_ARG((heads == 0 || (q && q_out)) && (kv_heads == 0 || (k && k_out)) && (pairs == 0 || (positions && inv_freq)),
                   "%s: null pointer", who);
  const int64_t es = dtype == DT_F32 ? 4 : 2;
  bool vec = ((uintptr_t)q | (uintptr_t)k | (uintptr_t)q_out | (uintptr_t)k_out) % 16 == 0;
  for (int64_t s : {q_st, q_sh, k_st, k_sh, qo_st, qo_sh, ko_st, ko_sh}) vec = vec && (s * es) % 16 == 0;
  CORTEX_CHECK_ARG(vec, "%s: rows must be 16-byte aligned", who);
  CORTEX_CHECK_ARG(((uintptr_t)q_gain | (uintptr_t)k_gain) % 16 == 0, "%s: gains must be 16-byte aligned", who);
  RopeArgs a = {};
  a.side[0] = {q, q_st, q_sh, q_out, qo_st, qo_sh, q_gain, (int)heads, 1, 0};
  a.side[1] = {k, k_st, k_sh, k_out, ko_st, ko_sh, k_gain, (int)kv_heads, 1, 0};
  a.T = T;
  a.dim = (int)dim;
  a.pairs = (int)pairs;
  a.lanes = 1;
  while (a.lanes * 16 < dim) a.lanes <<= 1;
  a.positions = positions;
  a.p_st = p_st, a.p_sa = p_sa, a.n_axes = n_axes;
  a.inv_freq = inv_freq;
  a.axes = axes;
  a.eps = eps;
  a.gain_f32 = gain_dtype == DT_F32;
  a.err = err;
  int64_t grid = 0;
  for (RopeSide& o : a.side) {
    if (o.heads == 0) continue;
    // as many tokens a workgroup as its threads have loads in flight for, while every CU gets four workgroups
    int64_t tokens = 256 * 4 / ((int64_t)o.heads * a.lanes), spread = T / (2 * cu_count());
    tokens = tokens < spread ? tokens : spread;
    if (pairs && tokens > RP_ANGLES / pairs) tokens = RP_ANGLES / pairs;
    o.tokens = (int)(tokens < 1 ? 1 : tokens);
    grid += o.grid = (unsigned)cdiv(T, o.tokens);
  }
  CORTEX_CHECK_ARG(grid <= 0xffffffffLL / 256, "%s: %lld tokens are too many for one call", who, (long long)T);
  return dtype == DT_F32 ? launch<float>(a, norm, interleaved, stream) : launch<bf16>(a, norm, interleaved, stream);
}
