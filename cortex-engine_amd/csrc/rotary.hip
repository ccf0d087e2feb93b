// Norms of queries and keys per head and their rotation by position, in one pass.
//
//   x' = x / sqrt(mean_d x_d^2 + eps) * gain          (a row: one head of one token; or x' = x)
//   angle of pair p = position[axis(p)] * inv_freq[p]
//   y_i = x'_i cos - x'_j sin,  y_j = x'_j cos + x'_i sin
//
// with (i, j) = (p, p + pairs) or (2 p, 2 p + 1); dims past the pairs are only normed.  Everything between the load of a
// row and its store is in fp32, rounded once.
//
// The angle is the product in 64 bits: at position 2^20 a product in 32 is off by up to 0.06 rad.  It is reduced to
// [-pi/4, pi/4] and a quadrant in 64 bits, so that sine and cosine are those of a small fp32 argument.  The angles of a token are
// the same for all its heads: a workgroup computes them once, into LDS.
#include <hip/hip_runtime.h>

#include "common.h"
#include "cortex_hip.h"

namespace cortex {
namespace {

constexpr int RP_ERR = 8;         // bit of *err: an axis outside the positions
constexpr int RP_AHEAD = 4;       // eights of values in flight a thread
constexpr int RP_ANGLES = 2048;   // (token, pair) angles of a workgroup, at most
constexpr int RP_MAX_DIM = 256;

struct RopeArgs {
  int64_t T;
  int heads, all;  // query heads, and with the key heads
  int dim, pairs, lpr, tokens;
  const void* x[2];
  int64_t st[2], sh[2];
  void* y[2];
  int64_t yt[2], yh[2];
  const int64_t* positions;
  int64_t p_st, p_sa, n_axes;
  const float* inv_freq;
  const int32_t* axes;
  float eps;
  const void* gain[2];
  int gain_f32;
  int32_t* err;
};

template <class X>
__device__ __forceinline__ void load8(const X* p, float (&f)[8]) {
  if constexpr (sizeof(X) == 4) {
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(p + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) f[i + e] = v[e];
    }
  } else {
    const bf16x8 v = *reinterpret_cast<const bf16x8*>(p);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = (float)v[e];
  }
}
__device__ __forceinline__ void save8(float* p, const float (&f)[8]) {
  reinterpret_cast<f32x4*>(p)[0] = f32x4{f[0], f[1], f[2], f[3]};
  reinterpret_cast<f32x4*>(p)[1] = f32x4{f[4], f[5], f[6], f[7]};
}
__device__ __forceinline__ void save8(bf16* p, const float (&f)[8]) {
  bf16x8 v;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (bf16)f[e];
  *reinterpret_cast<bf16x8*>(p) = v;
}

// Cosine and sine of a 64-bit angle, each rounded from an fp32 argument of at most pi/4.
__device__ __forceinline__ float2 turn(double angle) {
  const double n = rint(angle * 0.63661977236758134308);  // quarter turns
  // pi/2 as the double next to it and the rest: n of each, the first product exact in the fma
  const double r = fma(-n, 6.123233995736766036e-17, fma(-n, 1.5707963267948965580, angle));
  float s, c;
  sincosf((float)r, &s, &c);
  const int quadrant = (int)((int64_t)n & 3);
  const float a = (quadrant & 1) ? s : c, b = (quadrant & 1) ? c : s;
  return make_float2((quadrant == 1 || quadrant == 2) ? -a : a, (quadrant & 2) ? -b : b);
}

// A workgroup takes `tokens` tokens, a thread eight values of a (token, head) row, `lpr` lanes a row.
template <class X, bool NORM, bool INTER>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(RopeArgs a) {
  __shared__ __attribute__((aligned(16))) float2 angles[RP_ANGLES];  // cosine, sine
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t t0 = (int64_t)blockIdx.x * a.tokens;
  const int count = (int)min((int64_t)a.tokens, a.T - t0);
  const int per = a.all * a.lpr, items = count * per;
  const int d = (tid & (a.lpr - 1)) * 8;  // (256 is a multiple of lpr)
  const bool in_row = d < a.dim, turned = d < 2 * a.pairs;
  const bool second = !INTER && d >= a.pairs;  // the half whose partners are `pairs` below
  const int pair = INTER ? d >> 1 : second ? d - a.pairs : d;
  const int partner = second ? lane - (a.pairs >> 3) : lane + (a.pairs >> 3);
  bool ready = false;
  float gain[2][8];
  for (int i0 = 0; i0 < items; i0 += 256 * RP_AHEAD) {
    float x[RP_AHEAD][8];
#pragma unroll
    for (int s = 0; s < RP_AHEAD; ++s) {
      const int i = i0 + 256 * s + tid;
      if (i < items && in_row) {
        const int k = i / per, r = (i - k * per) / a.lpr;
        const int which = r >= a.heads;
        load8(reinterpret_cast<const X*>(a.x[which]) + (t0 + k) * a.st[which] + (r - (which ? a.heads : 0)) * a.sh[which] + d,
              x[s]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[s][e] = 0.0f;
      }
    }
    if (!ready) {  // beside the first rows: gains and angles
      if constexpr (NORM) {
#pragma unroll
        for (int w = 0; w < 2; ++w) {
#pragma unroll
          for (int e = 0; e < 8; ++e) gain[w][e] = 1.0f;
          if (a.gain[w] && in_row) {
            if (a.gain_f32)
              load8(reinterpret_cast<const float*>(a.gain[w]) + d, gain[w]);
            else
              load8(reinterpret_cast<const bf16*>(a.gain[w]) + d, gain[w]);
          }
        }
      }
      for (int i = tid; i < count * a.pairs; i += 256) {
        const int k = i / a.pairs, p = i - k * a.pairs;
        const int axis = a.axes ? a.axes[p] : 0;
        const bool there = (uint64_t)(int64_t)axis < (uint64_t)a.n_axes;
        if (!there && a.err) atomicOr(a.err, RP_ERR);
        const int64_t at = there ? a.positions[(t0 + k) * a.p_st + axis * a.p_sa] : 0;
        angles[i] = turn((double)at * (double)a.inv_freq[p]);
      }
      __syncthreads();
      ready = true;
    }
#pragma unroll
    for (int s = 0; s < RP_AHEAD; ++s) {
      if (i0 + 256 * s >= items) break;
      const int i = i0 + 256 * s + tid;
      const int k = min(i / per, count - 1), r = (i - k * per) / a.lpr;
      const int which = r >= a.heads;
      float(&f)[8] = x[s];
      if constexpr (NORM) {
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += f[e] * f[e];
        for (int o = 1; o < a.lpr; o <<= 1) sum += __shfl_xor(sum, o, 64);
        const float inv = 1.0f / sqrtf(sum / (float)a.dim + a.eps);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = f[e] * inv * (which ? gain[1][e] : gain[0][e]);
      }
      const float2* at = angles + k * a.pairs + (turned ? pair : 0);
      if constexpr (INTER) {
        if (turned) {
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const float2 t = at[e >> 1];
            const float u = f[e], v = f[e + 1];
            f[e] = u * t.x - v * t.y;
            f[e + 1] = v * t.x + u * t.y;
          }
        }
      } else {
        float other[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) other[e] = __shfl(f[e], partner, 64);
        if (turned) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float2 t = at[e];
            f[e] = f[e] * t.x + (second ? other[e] : -other[e]) * t.y;
          }
        }
      }
      if (i < items && in_row)
        save8(reinterpret_cast<X*>(a.y[which]) + (t0 + k) * a.yt[which] + (r - (which ? a.heads : 0)) * a.yh[which] + d, f);
    }
  }
}

template <class X>
int launch(const RopeArgs& a, bool norm, bool interleaved, unsigned grid, hipStream_t stream) {
  const dim3 block(256);
  if (norm && interleaved)
    hipLaunchKernelGGL((qk_norm_rope_kernel<X, true, true>), dim3(grid), block, 0, stream, a);
  else if (norm)
    hipLaunchKernelGGL((qk_norm_rope_kernel<X, true, false>), dim3(grid), block, 0, stream, a);
  else if (interleaved)
    hipLaunchKernelGGL((qk_norm_rope_kernel<X, false, true>), dim3(grid), block, 0, stream, a);
  else
    hipLaunchKernelGGL((qk_norm_rope_kernel<X, false, false>), dim3(grid), block, 0, stream, a);
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
  a.T = T;
  a.heads = (int)heads;
  a.all = (int)(heads + kv_heads);
  a.dim = (int)dim;
  a.pairs = (int)pairs;
  a.lpr = 1;
  while (a.lpr * 8 < dim) a.lpr <<= 1;
  a.x[0] = q, a.x[1] = k;
  a.st[0] = q_st, a.st[1] = k_st, a.sh[0] = q_sh, a.sh[1] = k_sh;
  a.y[0] = q_out, a.y[1] = k_out;
  a.yt[0] = qo_st, a.yt[1] = ko_st, a.yh[0] = qo_sh, a.yh[1] = ko_sh;
  a.positions = positions;
  a.p_st = p_st, a.p_sa = p_sa, a.n_axes = n_axes;
  a.inv_freq = inv_freq;
  a.axes = axes;
  a.eps = eps;
  a.gain[0] = q_gain, a.gain[1] = k_gain;
  a.gain_f32 = gain_dtype == DT_F32;
  a.err = err;
  // as many tokens a workgroup as its threads have loads in flight for, while every CU gets eight workgroups
  int64_t tokens = 256 * RP_AHEAD / ((int64_t)a.all * a.lpr), spread = T / (8 * cu_count());
  tokens = tokens < spread ? tokens : spread;
  if (pairs && tokens > RP_ANGLES / pairs) tokens = RP_ANGLES / pairs;
  a.tokens = (int)(tokens < 1 ? 1 : tokens);
  const int64_t grid = cdiv(T, a.tokens);
  CORTEX_CHECK_ARG(grid <= 0xffffffffLL / 256, "%s: %lld tokens are too many for one call", who, (long long)T);
  return dtype == DT_F32 ? launch<float>(a, norm, interleaved, (unsigned)grid, stream)
                         : launch<bf16>(a, norm, interleaved, (unsigned)grid, stream);
}
