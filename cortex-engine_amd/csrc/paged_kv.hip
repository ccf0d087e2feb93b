// Paged K/V cache: append of new tokens' rows, and eviction by accumulated attention weight.
//
// Eviction keeps a fixed number of slots per key/value head and leaves them where they are: only the kept slots
// past the budget move, each into a slot below it that is given up.  Attention does not depend on the order of
// its keys (their positions are in the keys, and beside them in `position`), so nothing else has to move; a
// compaction that kept the order would move most of the rows.  Sources (at or past the budget) and destinations
// (below it) are disjoint: every row moves independently of the others.
#include <hip/hip_runtime.h>

#include "paged_kv.h"

namespace cortex {

int kv_check(const char* who, const cortex_kv_pages* p, int64_t B, const int32_t* table, int64_t ld_table,
             int64_t max_pages, KvPages* out) {
  CORTEX_CHECK_ARG(p, "%s: null pages", who);
  CORTEX_CHECK_ARG(B >= 0 && max_pages >= 0, "%s: negative shape", who);
  CORTEX_CHECK_ARG(p->dtype == DT_F32 || p->dtype == DT_BF16 || p->dtype == DT_I8,
                   "%s: pages of dtype %lld (f32, bf16 or int8)", who, (long long)p->dtype);
  CORTEX_CHECK_ARG(p->num_pages >= 1 && p->num_pages <= 0x7fffffffLL && p->kv_heads >= 1 && p->kv_heads <= 65535,
                   "%s: page count %lld or head count %lld outside its range", who, (long long)p->num_pages,
                   (long long)p->kv_heads);
  const int64_t ps = p->page_size;
  CORTEX_CHECK_ARG(ps >= 8 && ps <= 65536 && (ps & (ps - 1)) == 0,
                   "%s: page size %lld is not a power of two from 8 to 65536", who, (long long)ps);
  CORTEX_CHECK_ARG(p->head_dim >= 16 && p->head_dim <= 128 && p->head_dim % 16 == 0,
                   "%s: head dim %lld is not a multiple of 16 up to 128", who, (long long)p->head_dim);
  CORTEX_CHECK_ARG(p->k && p->v, "%s: null k or v pages", who);
  CORTEX_CHECK_ARG((p->dtype == DT_I8) == (p->k_scale != nullptr) && (p->k_scale != nullptr) == (p->v_scale != nullptr),
                   "%s: int8 pages need k_scale and v_scale, float pages take none", who);
  const int64_t es = p->dtype == DT_F32 ? 4 : p->dtype == DT_BF16 ? 2 : 1;
  bool vec = ((uintptr_t)p->k | (uintptr_t)p->v) % 16 == 0;
  for (int64_t s : {p->k_page, p->k_head, p->k_slot, p->v_page, p->v_head, p->v_slot})
    vec = vec && s >= 0 && (s * es) % 16 == 0;
  CORTEX_CHECK_ARG(vec, "%s: page rows must be 16-byte aligned, with strides >= 0", who);
  CORTEX_CHECK_ARG(p->k_slot >= p->head_dim && p->v_slot >= p->head_dim, "%s: rows of a page overlap", who);
  CORTEX_CHECK_ARG(B == 0 || max_pages == 0 || table, "%s: null block table", who);
  CORTEX_CHECK_ARG(B <= 1 || ld_table >= max_pages, "%s: rows of the block table overlap", who);
  CORTEX_CHECK_ARG(max_pages <= (1ll << 30) / ps, "%s: %lld pages of %lld slots are more than 2^30 slots", who,
                   (long long)max_pages, (long long)ps);
  *out = KvPages{p->k,       p->v,       p->k_scale, p->v_scale, p->weight,  p->position, p->k_page,
                 p->k_head,  p->k_slot,  p->v_page,  p->v_head,  p->v_slot,  table,       ld_table,
                 (int32_t)p->num_pages, (int32_t)p->kv_heads, (int32_t)p->head_dim,
                 __builtin_ctzll((unsigned long long)ps), max_pages * ps};
  return OK;
}

namespace {

// ---------------------------------------------------------------------------- append

struct AppendArgs {
  KvPages p;
  int64_t B, T;
  const void* k;
  int64_t k_st, k_sh;
  const void* v;
  int64_t v_st, v_sh;
  const int64_t* offsets;  // null: token t is sequence t's
  const int64_t* lengths;
  const int64_t* positions;
  int64_t* new_lengths;
  int32_t* err;
};

// Eight values of a row a lane.
__device__ __forceinline__ void load8(float (&f)[8], const float* p) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
}
__device__ __forceinline__ void load8(float (&f)[8], const bf16* p) {
  const bf16x8 a = *reinterpret_cast<const bf16x8*>(p);
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = (float)a[j];
}
__device__ __forceinline__ void store8(float* p, const float (&f)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}
__device__ __forceinline__ void store8(bf16* p, const float (&f)[8]) {
  bf16x8 a;
#pragma unroll
  for (int j = 0; j < 8; ++j) a[j] = (bf16)f[j];
  *reinterpret_cast<bf16x8*>(p) = a;
}

// The sequence of token t: the number of offsets[1 ..] that are <= t.
__device__ int64_t sequence_of(const int64_t* offsets, int64_t B, int64_t t) {
  int64_t lo = 0, hi = B;  // offsets[lo] <= t < offsets[hi + 1] for ascending offsets
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (offsets[mid + 1] <= t)
      lo = mid + 1;
    else
      hi = mid;
  }
  return lo;
}

// One workgroup a token; LPR lanes a (key or value, head) row.
template <class X, class P>
__global__ __launch_bounds__(256) void kv_append_kernel(AppendArgs a, int lpr) {
  const int tid = threadIdx.x;
  const KvPages& p = a.p;
  const int64_t t = blockIdx.x;
  int64_t b = t, first = t;
  if (a.offsets) {
    b = sequence_of(a.offsets, a.B, t);
    if (b >= a.B) return;  // behind the last sequence
    first = a.offsets[b];
    if (t < first) return;  // before the first
  }
  bool ok = true;
  const int64_t len = p.length_of(a.lengths, b, p.max_slots, &ok);
  const int64_t slot = len + (t - first);
  const int page = p.page_of(b, slot);
  if (tid == 0 && (!ok || page < 0)) kv_flag(a.err);
  // lengths may be new_lengths: with a token a sequence this workgroup is the only one that reads lengths[b]
  if (!a.offsets) {
    __syncthreads();
    if (tid == 0 && a.new_lengths) a.new_lengths[b] = page < 0 && slot >= p.max_slots ? len : len + 1;
  }
  if (page < 0) return;
  const int row = p.row_of(slot);
  const int d = (tid % lpr) * 8;
  const int rows = 2 * p.kv_heads, step = 256 / lpr;
  for (int r0 = 0; r0 < rows; r0 += step) {  // whole groups of lanes: the shuffles below take all of them
    const int r = r0 + tid / lpr;
    const bool in = r < rows && d < p.head_dim;
    const int h = r >> 1;
    const bool is_v = r & 1;
    float f[8] = {};
    if (in) load8(f, reinterpret_cast<const X*>(is_v ? a.v : a.k) + t * (is_v ? a.v_st : a.k_st) + h * (is_v ? a.v_sh : a.k_sh) + d);
    const int64_t at = is_v ? page * p.v_page + h * p.v_head + row * p.v_slot : page * p.k_page + h * p.k_head + row * p.k_slot;
    P* to = reinterpret_cast<P*>(is_v ? p.v : p.k) + at + d;
    if constexpr (sizeof(P) == 1) {
      uint32_t most = 0;  // the largest |x|; an infinity or a NaN is above every number's bits
#pragma unroll
      for (int j = 0; j < 8; ++j) most = max(most, __float_as_uint(f[j]) & 0x7fffffffu);
      for (int o = 1; o < lpr; o <<= 1) most = max(most, (uint32_t)__shfl_xor((int)most, o, 64));
      const bool finite = most < 0x7f800000u;
      const float s = finite ? fmaxf(__uint_as_float(most), 1e-8f) / 127.0f : __uint_as_float(0x7fc00000u);
      if (in) {
        union {
          int8_t c[8];
          uint2 u;
        } q;
#pragma unroll
        for (int j = 0; j < 8; ++j) q.c[j] = finite ? (int8_t)(int)fminf(fmaxf(rintf(f[j] / s), -127.0f), 127.0f) : 0;
        *reinterpret_cast<uint2*>(to) = q.u;
        if (d == 0) (is_v ? p.v_scale : p.k_scale)[p.scalar_at(page, h, row)] = s;
      }
    } else if (in) {
      store8(to, f);
    }
    if (in && d == 0 && !is_v) {
      const int64_t i = p.scalar_at(page, h, row);
      if (p.weight) p.weight[i] = 0.0f;
      if (p.position) p.position[i] = (int32_t)(a.positions ? a.positions[t] : slot);
    }
  }
}

// The lengths after ragged appends, in a launch of its own: lengths may be new_lengths.
__global__ void kv_lengths_kernel(AppendArgs a) {
  const int64_t b = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (b >= a.B) return;
  bool ok = true;
  const int64_t len = a.p.length_of(a.lengths, b, a.p.max_slots, &ok);
  const int64_t lo = min(max(a.offsets[b], (int64_t)0), a.T), hi = min(max(a.offsets[b + 1], lo), a.T);
  a.new_lengths[b] = min(len + (hi - lo), a.p.max_slots);
}

// ---------------------------------------------------------------------------- eviction

struct PlanArgs {
  KvPages p;
  const int64_t* lengths;
  int64_t max_length, budget, recent, cap;
  int32_t* dst;
  int32_t* src;
  int32_t* counts;
  int64_t* new_lengths;
  int32_t* err;
};

constexpr int EP_THREADS = 1024;
constexpr int EP_WAVES = EP_THREADS / 64;
// Ranks held in LDS (16 or 128 KiB); a sequence with more slots computes them again where they are read.
constexpr int EP_FEW = 4096, EP_MANY = 32768;

// The rank of a slot as an unsigned number: protected slots first, then NaN, then by weight; a slot without a page
// below all of them.
__device__ __forceinline__ uint32_t rank_of(const PlanArgs& a, int64_t b, int h, int64_t j, int64_t above) {
  const int page = a.p.page_of(b, j);
  if (page < 0) return 0;
  const int64_t i = a.p.scalar_at(page, h, a.p.row_of(j));
  if ((int64_t)a.p.position[i] > above) return 0xffffffffu;
  const float w = a.p.weight[i];
  if (w != w) return 0xfffffffeu;
  const uint32_t u = __float_as_uint(w + 0.0f);  // -0 and 0 are equal
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

__device__ __forceinline__ int wave_scan(int v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(v, o, 64);
    if (lane >= o) v += u;
  }
  return v;
}

// Sum of v over the threads before this one, and over all of them (in *total).
__device__ int block_scan(int v, int* part, int tid, int* total) {
  const int lane = tid & 63, wid = tid >> 6;
  const int inc = wave_scan(v, lane);
  __syncthreads();  // (part may still be read from the call before)
  if (lane == 63) part[wid] = inc;
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < EP_WAVES; ++w) {
    const int s = part[w];
    if (w < wid) before += s;
    all += s;
  }
  *total = all;
  return before + inc - v;
}

// One workgroup a (sequence, key head): the rank of every slot, the budget-th largest by a radix selection over
// four bytes, then holes and movers in slot order by prefix sums.
template <int KEYS>
__global__ __launch_bounds__(EP_THREADS) void kv_evict_plan_kernel(PlanArgs a) {
  __shared__ uint32_t keys[KEYS];
  __shared__ int hist[EP_WAVES][256];
  __shared__ int part[EP_WAVES];
  __shared__ int picked[3];
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int H = a.p.kv_heads;
  const int64_t b = blockIdx.x / H;
  const int h = blockIdx.x - (int)b * H;
  int32_t* dst = a.dst + (int64_t)blockIdx.x * a.cap;
  int32_t* src = a.src + (int64_t)blockIdx.x * a.cap;
  bool ok = true;
  const int64_t n = a.p.length_of(a.lengths, b, a.max_length, &ok);
  if (!ok && tid == 0) kv_flag(a.err);
  if (h == 0 && tid == 0) a.new_lengths[b] = min(n, a.budget);
  int moved = 0;
  if (n > a.budget && a.budget > 0) {
    // the newest position
    int newest = INT32_MIN;
    bool lost = false;
    for (int64_t j = tid; j < n; j += EP_THREADS) {
      const int page = a.p.page_of(b, j);
      if (page < 0)
        lost = true;
      else
        newest = max(newest, a.p.position[a.p.scalar_at(page, h, a.p.row_of(j))]);
    }
    if (lost) kv_flag(a.err);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) newest = max(newest, __shfl_xor(newest, o, 64));
    if (lane == 0) part[wid] = newest;
    __syncthreads();
    for (int w = 0; w < EP_WAVES; ++w) newest = max(newest, part[w]);
    const int64_t above = (int64_t)newest - a.recent;
    const bool held = n <= KEYS;
    if (held)
      for (int64_t j = tid; j < n; j += EP_THREADS) keys[j] = rank_of(a, b, h, j, above);
    auto key = [&](int64_t j) { return held ? keys[j] : rank_of(a, b, h, j, above); };

    // the budget-th largest rank, a byte a round: `kept` of the slots with the rank found so far are kept
    uint32_t found = 0;
    int kept = (int)a.budget;
    for (int shift = 24; shift >= 0; shift -= 8) {
      __syncthreads();
      for (int i = tid; i < EP_WAVES * 256; i += EP_THREADS) hist[0][i] = 0;
      __syncthreads();
      for (int64_t j = tid; j < n; j += EP_THREADS) {
        const uint32_t x = key(j);
        if (shift == 24 || (x >> (shift + 8)) == (found >> (shift + 8))) atomicAdd(&hist[wid][(x >> shift) & 255], 1);
      }
      __syncthreads();
      if (wid == 0) {  // lane l has the bins 255 - 4 l .. 252 - 4 l, the largest ranks first
        int c[4], s = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          c[i] = 0;
          for (int w = 0; w < EP_WAVES; ++w) c[i] += hist[w][255 - 4 * lane - i];
          s += c[i];
        }
        int before = wave_scan(s, lane) - s;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (before < kept && before + c[i] >= kept) {  // (one bin of one lane)
            picked[0] = 255 - 4 * lane - i;
            picked[1] = before;
          }
          before += c[i];
        }
      }
      __syncthreads();
      found |= (uint32_t)picked[0] << shift;
      kept -= picked[1];
    }

    // thread i takes the slots [i R, (i + 1) R), R odd: its LDS reads are free of bank conflicts
    const int64_t R = cdiv(n, EP_THREADS) | 1;
    const int64_t j0 = min((int64_t)tid * R, n), j1 = min(j0 + R, n);
    int ties = 0, all;
    for (int64_t j = j0; j < j1; ++j) ties += key(j) == found;
    ties = block_scan(ties, part, tid, &all);  // (now: the ties before this thread's slots)
    int holes = 0, movers = 0, tie = ties;
    for (int64_t j = j0; j < j1; ++j) {
      const uint32_t x = key(j);
      const bool keep = x > found || (x == found && tie++ < kept);
      holes += !keep && j < a.budget;
      movers += keep && j >= a.budget;
    }
    int hole = block_scan(holes, part, tid, &all);
    int mover = block_scan(movers, part, tid, &moved);
    tie = ties;
    for (int64_t j = j0; j < j1; ++j) {
      const uint32_t x = key(j);
      const bool keep = x > found || (x == found && tie++ < kept);
      if (!keep && j < a.budget) dst[hole++] = (int32_t)j;
      if (keep && j >= a.budget) src[mover++] = (int32_t)j;
    }
  }
  if (tid == 0) a.counts[blockIdx.x] = moved;
  for (int64_t i = moved + tid; i < a.cap; i += EP_THREADS) dst[i] = src[i] = -1;
}

struct ApplyArgs {
  KvPages p;
  const int32_t* dst;
  const int32_t* src;
  int64_t cap;
  const int32_t* counts;
  int32_t* err;
  int chunks;     // workgroups a (sequence, head)
  int lanes;      // lanes a row (a power of two), 16 bytes each
  int row_bytes;
};

constexpr int EA_ROWS = 4;  // rows of a group of lanes

__global__ __launch_bounds__(256) void kv_evict_apply_kernel(ApplyArgs a, int es) {
  const int tid = threadIdx.x;
  const int bh = blockIdx.x / a.chunks, chunk = blockIdx.x - bh * a.chunks;
  const int64_t b = bh / a.p.kv_heads;
  const int h = bh - (int)b * a.p.kv_heads;
  const int groups = 256 / a.lanes, group = tid / a.lanes, c = (tid % a.lanes) * 16;
  const int64_t n = min((int64_t)a.counts[bh], a.cap);
#pragma unroll
  for (int r = 0; r < EA_ROWS; ++r) {
    const int64_t i = ((int64_t)chunk * EA_ROWS + r) * groups + group;
    if (i >= n) return;
    const int64_t to = a.dst[(int64_t)bh * a.cap + i], from = a.src[(int64_t)bh * a.cap + i];
    const int tp = a.p.page_of(b, to), fp = a.p.page_of(b, from);
    if (tp < 0 || fp < 0) {
      if (c == 0) kv_flag(a.err);
      continue;
    }
    const int tr = a.p.row_of(to), fr = a.p.row_of(from);
    if (c < a.row_bytes) {
      char* k = reinterpret_cast<char*>(a.p.k) + h * a.p.k_head * es + c;
      char* v = reinterpret_cast<char*>(a.p.v) + h * a.p.v_head * es + c;
      const uint4 x = *reinterpret_cast<const uint4*>(k + (fp * a.p.k_page + fr * a.p.k_slot) * es);
      const uint4 y = *reinterpret_cast<const uint4*>(v + (fp * a.p.v_page + fr * a.p.v_slot) * es);
      *reinterpret_cast<uint4*>(k + (tp * a.p.k_page + tr * a.p.k_slot) * es) = x;
      *reinterpret_cast<uint4*>(v + (tp * a.p.v_page + tr * a.p.v_slot) * es) = y;
    }
    if (c == 0) {
      const int64_t t = a.p.scalar_at(tp, h, tr), f = a.p.scalar_at(fp, h, fr);
      if (a.p.k_scale) a.p.k_scale[t] = a.p.k_scale[f], a.p.v_scale[t] = a.p.v_scale[f];
      if (a.p.weight) a.p.weight[t] = a.p.weight[f];
      if (a.p.position) a.p.position[t] = a.p.position[f];
    }
  }
}

int pow2_lanes(int64_t n) {
  int l = 1;
  while (l < n) l <<= 1;
  return l;
}

template <class X>
int launch_append(const AppendArgs& a, int dtype, hipStream_t stream) {
  const int lpr = pow2_lanes(a.p.head_dim / 8);
  const dim3 grid((unsigned)a.T), block(256);
  if (a.T > 0) {
    if (dtype == DT_F32)
      hipLaunchKernelGGL((kv_append_kernel<X, float>), grid, block, 0, stream, a, lpr);
    else if (dtype == DT_BF16)
      hipLaunchKernelGGL((kv_append_kernel<X, bf16>), grid, block, 0, stream, a, lpr);
    else
      hipLaunchKernelGGL((kv_append_kernel<X, int8_t>), grid, block, 0, stream, a, lpr);
    CORTEX_CHECK_LAUNCH("kv_append_kernel");
  }
  if (a.offsets && a.new_lengths) {
    hipLaunchKernelGGL(kv_lengths_kernel, dim3((unsigned)cdiv(a.B, 256)), block, 0, stream, a);
    CORTEX_CHECK_LAUNCH("kv_lengths_kernel");
  }
  return OK;
}

}  // namespace

}  // namespace cortex

using namespace cortex;

extern "C" int cortex_kv_append(const cortex_kv_pages* pages, int64_t B, int64_t n_tokens, int x_dtype, const void* k,
                                int64_t k_st, int64_t k_sh, const void* v, int64_t v_st, int64_t v_sh,
                                const int32_t* block_table, int64_t ld_table, int64_t max_pages,
                                const int64_t* offsets, const int64_t* lengths, const int64_t* positions,
                                int64_t* new_lengths, int32_t* err, hipStream_t stream) {
  const char* who = "cortex_kv_append";
  AppendArgs a = {};
  if (int rc = kv_check(who, pages, B, block_table, ld_table, max_pages, &a.p)) return rc;
  CORTEX_CHECK_ARG(n_tokens >= 0 && n_tokens <= 0x7fffffffLL, "%s: %lld tokens", who, (long long)n_tokens);
  CORTEX_CHECK_ARG(offsets || n_tokens == B, "%s: without offsets there is one token a sequence", who);
  CORTEX_CHECK_ARG(x_dtype == DT_F32 || x_dtype == DT_BF16, "%s: rows of dtype %d (f32 or bf16)", who, x_dtype);
  if (B == 0) return OK;
  CORTEX_CHECK_ARG(lengths, "%s: null lengths", who);
  if (n_tokens > 0) {
    CORTEX_CHECK_ARG(k && v, "%s: null k or v", who);
    const int64_t es = x_dtype == DT_F32 ? 4 : 2;
    bool vec = ((uintptr_t)k | (uintptr_t)v) % 16 == 0;
    for (int64_t s : {k_st, k_sh, v_st, v_sh}) vec = vec && (s * es) % 16 == 0;
    CORTEX_CHECK_ARG(vec, "%s: rows must be 16-byte aligned", who);
  }
  a.B = B;
  a.T = n_tokens;
  a.k = k;
  a.k_st = k_st;
  a.k_sh = k_sh;
  a.v = v;
  a.v_st = v_st;
  a.v_sh = v_sh;
  a.offsets = offsets;
  a.lengths = lengths;
  a.positions = positions;
  a.new_lengths = new_lengths;
  a.err = err;
  return x_dtype == DT_F32 ? launch_append<float>(a, (int)pages->dtype, stream)
                           : launch_append<bf16>(a, (int)pages->dtype, stream);
}

extern "C" int cortex_kv_evict_plan(const cortex_kv_pages* pages, int64_t B, const int32_t* block_table,
                                    int64_t ld_table, int64_t max_pages, const int64_t* lengths, int64_t max_length,
                                    int64_t budget, int64_t recent, int32_t* dst, int32_t* src, int32_t* counts,
                                    int64_t* new_lengths, int32_t* err, hipStream_t stream) {
  const char* who = "cortex_kv_evict_plan";
  PlanArgs a = {};
  if (int rc = kv_check(who, pages, B, block_table, ld_table, max_pages, &a.p)) return rc;
  CORTEX_CHECK_ARG(pages->weight && pages->position, "%s: the pages need weight and position", who);
  CORTEX_CHECK_ARG(budget >= 0 && recent >= 0, "%s: negative budget or recent", who);
  CORTEX_CHECK_ARG(recent <= budget, "%s: recent (%lld) exceeds the budget (%lld)", who, (long long)recent,
                   (long long)budget);
  if (B == 0) return OK;
  a.max_length = max_length < 0 || max_length > a.p.max_slots ? a.p.max_slots : max_length;
  a.budget = budget;
  a.recent = recent;
  a.cap = a.max_length > budget ? (a.max_length - budget < budget ? a.max_length - budget : budget) : 0;
  CORTEX_CHECK_ARG(lengths && counts && new_lengths && ((dst && src) || a.cap == 0), "%s: null pointer", who);
  CORTEX_CHECK_ARG(new_lengths != lengths, "%s: new_lengths may not be lengths", who);
  CORTEX_CHECK_ARG(B * pages->kv_heads <= 0x7fffffffLL, "%s: too many heads", who);
  a.lengths = lengths;
  a.dst = dst;
  a.src = src;
  a.counts = counts;
  a.new_lengths = new_lengths;
  a.err = err;
  const dim3 grid((unsigned)(B * pages->kv_heads));
  if (a.max_length <= EP_FEW)
    hipLaunchKernelGGL(kv_evict_plan_kernel<EP_FEW>, grid, dim3(EP_THREADS), 0, stream, a);
  else
    hipLaunchKernelGGL(kv_evict_plan_kernel<EP_MANY>, grid, dim3(EP_THREADS), 0, stream, a);
  CORTEX_CHECK_LAUNCH("kv_evict_plan_kernel");
  return OK;
}

extern "C" int cortex_kv_evict_apply(const cortex_kv_pages* pages, int64_t B, const int32_t* block_table,
                                     int64_t ld_table, int64_t max_pages, const int32_t* dst, const int32_t* src,
                                     int64_t cap, const int32_t* counts, int32_t* err, hipStream_t stream) {
  const char* who = "cortex_kv_evict_apply";
  ApplyArgs a = {};
  if (int rc = kv_check(who, pages, B, block_table, ld_table, max_pages, &a.p)) return rc;
  CORTEX_CHECK_ARG(cap >= 0, "%s: negative cap", who);
  if (B == 0 || cap == 0) return OK;
  CORTEX_CHECK_ARG(dst && src && counts, "%s: null pointer", who);
  const int es = pages->dtype == DT_F32 ? 4 : pages->dtype == DT_BF16 ? 2 : 1;
  a.dst = dst;
  a.src = src;
  a.cap = cap;
  a.counts = counts;
  a.err = err;
  a.row_bytes = (int)pages->head_dim * es;
  a.lanes = pow2_lanes(a.row_bytes / 16);
  const int64_t chunks = cdiv(cap, (256 / a.lanes) * EA_ROWS);
  CORTEX_CHECK_ARG(chunks * B * pages->kv_heads <= 0x7fffffffLL, "%s: too many rows", who);
  a.chunks = (int)chunks;
  hipLaunchKernelGGL(kv_evict_apply_kernel, dim3((unsigned)(chunks * B * pages->kv_heads)), dim3(256), 0, stream, a, es);
  CORTEX_CHECK_LAUNCH("kv_evict_apply_kernel");
  return OK;
}
