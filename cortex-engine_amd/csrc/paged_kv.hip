// Paged K/V cache: append of new tokens' rows, and eviction by accumulated attention weight.
//
// Eviction keeps a fixed number of slots per key/value head and leaves them where they are: only the kept slots
// past the budget move, each into a slot below it that is given up.  Attention does not depend on the order of
// its keys (their positions are in the keys, and beside them in `position`), so nothing else has to move; a
// compaction that kept the order would move most of the rows.  Sources (at or past the budget) and destinations
// (below it) are disjoint: every row moves independently of the others.
#include <hip/hip_runtime.h>

#include <algorithm>

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
  CORTEX_CHECK_ARG(((uintptr_t)p->k_scale | (uintptr_t)p->v_scale | (uintptr_t)p->weight | (uintptr_t)p->position) % 16 == 0,
                   "%s: scales, weight and position must be 16-byte aligned", who);
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

bool kv_rows_meet(const cortex_kv_pages* p) {
  struct Dim {
    int64_t stride, size;
  };
  auto steps_over = [&](Dim a, Dim b, Dim c, Dim d) {  // all rows of the dimensions, one behind the other
    Dim dims[] = {a, b, c, d};
    std::sort(dims, dims + 4, [](const Dim& x, const Dim& y) { return x.stride < y.stride; });
    __int128 extent = p->head_dim;
    for (const Dim& x : dims) {
      if (x.size < 2) continue;
      if (x.stride < extent) return false;
      extent += (__int128)x.stride * (x.size - 1);
    }
    return true;
  };
  const int64_t es = p->dtype == DT_F32 ? 4 : p->dtype == DT_BF16 ? 2 : 1;
  const Dim kd[] = {{p->k_page, p->num_pages}, {p->k_head, p->kv_heads}, {p->k_slot, p->page_size}};
  const Dim vd[] = {{p->v_page, p->num_pages}, {p->v_head, p->kv_heads}, {p->v_slot, p->page_size}};
  const uintptr_t k = (uintptr_t)p->k, v = (uintptr_t)p->v;
  Dim apart = {0, 1};  // v as a second part of k
  if (p->k_page == p->v_page && p->k_head == p->v_head && p->k_slot == p->v_slot)
    apart = {(int64_t)((k < v ? v - k : k - v) / es), 2};
  return k == v || !steps_over(kd[0], kd[1], kd[2], apart) || !steps_over(vd[0], vd[1], vd[2], apart);
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

// Eight values of a row as they are loaded, and as numbers.
template <class X>
struct Eight {
  i32x4 w[sizeof(X) / 2];
  __device__ __forceinline__ void load(const X* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(X) / 2; ++i) w[i] = reinterpret_cast<const i32x4*>(p)[i];
  }
  __device__ __forceinline__ void numbers(float (&f)[8]) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (sizeof(X) == 4)
        f[j] = __int_as_float(w[j >> 2][j & 3]);
      else
        f[j] = __int_as_float((j & 1) ? (w[0][j >> 1] & 0xffff0000) : (w[0][j >> 1] << 16));
    }
  }
};
// (non-temporal: rows are written once, and read much later than most of what is in the caches.  16,800 tokens of 8 heads
// x 128 in bf16: 33.7 us with plain stores, 26.4 with these)
__device__ __forceinline__ void store8(float* p, const float (&f)[8]) {
  __builtin_nontemporal_store(f32x4{f[0], f[1], f[2], f[3]}, reinterpret_cast<f32x4*>(p));
  __builtin_nontemporal_store(f32x4{f[4], f[5], f[6], f[7]}, reinterpret_cast<f32x4*>(p) + 1);
}
__device__ __forceinline__ void store8(bf16* p, const float (&f)[8]) {
  bf16x8 a;
#pragma unroll
  for (int j = 0; j < 8; ++j) a[j] = (bf16)f[j];
  __builtin_nontemporal_store(__builtin_bit_cast(i32x4, a), reinterpret_cast<i32x4*>(p));
}

// The length after n more tokens.  A negative one stays as it is: as 0 the next call would write over the first rows.
__device__ __forceinline__ int64_t length_after(const KvPages& p, int64_t len, int64_t n) {
  return len < 0 ? len : min(min(len, p.max_slots) + n, p.max_slots);
}

// The lengths after a ragged append, by thread `at` of `threads`.
__device__ void lengths_after(const AppendArgs& a, int at, int threads) {
  if (!a.new_lengths) return;
  for (int64_t b = at; b < a.B; b += threads) {
    const int64_t lo = min(max(a.offsets[b], (int64_t)0), a.T), hi = min(max(a.offsets[b + 1], lo), a.T);
    a.new_lengths[b] = length_after(a.p, a.lengths[b], hi - lo);
  }
}

// The sequence of token t: how many of offsets[1 .. B] are <= t.
__device__ int64_t sequence_of(const int64_t* offsets, int64_t B, int64_t t) {
  int64_t lo = 0, hi = B;
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (offsets[mid + 1] <= t)
      lo = mid + 1;
    else
      hi = mid;
  }
  return lo;
}

constexpr int AP_TOKENS = 64;  // tokens of a workgroup, at most
constexpr int AP_AHEAD = 4;    // values in flight, in eights a thread

// A workgroup takes `tokens` tokens, a thread eight values of a (token, key or value, head) row; `lpr` lanes a row.  The
// first threads look up where the tokens go while the others load the rows.  Bound by HBM for many tokens (16,800 of 8
// heads x 128, bf16, 139 MB: 26.4 us, 5.3 TB/s), by the chain of lookups for few.  Int8 pages (105 MB) take 53.9 us, 2.0 TB/s:
// eight divisions a thread, the row's maximum over its lanes and stores of eight bytes; which of them bounds it was not measured.
template <class X, class P>
__global__ __launch_bounds__(256) void kv_append_kernel(AppendArgs a, int lpr, int tokens) {
  __shared__ int at_page[AP_TOKENS], at_row[AP_TOKENS], at_slot[AP_TOKENS];
  const int tid = threadIdx.x;
  const KvPages& p = a.p;
  const int64_t t0 = (int64_t)blockIdx.x * tokens;
  const int count = (int)min((int64_t)tokens, a.T - t0);
  if (a.offsets && blockIdx.x == 0 && a.new_lengths != a.lengths) lengths_after(a, tid, 256);
  if (tid < count) {
    const int64_t t = t0 + tid;
    int64_t b = t, first = t;
    bool mine = true;
    if (a.offsets) {
      b = sequence_of(a.offsets, a.B, t);
      mine = b < a.B && (first = a.offsets[b]) <= t;  // not behind the last sequence, nor before the first
    }
    int page = -1;
    if (mine) {
      const int64_t len = a.lengths[b], slot = min(len, p.max_slots) + (t - first);
      if (len >= 0 && len <= p.max_slots) page = p.page_of(b, slot);  // (a malformed length has no slots)
      if (page < 0) kv_flag(a.err);
      at_row[tid] = p.row_of(slot);
      at_slot[tid] = (int)slot;
      // (may be lengths[b], which this thread alone reads: a token a sequence)
      if (!a.offsets && a.new_lengths) a.new_lengths[b] = length_after(p, len, 1);
    }
    at_page[tid] = page;
  }
  const int rows = 2 * p.kv_heads, per = rows * lpr, items = count * per;
  const int d = (tid & (lpr - 1)) * 8;  // (256 is a multiple of lpr)
  bool looked = false;
  for (int i0 = 0; i0 < items; i0 += 256 * AP_AHEAD) {
    Eight<X> x[AP_AHEAD];
#pragma unroll
    for (int s = 0; s < AP_AHEAD; ++s) {
      const int i = i0 + 256 * s + tid;
      if (i < items && d < p.head_dim) {
        const int k = i / per, r = (i - k * per) / lpr, h = r >> 1;
        x[s].load((r & 1) ? reinterpret_cast<const X*>(a.v) + (t0 + k) * a.v_st + h * a.v_sh + d
                          : reinterpret_cast<const X*>(a.k) + (t0 + k) * a.k_st + h * a.k_sh + d);
      } else {
        x[s] = Eight<X>{};
      }
    }
    if (!looked) __syncthreads();  // the lookups
    looked = true;
#pragma unroll
    for (int s = 0; s < AP_AHEAD; ++s) {
      const int i = i0 + 256 * s + tid;
      if (i0 + 256 * s >= items) break;
      const int k = min(i / per, count - 1), r = (i - k * per) / lpr, h = r >> 1;
      const int page = at_page[k], row = at_row[k];
      const bool in = i < items && d < p.head_dim && page >= 0, is_v = r & 1;
      float f[8];
      x[s].numbers(f);
      const int64_t to = (is_v ? page * p.v_page + h * p.v_head + row * p.v_slot
                               : page * p.k_page + h * p.k_head + row * p.k_slot) + d;
      if constexpr (sizeof(P) == 1) {
        uint32_t most = 0;  // the largest |x|; an infinity or a NaN is above every number's bits
#pragma unroll
        for (int j = 0; j < 8; ++j) most = max(most, __float_as_uint(f[j]) & 0x7fffffffu);
        for (int o = 1; o < lpr; o <<= 1) most = max(most, (uint32_t)__shfl_xor((int)most, o, 64));
        const bool finite = most < 0x7f800000u;
        const float s8 = finite ? fmaxf(__uint_as_float(most), 1e-8f) / 127.0f : __uint_as_float(0x7fc00000u);
        union {
          int8_t c[8];
          uint2 u;
        } q;
#pragma unroll
        for (int j = 0; j < 8; ++j) q.c[j] = finite ? (int8_t)(int)fminf(fmaxf(rintf(f[j] / s8), -127.0f), 127.0f) : 0;
        if (in) {
          *reinterpret_cast<uint2*>(reinterpret_cast<P*>(is_v ? p.v : p.k) + to) = q.u;
          if (d == 0) (is_v ? p.v_scale : p.k_scale)[p.scalar_at(page, h, row)] = s8;
        }
      } else if (in) {
        store8(reinterpret_cast<P*>(is_v ? p.v : p.k) + to, f);
      }
      if (in && d == 0 && !is_v) {
        const int64_t e = p.scalar_at(page, h, row);
        if (p.weight) p.weight[e] = 0.0f;
        if (p.position) p.position[e] = a.positions ? (int32_t)a.positions[t0 + k] : at_slot[k];
      }
    }
  }
}

// Where there are no tokens, or lengths are new_lengths: in a launch of its own, behind the appends that read them.
__global__ void kv_lengths_kernel(AppendArgs a) { lengths_after(a, blockIdx.x * blockDim.x + threadIdx.x, gridDim.x * blockDim.x); }

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

constexpr int EP_COPIES = 8;  // of the histogram, by lane: fewer lanes of a wavefront meet in one counter

// The rank of a slot as an unsigned number: protected slots first, then NaN, then by weight (a slot without a page has 0,
// below all of them).
__device__ __forceinline__ uint32_t rank_of(float w, int position, int64_t above) {
  if ((int64_t)position > above) return 0xffffffffu;
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
template <int WAVES>
__device__ int block_scan(int v, int* part, int tid, int* total) {
  const int lane = tid & 63, wid = tid >> 6;
  const int inc = wave_scan(v, lane);
  __syncthreads();  // (part may still be read from the call before)
  if (lane == 63) part[wid] = inc;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    const int s = part[w];
    if (w < wid) before += s;
    all += s;
  }
  *total = all;
  return before + inc - v;
}

// One workgroup a (sequence, key head): the rank of every slot, the budget-th largest by a radix selection of up to
// four bytes, then holes and movers in slot order by prefix sums.  Bound by the chain of rounds between barriers, not by
// bytes (256 heads of 2000 .. 9001 slots, 11 MB: 22 .. 24 us; 12 up to the ranks and the lists, 9 the selection, 3 the end;
// 512 threads 29, 256 49).  A thread takes Q runs of eight consecutive slots (one page each, four vector loads) and keeps
// their ranks in registers (Q 4 spills 6 of 128); Q 0: as many runs as there are, read again in every pass.
template <int THREADS, int Q>
__global__ __launch_bounds__(THREADS) void kv_evict_plan_kernel(PlanArgs a) {
  constexpr int WAVES = THREADS / 64;
  __shared__ __attribute__((aligned(16))) int hist[2][EP_COPIES][256];  // of this round, and cleared for the next
  __shared__ int part[WAVES];
  __shared__ int picked[3];
  __shared__ uint16_t list[Q ? 8 * Q * THREADS : 1];  // holes, then movers
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int H = a.p.kv_heads;
  const int64_t b = blockIdx.x / H;
  const int h = blockIdx.x - (int)b * H;
  int32_t* dst = a.dst + (int64_t)blockIdx.x * a.cap;
  int32_t* src = a.src + (int64_t)blockIdx.x * a.cap;
  bool ok = true;
  const int n = (int)a.p.length_of(a.lengths, b, a.max_length, &ok);
  if (!ok && tid == 0) kv_flag(a.err);
  if (h == 0 && tid == 0) a.new_lengths[b] = a.lengths[b] < 0 ? a.lengths[b] : min((int64_t)n, a.budget);
  int moved = 0;
  if (n > a.budget && a.budget > 0) {
    const int budget = (int)a.budget;
    const int runs = Q ? Q : (int)cdiv(cdiv(n, 8), THREADS), j0 = tid * runs * 8;
    bool lost = false;
    // run i of this thread: eight weights and positions, or false where there are none
    auto load = [&](int i, float (&w)[8], int (&pos)[8]) {
      const int j = j0 + 8 * i;
      if (j >= n) return false;
      const int page = a.p.page_of(b, j);
      if (page < 0) {
        lost = true;
        return false;
      }
      const int64_t at = a.p.scalar_at(page, h, a.p.row_of(j));
#pragma unroll
      for (int x = 0; x < 8; x += 4) {
        *reinterpret_cast<float4*>(w + x) = *reinterpret_cast<const float4*>(a.p.weight + at + x);
        *reinterpret_cast<int4*>(pos + x) = *reinterpret_cast<const int4*>(a.p.position + at + x);
      }
      return true;
    };
    float w[Q ? Q : 1][8];
    int pos[Q ? Q : 1][8];
    bool there[Q ? Q : 1];
    // the newest position
    int newest = INT32_MIN;
    auto newer = [&](int i, const int (&x)[8]) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (j0 + 8 * i + e < n) newest = max(newest, x[e]);
    };
    if constexpr (Q > 0) {
#pragma unroll
      for (int i = 0; i < Q; ++i) there[i] = load(i, w[i], pos[i]);
#pragma unroll
      for (int i = 0; i < Q; ++i)
        if (there[i]) newer(i, pos[i]);
    } else {
      for (int i = 0; i < runs; ++i)
        if (load(i, w[0], pos[0])) newer(i, pos[0]);
    }
    if (lost) kv_flag(a.err);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) newest = max(newest, __shfl_xor(newest, o, 64));
    if (lane == 0) part[wid] = newest;
    __syncthreads();
#pragma unroll
    for (int x = 0; x < WAVES; ++x) newest = max(newest, part[x]);
    const int64_t above = (int64_t)newest - a.recent;
    uint32_t key[Q ? Q : 1][8];
    auto rank = [&](int i, bool in, const float (&x)[8], const int (&y)[8]) {
#pragma unroll
      for (int e = 0; e < 8; ++e) key[i][e] = in ? rank_of(x[e], y[e], above) : 0u;
    };
    if constexpr (Q > 0) {
#pragma unroll
      for (int i = 0; i < Q; ++i) rank(i, there[i], w[i], pos[i]);
    }
    // f(slot, rank) for this thread's slots, ascending
    auto each = [&](auto f) {
      if constexpr (Q > 0) {
#pragma unroll
        for (int i = 0; i < Q; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (j0 + 8 * i + e < n) f(j0 + 8 * i + e, key[i][e]);
      } else {
        for (int i = 0; i < runs && j0 + 8 * i < n; ++i) {
          rank(0, load(i, w[0], pos[0]), w[0], pos[0]);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (j0 + 8 * i + e < n) f(j0 + 8 * i + e, key[0][e]);
        }
      }
    };

    // the budget-th largest rank, a byte a round; of the slots that share the bytes found so far, `kept` are kept.  Where
    // that is all of them the bytes below do not matter: every slot from `found` up stays
    uint32_t found = 0;
    int kept = budget;
    bool whole = false;
    for (int i = tid; i < EP_COPIES * 256; i += THREADS) hist[0][0][i] = 0;
    __syncthreads();
    for (int shift = 24; shift >= 0 && !whole; shift -= 8) {
      int(*now)[256] = hist[(shift >> 3) & 1 ^ 1], *next = hist[(shift >> 3) & 1][0];
      each([&](int, uint32_t x) {
        if (shift == 24 || (x >> (shift + 8)) == (found >> (shift + 8))) atomicAdd(&now[lane % EP_COPIES][((x >> shift) & 255)], 1);
      });
      __syncthreads();
      if (wid == 0) {  // lane l has the bins 252 - 4 l .. 255 - 4 l
        int4 c = {0, 0, 0, 0};
#pragma unroll
        for (int x = 0; x < EP_COPIES; ++x) {
          const int4 y = *reinterpret_cast<const int4*>(&now[x][252 - 4 * lane]);
          c.x += y.x, c.y += y.y, c.z += y.z, c.w += y.w;
        }
        const int count[4] = {c.w, c.z, c.y, c.x};  // the largest ranks first
        const int sum = (c.x + c.y) + (c.z + c.w);
        int before = wave_scan(sum, lane) - sum;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (before < kept && before + count[i] >= kept)  // (one bin of one lane)
            picked[0] = 255 - 4 * lane - i, picked[1] = before, picked[2] = count[i];
          before += count[i];
        }
      } else {
        for (int i = tid - 64; i < EP_COPIES * 256; i += THREADS - 64) next[i] = 0;
      }
      __syncthreads();
      found |= (uint32_t)picked[0] << shift;
      kept -= picked[1];
      whole = kept == picked[2];
    }

    int tie = 0, all;
    if (!whole) {  // equal ranks: the lower slots stay
      int ties = 0;
      each([&](int, uint32_t x) { ties += x == found; });
      tie = block_scan<WAVES>(ties, part, tid, &all);
    }
    auto stays = [=](uint32_t x, int& t) { return x > found || (x == found && (whole || t++ < kept)); };
    int holes = 0, movers = 0, t = tie;
    each([&](int j, uint32_t x) {
      const bool stay = stays(x, t);
      holes += !stay && j < budget;
      movers += stay && j >= budget;
    });
    int hole, mover;
    if constexpr (Q > 0) {  // both at once: at most half of 32768 slots each
      const int both = block_scan<WAVES>(holes << 16 | movers, part, tid, &all);
      hole = both >> 16, mover = both & 0xffff, moved = all & 0xffff;
    } else {
      hole = block_scan<WAVES>(holes, part, tid, &all);
      mover = block_scan<WAVES>(movers, part, tid, &moved);
    }
    t = tie;
    each([&](int j, uint32_t x) {
      const bool stay = stays(x, t), low = j < budget;
      if (stay != low) {
        if constexpr (Q > 0)
          list[low ? hole : moved + mover] = (uint16_t)j;
        else
          (low ? dst : src)[low ? hole : mover] = j;
      }
      hole += !stay && low;
      mover += stay && !low;
    });
    if constexpr (Q > 0) {  // in whole lines
      __syncthreads();
      for (int i = tid; i < moved; i += THREADS) dst[i] = list[i], src[i] = list[moved + i];
    }
  }
  if (tid == 0) a.counts[blockIdx.x] = moved;
  for (int64_t i = moved + tid; i < a.cap; i += THREADS) dst[i] = src[i] = -1;
}

constexpr int EA_PER_CU = 16;

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

// `lanes` lanes a row, 16 bytes of the key and of the value each; a group of lanes takes a row at a time, with the next
// row's place looked up beside it.  Bound by HBM: rows of 256 bytes read and written at random (32 sequences of 2000 ..
// 9001 slots down to 2048, 8 heads x 128 in bf16, 305 MB: 68.5 us, 4.5 TB/s; four rows a group at once 83 us, one 72
// with plain and with non-temporal stores, in a workgroup for every 16 rows that there may be: 15 us without a move).
__global__ __launch_bounds__(256) void kv_evict_apply_kernel(ApplyArgs a, int es) {
  const int tid = threadIdx.x;
  const int bh = blockIdx.x / a.chunks, chunk = blockIdx.x - bh * a.chunks;
  const int64_t b = bh / a.p.kv_heads;
  const int h = bh - (int)b * a.p.kv_heads;
  const int groups = 256 / a.lanes, c = (tid % a.lanes) * 16;
  const int64_t step = (int64_t)a.chunks * groups, row0 = (int64_t)bh * a.cap;
  int64_t i = (int64_t)chunk * groups + tid / a.lanes;
  if (i >= a.cap) return;
  int to = a.dst[row0 + i], from = a.src[row0 + i];  // (beside the count of moves)
  const int64_t n = min((int64_t)a.counts[bh], a.cap);
  while (i < n) {
    const int tp = a.p.page_of(b, to), fp = a.p.page_of(b, from);
    const int64_t tr = a.p.row_of(to), fr = a.p.row_of(from);
    i += step;
    if (i < n) to = a.dst[row0 + i], from = a.src[row0 + i];
    if (tp < 0 || fp < 0) {
      if (c == 0) kv_flag(a.err);
      continue;
    }
    if (c < a.row_bytes) {
      char* k = reinterpret_cast<char*>(a.p.k) + h * a.p.k_head * es + c;
      char* v = reinterpret_cast<char*>(a.p.v) + h * a.p.v_head * es + c;
      const i32x4 x = *reinterpret_cast<const i32x4*>(k + (fp * a.p.k_page + fr * a.p.k_slot) * es);
      const i32x4 y = *reinterpret_cast<const i32x4*>(v + (fp * a.p.v_page + fr * a.p.v_slot) * es);
      __builtin_nontemporal_store(x, reinterpret_cast<i32x4*>(k + (tp * a.p.k_page + tr * a.p.k_slot) * es));
      __builtin_nontemporal_store(y, reinterpret_cast<i32x4*>(v + (tp * a.p.v_page + tr * a.p.v_slot) * es));
    }
    if (c == 0) {
      const int64_t t = a.p.scalar_at(tp, h, (int)tr), f = a.p.scalar_at(fp, h, (int)fr);
      if (a.p.weight) a.p.weight[t] = a.p.weight[f];
      if (a.p.position) a.p.position[t] = a.p.position[f];
      if (a.p.k_scale) a.p.k_scale[t] = a.p.k_scale[f], a.p.v_scale[t] = a.p.v_scale[f];
    }
  }
}

int pow2_lanes(int64_t n) {
  int l = 1;
  while (l < n) l <<= 1;
  return l;
}

// Whether n values of 64 bits at a share memory with m at b.
bool meet(const int64_t* a, int64_t n, const int64_t* b, int64_t m) {
  const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
  return a && b && x < y + 8 * (uintptr_t)m && y < x + 8 * (uintptr_t)n;
}

template <class X>
int launch_append(const AppendArgs& a, const cortex_kv_pages* pages, hipStream_t stream) {
  const int dtype = (int)pages->dtype;
  const int lpr = pow2_lanes(a.p.head_dim / 8);
  // as many tokens a workgroup as its threads have loads in flight for, while every CU gets eight workgroups
  int64_t tokens = 256 * AP_AHEAD / (2ll * a.p.kv_heads * lpr), spread = a.T / (8 * cu_count());
  tokens = tokens < spread ? tokens : spread;
  tokens = tokens < 1 ? 1 : tokens > AP_TOKENS ? AP_TOKENS : tokens;
  CORTEX_CHECK_ARG(cdiv(a.T, tokens) <= 0xffffffffLL / 256, "cortex_kv_append: %lld tokens are too many for one call",
                   (long long)a.T);  // (a launch has fewer than 2^32 threads)
  const dim3 grid((unsigned)cdiv(a.T, tokens)), block(256);
  if (a.T > 0) {
    CORTEX_CHECK_ARG(!kv_rows_meet(pages), "cortex_kv_append: rows of k and v share memory");
    if (dtype == DT_F32)
      hipLaunchKernelGGL((kv_append_kernel<X, float>), grid, block, 0, stream, a, lpr, (int)tokens);
    else if (dtype == DT_BF16)
      hipLaunchKernelGGL((kv_append_kernel<X, bf16>), grid, block, 0, stream, a, lpr, (int)tokens);
    else
      hipLaunchKernelGGL((kv_append_kernel<X, int8_t>), grid, block, 0, stream, a, lpr, (int)tokens);
    CORTEX_CHECK_LAUNCH("kv_append_kernel");
  }
  if (a.offsets && a.new_lengths && (a.T == 0 || a.new_lengths == a.lengths)) {
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
  CORTEX_CHECK_ARG((new_lengths == lengths || !meet(new_lengths, B, lengths, B)) && !meet(new_lengths, B, offsets, B + 1) &&
                       !meet(new_lengths, B, positions, n_tokens),
                   "%s: new_lengths overlaps an input (it may only be lengths itself)", who);
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
  return x_dtype == DT_F32 ? launch_append<float>(a, pages, stream) : launch_append<bf16>(a, pages, stream);
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
  // (a launch has fewer than 2^32 threads)
  CORTEX_CHECK_ARG(B <= 0xffffffffLL / 1024 / pages->kv_heads, "%s: too many heads", who);
  CORTEX_CHECK_ARG(!meet(new_lengths, B, lengths, B), "%s: new_lengths may not be lengths, nor overlap them", who);
  a.lengths = lengths;
  a.dst = dst;
  a.src = src;
  a.counts = counts;
  a.new_lengths = new_lengths;
  a.err = err;
  const dim3 grid((unsigned)(B * pages->kv_heads));
  // the runs of eight slots that the longest sequence has for each thread
  if (a.max_length <= 8 * 256)
    hipLaunchKernelGGL((kv_evict_plan_kernel<256, 1>), grid, dim3(256), 0, stream, a);
  else if (a.max_length <= 8 * 1024)
    hipLaunchKernelGGL((kv_evict_plan_kernel<1024, 1>), grid, dim3(1024), 0, stream, a);
  else if (a.max_length <= 2 * 8 * 1024)
    hipLaunchKernelGGL((kv_evict_plan_kernel<1024, 2>), grid, dim3(1024), 0, stream, a);
  else if (a.max_length <= 4 * 8 * 1024)
    hipLaunchKernelGGL((kv_evict_plan_kernel<1024, 4>), grid, dim3(1024), 0, stream, a);
  else
    hipLaunchKernelGGL((kv_evict_plan_kernel<1024, 0>), grid, dim3(1024), 0, stream, a);
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
  CORTEX_CHECK_ARG(B <= 0xffffffffLL / 256 / pages->kv_heads, "%s: too many heads", who);
  CORTEX_CHECK_ARG(!kv_rows_meet(pages), "%s: rows of k and v share memory", who);
  const int es = pages->dtype == DT_F32 ? 4 : pages->dtype == DT_BF16 ? 2 : 1;
  a.dst = dst;
  a.src = src;
  a.cap = cap;
  a.counts = counts;
  a.err = err;
  a.row_bytes = (int)pages->head_dim * es;
  a.lanes = pow2_lanes(a.row_bytes / 16);
  // up to EA_PER_CU workgroups a CU for all heads together
  int64_t chunks = cdiv((int64_t)cu_count() * EA_PER_CU, B * pages->kv_heads);
  if (chunks > cdiv(cap, 256 / a.lanes)) chunks = cdiv(cap, 256 / a.lanes);
  a.chunks = (int)chunks;
  hipLaunchKernelGGL(kv_evict_apply_kernel, dim3((unsigned)(chunks * B * pages->kv_heads)), dim3(256), 0, stream, a, es);
  CORTEX_CHECK_LAUNCH("kv_evict_apply_kernel");
  return OK;
}
