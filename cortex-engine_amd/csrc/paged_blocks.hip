// Paged K/V cache by whole pages: copies of pages, the bounds of a page's keys, and the pages that a query may find its
// largest scores in.
//
// The bounds of a page are, for every dim, the largest and the smallest value of its keys.  With them
//   q . k  <=  sum_d max(q_d max_d, q_d min_d)  =  max(q, 0) . max + min(q, 0) . min
// for every key k of the page: one product of 2 head_dim terms stands for page_size of them.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "paged_kv.h"

namespace cortex {
namespace {

int row_bytes_of(const cortex_kv_pages* p) {
  return (int)p->head_dim * (p->dtype == DT_F32 ? 4 : p->dtype == DT_BF16 ? 2 : 1);
}
int pow2_from(int n) {
  int l = 1;
  while (l < n) l <<= 1;
  return l;
}
// head_dim values of a page's bounds: of the keys' type, fp32 for int8
int bound_bytes_of(const cortex_kv_pages* p) { return p->dtype == DT_BF16 ? 2 : 4; }

// ---------------------------------------------------------------------------- copy

struct CopyArgs {
  KvPages from, to;
  const char* from_bounds;
  char* to_bounds;
  const int32_t* src;
  const int32_t* dst;
  int32_t* err;
  int parts;       // workgroups a page
  int rows;        // rows of a workgroup, a multiple of 4
  int lanes;       // lanes a row (a power of two), 16 bytes each
  int row_bytes;
  int bounds_bytes;  // of a page
  int es;
};

constexpr int CP_AHEAD = 4;  // rows in flight, keys and values of each

// `lanes` lanes a row, 16 bytes of the key and of the value each; the arrays by row lie in the order of a page's
// (head, row) and are copied 16 bytes at a time.
__global__ __launch_bounds__(256) void kv_copy_pages_kernel(CopyArgs a) {
  const int tid = threadIdx.x;
  const int64_t i = blockIdx.x / a.parts;
  const int part = (int)(blockIdx.x - i * a.parts);
  const int sp = a.src[i], dp = a.dst[i];
  if ((uint32_t)sp >= (uint32_t)a.from.num_pages || (uint32_t)dp >= (uint32_t)a.to.num_pages) {
    if (part == 0 && tid == 0) kv_flag(a.err);
    return;
  }
  const int all = a.from.kv_heads << a.from.shift;
  const int r0 = part * a.rows, r1 = min(all, r0 + a.rows);
  const int groups = 256 / a.lanes, c = (tid % a.lanes) * 16;
  const int mask = (1 << a.from.shift) - 1;
  const char* k = reinterpret_cast<const char*>(a.from.k) + sp * a.from.k_page * a.es + c;
  const char* v = reinterpret_cast<const char*>(a.from.v) + sp * a.from.v_page * a.es + c;
  char* ko = reinterpret_cast<char*>(a.to.k) + dp * a.to.k_page * a.es + c;
  char* vo = reinterpret_cast<char*>(a.to.v) + dp * a.to.v_page * a.es + c;
  if (c < a.row_bytes) {
    for (int r = r0 + tid / a.lanes; r < r1; r += groups * CP_AHEAD) {
      i32x4 x[CP_AHEAD], y[CP_AHEAD];
#pragma unroll
      for (int s = 0; s < CP_AHEAD; ++s) {
        const int at = min(r + s * groups, r1 - 1), h = at >> a.from.shift, row = at & mask;
        x[s] = *reinterpret_cast<const i32x4*>(k + (h * a.from.k_head + row * a.from.k_slot) * a.es);
        y[s] = *reinterpret_cast<const i32x4*>(v + (h * a.from.v_head + row * a.from.v_slot) * a.es);
      }
#pragma unroll
      for (int s = 0; s < CP_AHEAD; ++s) {
        const int at = r + s * groups, h = at >> a.to.shift, row = at & mask;
        if (at < r1) {
          __builtin_nontemporal_store(x[s], reinterpret_cast<i32x4*>(ko + (h * a.to.k_head + row * a.to.k_slot) * a.es));
          __builtin_nontemporal_store(y[s], reinterpret_cast<i32x4*>(vo + (h * a.to.v_head + row * a.to.v_slot) * a.es));
        }
      }
    }
  }
  const int64_t from = (int64_t)sp * all, to = (int64_t)dp * all;
  auto by_row = [&](const void* x, void* y) {
    if (x == nullptr) return;
    for (int r = r0 + 4 * tid; r < r1; r += 4 * 256)
      *reinterpret_cast<i32x4*>(reinterpret_cast<int32_t*>(y) + to + r) =
          *reinterpret_cast<const i32x4*>(reinterpret_cast<const int32_t*>(x) + from + r);
  };
  by_row(a.from.weight, a.to.weight);
  by_row(a.from.position, a.to.position);
  by_row(a.from.k_scale, a.to.k_scale);
  by_row(a.from.v_scale, a.to.v_scale);
  if (part == 0 && a.from_bounds)
    for (int x = 16 * tid; x < a.bounds_bytes; x += 16 * 256)
      *reinterpret_cast<i32x4*>(a.to_bounds + (int64_t)dp * a.bounds_bytes + x) =
          *reinterpret_cast<const i32x4*>(a.from_bounds + (int64_t)sp * a.bounds_bytes + x);
}

// ---------------------------------------------------------------------------- bounds

struct BoundsArgs {
  KvPages p;
  void* bounds;
  const int64_t* lengths;
  const int64_t* since;
  int64_t max_length;
  int32_t* err;
  int chunks;  // workgroups a sequence
  int lanes;   // lanes a row
};

// The larger and the smaller of two numbers, NaN where either is.
__device__ __forceinline__ float most_of(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float least_of(float a, float b) { return __builtin_elementwise_minimum(a, b); }

constexpr int KB_AHEAD = 4;  // rows in flight a lane

// A wavefront takes a (page, key head) at a time: `lanes` lanes a row, 16 bytes each, the groups of lanes joined at the end.
template <class P>
__global__ __launch_bounds__(256) void kv_bounds_kernel(BoundsArgs a) {
  constexpr int ES = sizeof(P), N = 16 / ES;
  typedef typename std::conditional<ES == 2, bf16, float>::type O;
  const KvPages& p = a.p;
  const int lane = threadIdx.x & 63, wid = wave_uniform((int)threadIdx.x >> 6);
  const int b = blockIdx.x / a.chunks, chunk = blockIdx.x - b * a.chunks;
  bool ok = true;
  const int64_t n = p.length_of(a.lengths, b, a.max_length, &ok);
  if (!ok && chunk == 0 && threadIdx.x == 0) kv_flag(a.err);
  const int64_t begin = a.since ? min(max(a.since[b], (int64_t)0), n) : 0;
  if (begin == n) return;
  const int first = (int)(begin >> p.shift), blocks = (int)((n - 1) >> p.shift) + 1 - first;
  const int groups = 64 / a.lanes, group = lane / a.lanes, d = (lane % a.lanes) * N;
  const bool in = d < p.head_dim;
  const int64_t items = (int64_t)blocks * p.kv_heads;
  for (int64_t i = (int64_t)chunk * 4 + wid; i < items; i += (int64_t)a.chunks * 4) {
    const int block = (int)(i / p.kv_heads), h = (int)(i - (int64_t)block * p.kv_heads);
    const int64_t j = (int64_t)(first + block) << p.shift;
    const int page = p.page_of(b, j);
    if (page < 0) {
      if (lane == 0) kv_flag(a.err);
      continue;
    }
    const int used = (int)min(n - j, 1ll << p.shift);
    const char* k = reinterpret_cast<const char*>(p.k) + (page * p.k_page + h * p.k_head + (in ? d : 0)) * ES;
    const float* scale = ES == 1 ? p.k_scale + p.scalar_at(page, h, 0) : nullptr;
    float most[N], least[N];
#pragma unroll
    for (int e = 0; e < N; ++e) most[e] = -INFINITY, least[e] = INFINITY;
    for (int r = group; r < used; r += groups * KB_AHEAD) {
      i32x4 x[KB_AHEAD];
      float s[KB_AHEAD];
#pragma unroll
      for (int y = 0; y < KB_AHEAD; ++y) {  // (the last row again where there are no more: it changes nothing)
        const int row = min(r + y * groups, used - 1);
        x[y] = *reinterpret_cast<const i32x4*>(k + row * p.k_slot * ES);
        s[y] = ES == 1 ? scale[row] : 1.0f;
      }
#pragma unroll
      for (int y = 0; y < KB_AHEAD; ++y) {
        P v[N];
        __builtin_memcpy(v, &x[y], 16);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float f = ES == 1 ? to_f32(v[e]) * s[y] : to_f32(v[e]);
          most[e] = most_of(most[e], f);
          least[e] = least_of(least[e], f);
        }
      }
    }
    for (int o = a.lanes; o < 64; o <<= 1)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        most[e] = most_of(most[e], __shfl_xor(most[e], o, 64));
        least[e] = least_of(least[e], __shfl_xor(least[e], o, 64));
      }
    if (group == 0 && in) {
      O out[2][N];
#pragma unroll
      for (int e = 0; e < N; ++e) out[0][e] = from_f32<O>(most[e]), out[1][e] = from_f32<O>(least[e]);
      O* to = reinterpret_cast<O*>(a.bounds) + ((int64_t)page * p.kv_heads + h) * 2 * p.head_dim + d;
#pragma unroll
      for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int x = 0; x < (int)(N * sizeof(O) / 16); ++x) {
          i32x4 w;
          __builtin_memcpy(&w, reinterpret_cast<const char*>(out[y]) + 16 * x, 16);
          reinterpret_cast<i32x4*>(to + y * p.head_dim)[x] = w;
        }
    }
  }
}

// ---------------------------------------------------------------------------- selection

struct SelectArgs {
  KvPages p;
  const void* bounds;
  int B, heads, group;
  const void* q;
  int64_t q_sb, q_sh;
  const int64_t* lengths;
  int64_t max_length;
  int count, first, recent;
  int32_t* table;  // (B, kv_heads, keep)
  int64_t* new_lengths;
  int keep;
  int32_t* err;
  uint32_t* rank;  // workspace: (B, kv_heads, ld)
  int64_t ld;
  int tiles;       // of 16 blocks a (sequence, key head) at most
};

// Ranks: 0 for a block without a page, then by score, NaN above every number, then the blocks that are always kept.
constexpr uint32_t KEPT = 0xffffffffu, NOT_A_NUMBER = 0xfffffffeu;
__device__ __forceinline__ uint32_t rank_of(float score) {
  if (score != score) return NOT_A_NUMBER;
  const uint32_t u = __float_as_uint(score + 0.0f);  // -0 and 0 are equal
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

__device__ __forceinline__ int blocks_of(const SelectArgs& a, int64_t n) {
  return (int)((n + (1ll << a.p.shift) - 1) >> a.p.shift);
}

// The ranks of 16 blocks a wavefront.  The sums are in 64 bits and rounded to 32 once: which blocks are chosen does not
// depend on an order of sums.  v_mfma_f64_4x4x4 multiplies four 4 x 4 tiles: lane 16 g + r loads eight dims 8 (4 c + g) ..
// of the bounds of block r and of the query of head r % 4, and gets the sum of block 4 ((l % 16) / 4) + l / 16 and
// head l % 4.  DHP: head_dim rounded up to 32.
template <class O, class Q, int DHP>
__global__ __launch_bounds__(256) void kv_rank_kernel(SelectArgs a) {
  constexpr int NC = DHP / 32;
  const KvPages& p = a.p;
  const int lane = threadIdx.x & 63, wid = wave_uniform((int)threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int64_t w = (int64_t)blockIdx.x * 4 + wid;
  const int bh = (int)(w / a.tiles), tile = (int)(w - (int64_t)bh * a.tiles);
  if (bh >= a.B * p.kv_heads) return;
  const int b = bh / p.kv_heads, h = bh - b * p.kv_heads;
  bool ok = true;
  const int64_t n = p.length_of(a.lengths, b, a.max_length, &ok);
  const int blocks = blocks_of(a, n);
  if (blocks <= a.count || tile * 16 >= blocks) return;  // (all of them are kept)
  const int block = min(tile * 16 + r, blocks - 1);
  const int page = p.page_of(b, (int64_t)block << p.shift);
  if (page < 0 && g == 0) kv_flag(a.err);
  const O* bounds = reinterpret_cast<const O*>(a.bounds) + ((int64_t)max(page, 0) * p.kv_heads + h) * 2 * p.head_dim;
  double key[2][NC][8];
#pragma unroll
  for (int y = 0; y < 2; ++y)
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int d = 8 * (4 * c + g);
      O x[8] = {};
      if (d < p.head_dim) __builtin_memcpy(x, __builtin_assume_aligned(bounds + y * p.head_dim + d, 16), sizeof(x));
#pragma unroll
      for (int e = 0; e < 8; ++e) key[y][c][e] = (double)to_f32(x[e]);
    }
  uint32_t best = 0;
  for (int i0 = 0; i0 < a.group; i0 += 4) {
    const Q* q = reinterpret_cast<const Q*>(a.q) + b * a.q_sb + (int64_t)(h * a.group + min(i0 + (r & 3), a.group - 1)) * a.q_sh;
    double sum = 0.0;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int d = 8 * (4 * c + g);
      Q x[8] = {};
      if (d < p.head_dim) __builtin_memcpy(x, __builtin_assume_aligned(q + d, 16), sizeof(x));
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float f = to_f32(x[e]);
        // (a NaN reaches the sum by the first)
        sum = __builtin_amdgcn_mfma_f64_4x4x4f64(key[0][c][e], (double)(f < 0.0f ? 0.0f : f), sum, 0, 0, 0);
        sum = __builtin_amdgcn_mfma_f64_4x4x4f64(key[1][c][e], (double)(f < 0.0f ? f : 0.0f), sum, 0, 0, 0);
      }
    }
    best = max(best, rank_of((float)sum));
  }
  best = max(best, (uint32_t)__shfl_xor((int)best, 1, 64));
  best = max(best, (uint32_t)__shfl_xor((int)best, 2, 64));
  // this lane's score is of block 4 (r / 4) + g; its lookup was of block r
  const int mine = tile * 16 + 4 * (r >> 2) + g;
  const int its_page = __shfl(page, 4 * (r >> 2) + g, 64);
  if ((r & 3) == 0 && mine < blocks) {
    if (its_page < 0) best = 0;
    if (mine < a.first || mine >= blocks - a.recent) best = KEPT;
    a.rank[(int64_t)bh * a.ld + mine] = best;
  }
}

__device__ __forceinline__ int scan64(int v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(v, o, 64);
    if (lane >= o) v += u;
  }
  return v;
}

constexpr int SL_THREADS = 256;

// The `count` largest ranks of a (sequence, key head) by a radix selection of a byte a round, and their pages in the
// order of the blocks.
__global__ __launch_bounds__(SL_THREADS) void kv_select_kernel(SelectArgs a) {
  constexpr int WAVES = SL_THREADS / 64;
  __shared__ __attribute__((aligned(16))) int hist[256];
  __shared__ int part[2][WAVES];
  __shared__ int picked[3];
  const KvPages& p = a.p;
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int b = blockIdx.x / p.kv_heads, h = blockIdx.x - b * p.kv_heads;
  bool ok = true;
  const int64_t n = p.length_of(a.lengths, b, a.max_length, &ok);
  const int blocks = blocks_of(a, n), kept = min(blocks, a.keep);
  const int32_t* pages = p.table + b * p.ld_table;
  int32_t* out = a.table + (int64_t)blockIdx.x * a.keep;
  if (h == 0 && tid == 0) {
    if (!ok) kv_flag(a.err);
    a.new_lengths[b] = n - ((int64_t)(blocks - kept) << p.shift);
  }
  for (int i = kept + tid; i < a.keep; i += SL_THREADS) out[i] = -1;
  if (blocks <= a.count) {
    for (int i = tid; i < blocks; i += SL_THREADS) {
      out[i] = pages[i];
      if ((uint32_t)pages[i] >= (uint32_t)p.num_pages) kv_flag(a.err);
    }
    return;
  }
  const uint32_t* rank = a.rank + (int64_t)blockIdx.x * a.ld;
  uint32_t found = 0;
  int need = a.count;
  for (int shift = 24; shift >= 0; shift -= 8) {
    hist[tid] = 0;
    __syncthreads();
    for (int i = tid; i < blocks; i += SL_THREADS) {
      const uint32_t x = rank[i];
      if (shift == 24 || (x >> (shift + 8)) == (found >> (shift + 8))) atomicAdd(&hist[(x >> shift) & 255], 1);
    }
    __syncthreads();
    if (wid == 0) {  // lane l has the bins 252 - 4 l .. 255 - 4 l
      const int4 c = *reinterpret_cast<const int4*>(&hist[252 - 4 * lane]);
      const int many[4] = {c.w, c.z, c.y, c.x};  // the largest ranks first
      const int sum = (c.x + c.y) + (c.z + c.w);
      int before = scan64(sum, lane) - sum;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (before < need && before + many[i] >= need)  // (one bin of one lane)
          picked[0] = 255 - 4 * lane - i, picked[1] = before, picked[2] = many[i];
        before += many[i];
      }
    }
    __syncthreads();
    found |= (uint32_t)picked[0] << shift;
    need -= picked[1];
    if (need == picked[2]) break;  // (all that share the bytes found are kept; every thread sees the same)
    __syncthreads();
  }
  // ranks above `found`, and of those equal to it in the bytes found the first `need`: in the order of the blocks
  int at = 0, tie = 0;
  const bool whole = need == picked[2];
  for (int i0 = 0; i0 < blocks; i0 += SL_THREADS) {
    const int i = i0 + tid;
    const uint32_t x = i < blocks ? rank[i] : 0;
    const bool there = i < blocks, above = there && (whole ? x >= found : x > found), equal = there && !whole && x == found;
    const uint64_t ties = __ballot(equal);
    __syncthreads();
    if (lane == 0) part[0][wid] = __popcll(ties);
    __syncthreads();
    int before = tie, sum = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      if (w < wid) before += part[0][w];
      sum += part[0][w];
    }
    before += __popcll(ties & ((1ull << lane) - 1));
    tie += sum;
    const bool keep = above || (equal && before < need);
    const uint64_t all = __ballot(keep);
    if (lane == 0) part[1][wid] = __popcll(all);
    __syncthreads();
    int to = at;
    sum = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      if (w < wid) to += part[1][w];
      sum += part[1][w];
    }
    to += __popcll(all & ((1ull << lane) - 1));
    at += sum;
    if (keep && to < kept) out[to] = pages[i];
  }
}

int check_bounds(const char* who, const cortex_kv_pages* pages) {
  CORTEX_CHECK_ARG(pages->bounds && (uintptr_t)pages->bounds % 16 == 0, "%s: the pages need 16-byte aligned bounds", who);
  return OK;
}

}  // namespace
}  // namespace cortex

using namespace cortex;

extern "C" int cortex_kv_copy_pages(const cortex_kv_pages* from, const cortex_kv_pages* to, int64_t n, const int32_t* src,
                                    const int32_t* dst, int32_t* err, hipStream_t stream) {
  const char* who = "cortex_kv_copy_pages";
  CopyArgs a = {};
  if (int rc = kv_check(who, from, 0, nullptr, 0, 0, &a.from)) return rc;
  if (int rc = kv_check(who, to, 0, nullptr, 0, 0, &a.to)) return rc;
  CORTEX_CHECK_ARG(from->kv_heads == to->kv_heads && from->page_size == to->page_size && from->head_dim == to->head_dim &&
                       from->dtype == to->dtype,
                   "%s: pages of different shapes", who);
  CORTEX_CHECK_ARG(!from->weight == !to->weight && !from->position == !to->position && !from->bounds == !to->bounds,
                   "%s: weight, position and bounds must be in both pools or in neither", who);
  CORTEX_CHECK_ARG(((uintptr_t)from->bounds | (uintptr_t)to->bounds) % 16 == 0, "%s: bounds must be 16-byte aligned", who);
  CORTEX_CHECK_ARG(n >= 0, "%s: negative count", who);
  if (n == 0) return OK;
  CORTEX_CHECK_ARG(src && dst, "%s: null pointer", who);
  CORTEX_CHECK_ARG(!kv_rows_meet(to), "%s: rows of k and v share memory", who);
  const int64_t all = from->kv_heads * from->page_size;
  CORTEX_CHECK_ARG(all <= 0x7fffffffLL - 65536, "%s: pages of %lld rows", who, (long long)all);
  a.from_bounds = reinterpret_cast<const char*>(from->bounds);
  a.to_bounds = reinterpret_cast<char*>(to->bounds);
  a.src = src;
  a.dst = dst;
  a.err = err;
  a.row_bytes = row_bytes_of(from);
  a.lanes = pow2_from(a.row_bytes / 16);
  a.es = a.row_bytes / (int)from->head_dim;
  a.bounds_bytes = (int)(from->kv_heads * 2 * from->head_dim * bound_bytes_of(from));
  // two rounds of loads a workgroup, one where that leaves CUs without any
  const int64_t one = (int64_t)(256 / a.lanes) * CP_AHEAD;
  const int64_t rows = n * cdiv(all, 2 * one) >= cu_count() ? 2 * one : one;
  a.rows = (int)rows;
  a.parts = (int)cdiv(all, rows);
  CORTEX_CHECK_ARG(n <= 0xffffffffLL / 256 / a.parts, "%s: %lld pages are too many for one call", who, (long long)n);
  hipLaunchKernelGGL(kv_copy_pages_kernel, dim3((unsigned)(n * a.parts)), dim3(256), 0, stream, a);
  CORTEX_CHECK_LAUNCH("kv_copy_pages_kernel");
  return OK;
}

extern "C" int cortex_kv_block_bounds(const cortex_kv_pages* pages, int64_t B, const int32_t* block_table, int64_t ld_table,
                                      int64_t max_pages, const int64_t* lengths, int64_t max_length, const int64_t* since,
                                      int64_t max_new, int32_t* err, hipStream_t stream) {
  const char* who = "cortex_kv_block_bounds";
  BoundsArgs a = {};
  if (int rc = kv_check(who, pages, B, block_table, ld_table, max_pages, &a.p)) return rc;
  if (int rc = check_bounds(who, pages)) return rc;
  a.max_length = max_length < 0 || max_length > a.p.max_slots ? a.p.max_slots : max_length;
  if (B == 0 || a.max_length == 0) return OK;
  CORTEX_CHECK_ARG(lengths, "%s: null lengths", who);
  a.bounds = pages->bounds;
  a.lengths = lengths;
  a.since = since;
  a.err = err;
  a.lanes = pow2_from(row_bytes_of(pages) / 16);
  // blocks that slots of a sequence are in: all, or those that max_new slots in a row touch
  int64_t blocks = cdiv(a.max_length, pages->page_size);
  if (since && max_new >= 0 && max_new < a.max_length) {
    const int64_t touched = max_new == 0 ? 0 : (max_new + pages->page_size - 2) / pages->page_size + 1;
    if (touched < blocks) blocks = touched;
  }
  if (blocks == 0) blocks = 1;
  const int64_t need = cdiv(blocks * pages->kv_heads, 4), share = cdiv((int64_t)cu_count() * 64, B);
  a.chunks = (int)(need < share ? need : share);
  CORTEX_CHECK_ARG(B <= 0xffffffffLL / 256 / a.chunks, "%s: %lld sequences are too many for one call", who, (long long)B);
  const dim3 grid((unsigned)(B * a.chunks)), block(256);
  if (pages->dtype == DT_F32)
    hipLaunchKernelGGL(kv_bounds_kernel<float>, grid, block, 0, stream, a);
  else if (pages->dtype == DT_BF16)
    hipLaunchKernelGGL(kv_bounds_kernel<bf16>, grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL(kv_bounds_kernel<int8_t>, grid, block, 0, stream, a);
  CORTEX_CHECK_LAUNCH("kv_bounds_kernel");
  return OK;
}

namespace cortex {
namespace {

// blocks of the longest sequence that a call expects
int64_t most_blocks(const cortex_kv_pages* pages, int64_t most) { return cdiv(most, pages->page_size); }
// ranks of a (sequence, key head) in the workspace: none where all blocks are kept
int64_t rank_ld(const cortex_kv_pages* pages, int64_t most, int64_t count) {
  const int64_t blocks = most_blocks(pages, most);
  return blocks <= count ? 0 : cdiv(blocks, 16) * 16;
}

template <class O, class Q>
void launch_rank(const SelectArgs& a, unsigned grid, hipStream_t stream) {
  if (a.p.head_dim <= 32)
    hipLaunchKernelGGL((kv_rank_kernel<O, Q, 32>), dim3(grid), dim3(256), 0, stream, a);
  else if (a.p.head_dim <= 64)
    hipLaunchKernelGGL((kv_rank_kernel<O, Q, 64>), dim3(grid), dim3(256), 0, stream, a);
  else if (a.p.head_dim <= 96)
    hipLaunchKernelGGL((kv_rank_kernel<O, Q, 96>), dim3(grid), dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((kv_rank_kernel<O, Q, 128>), dim3(grid), dim3(256), 0, stream, a);
}

}  // namespace
}  // namespace cortex

extern "C" int64_t cortex_kv_select_workspace_bytes(const cortex_kv_pages* pages, int64_t B, int64_t max_length,
                                                    int64_t count) {
  if (!pages || pages->page_size < 1 || pages->kv_heads < 1 || B < 0 || max_length < 0 || count < 0) return 0;
  return B * pages->kv_heads * rank_ld(pages, max_length, count) * 4;
}

extern "C" int cortex_kv_select(const cortex_kv_pages* pages, int64_t B, int64_t heads, const void* q, int64_t q_sb,
                                int64_t q_sh, const int32_t* block_table, int64_t ld_table, int64_t max_pages,
                                const int64_t* lengths, int64_t max_length, int64_t count, int64_t first, int64_t recent,
                                int32_t* table, int64_t* new_lengths, void* workspace, int64_t workspace_bytes, int32_t* err,
                                hipStream_t stream) {
  const char* who = "cortex_kv_select";
  SelectArgs a = {};
  if (int rc = kv_check(who, pages, B, block_table, ld_table, max_pages, &a.p)) return rc;
  if (int rc = check_bounds(who, pages)) return rc;
  CORTEX_CHECK_ARG(heads >= 1 && heads % pages->kv_heads == 0 && heads / pages->kv_heads <= 1024,
                   "%s: %lld query heads are not a multiple (up to 1024) of %lld key heads", who, (long long)heads,
                   (long long)pages->kv_heads);
  CORTEX_CHECK_ARG(count >= 1 && first >= 0 && recent >= 1 && first <= count - recent,
                   "%s: count %lld has to hold the first %lld and the last %lld (at least one) blocks", who, (long long)count,
                   (long long)first, (long long)recent);
  a.max_length = max_length < 0 || max_length > a.p.max_slots ? a.p.max_slots : max_length;
  if (B == 0) return OK;
  CORTEX_CHECK_ARG(q && lengths && new_lengths, "%s: null pointer", who);
  const int64_t es = pages->dtype == DT_F32 ? 4 : 2;
  CORTEX_CHECK_ARG((uintptr_t)q % 16 == 0 && (q_sb * es) % 16 == 0 && (q_sh * es) % 16 == 0,
                   "%s: query rows must be 16-byte aligned", who);
  const int64_t blocks = most_blocks(pages, a.max_length), ld = rank_ld(pages, a.max_length, count);
  const int64_t keep = count < blocks ? count : blocks;
  CORTEX_CHECK_ARG(table || keep == 0, "%s: null table", who);
  CORTEX_CHECK_ARG((workspace || ld == 0) && (uintptr_t)workspace % 16 == 0, "%s: null or unaligned workspace", who);
  // (a launch has fewer than 2^32 threads)
  CORTEX_CHECK_ARG(B <= 0xffffffffLL / SL_THREADS / pages->kv_heads &&
                       (ld == 0 || B * pages->kv_heads <= 0xffffff00LL / 64 / (ld / 16)),
                   "%s: %lld sequences of up to %lld blocks are too much for one call", who, (long long)B, (long long)blocks);
  if (workspace_bytes < B * pages->kv_heads * ld * 4) {
    set_error("%s: workspace of %lld bytes, %lld needed", who, (long long)workspace_bytes,
              (long long)(B * pages->kv_heads * ld * 4));
    return E_WORKSPACE;
  }
  a.bounds = pages->bounds;
  a.B = (int)B;
  a.heads = (int)heads;
  a.group = (int)(heads / pages->kv_heads);
  a.q = q;
  a.q_sb = q_sb;
  a.q_sh = q_sh;
  a.lengths = lengths;
  a.count = (int)(count < (1ll << 30) ? count : 1ll << 30);
  a.first = (int)(first < (1ll << 30) ? first : 1ll << 30);
  a.recent = (int)(recent < (1ll << 30) ? recent : 1ll << 30);
  a.table = table;
  a.new_lengths = new_lengths;
  a.keep = (int)keep;
  a.err = err;
  a.rank = reinterpret_cast<uint32_t*>(workspace);
  a.ld = ld;
  a.tiles = (int)(ld / 16);
  if (ld > 0) {
    const unsigned grid = (unsigned)cdiv(B * pages->kv_heads * a.tiles, 4);
    if (pages->dtype == DT_F32)
      launch_rank<float, float>(a, grid, stream);
    else if (pages->dtype == DT_BF16)
      launch_rank<bf16, bf16>(a, grid, stream);
    else
      launch_rank<float, bf16>(a, grid, stream);
    CORTEX_CHECK_LAUNCH("kv_rank_kernel");
  }
  hipLaunchKernelGGL(kv_select_kernel, dim3((unsigned)(B * pages->kv_heads)), dim3(SL_THREADS), 0, stream, a);
  CORTEX_CHECK_LAUNCH("kv_select_kernel");
  return OK;
}
