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
// (head, row) and are copied 16 bytes at a time.  Bound by HBM: 2053 pages of 16 rows x 8 heads x 128 in bf16 with weight and
// position, 273 MB read and written, 57.8 us among other calls, 4.7 TB/s; one page 2.5.
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
constexpr int KB_PER_CU = 32;  // workgroups (16 sequences of 1000 .. 15001 int8 keys, 4 heads x 128: 8 a CU 24.2 us, 16 21.8, 32 and 64 21.0)

// What two lanes have of the same dims, joined: the lanes of the lower half (of every 32, of every 64) go on with a, the
// others with b.
template <int SPAN, class F>
__device__ __forceinline__ float halves(float a, float b, F f) {
  if constexpr (SPAN == 64) {
    const auto u = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return f(__uint_as_float(u[0]), __uint_as_float(u[1]));
  } else {
    const auto u = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return f(__uint_as_float(u[0]), __uint_as_float(u[1]));
  }
}

// x[0 .. N): N dims of a row in each of 64 / lanes groups of lanes.  Joined over the groups, the first N / 4 (32 lanes a row:
// N / 2) hold dims N / 2 (lane / 32) + N / 4 (lane / 16 % 2) .. (N / 2 (lane / 32) ..).
template <int N, class F>
__device__ __forceinline__ void join_groups(float (&x)[N], int lanes, F f) {
#pragma unroll
  for (int e = 0; e < N / 2; ++e) x[e] = halves<64>(x[e], x[e + N / 2], f);
  if (lanes > 16) return;
#pragma unroll
  for (int e = 0; e < N / 4; ++e) x[e] = halves<32>(x[e], x[e + N / 4], f);
#pragma unroll
  for (int e = 0; e < N / 4; ++e) {
    if (lanes <= 8) x[e] = f(x[e], dpp_mov<0x128>(x[e]));
    if (lanes <= 4) x[e] = f(x[e], __shfl_xor(x[e], 4, 64));
    if (lanes <= 2) x[e] = f(x[e], dpp_mov<0x4E>(x[e]));
    if (lanes <= 1) x[e] = f(x[e], dpp_mov<0xB1>(x[e]));
  }
}

template <class O, int N>
__device__ __forceinline__ void store_bounds(O* to, const float* f) {
  O v[N];
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = from_f32<O>(f[e]);
  __builtin_memcpy(__builtin_assume_aligned(to, N * sizeof(O)), v, sizeof(v));
}

// A wavefront takes a (page, key head) at a time: `lanes` lanes a row, 16 bytes each, the groups of lanes joined at the end.
// 16 sequences of 1000 .. 15001 int8 keys, 4 heads x 128, 84 MB: 20.8 us, 4.0 TB/s.  A value takes a conversion, a product with
// its row's scale and half of a three-operand maximum and minimum each, about as long as its bytes: 20.3 us with the rows in
// cache, 15.6 without the arithmetic, 17.6 without the join, 10.2 with neither rows nor arithmetic.  The next page loaded while
// one is joined takes 184 registers: 32 us.  Joined by shuffles it was 24.6.
// The same keys in bf16, and in fp32 with 64 dims, 139 MB: 23.5 and 23.3 us, 5.9 TB/s.
// The last page of 32 sequences: 3.9 us, the chain length -> table -> rows.
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
  const int end = (int)((n - 1) >> p.shift) + 1;
  const int group = lane / a.lanes, groups = 64 / a.lanes, d = (lane & (a.lanes - 1)) * N;
  const bool in = d < p.head_dim;
  // blocks and heads of this wavefront: `step` further are `blocks` blocks and `heads` heads
  const int step = a.chunks * 4, blocks = step / p.kv_heads, heads = step - blocks * p.kv_heads;
  const int i0 = chunk * 4 + wid;
  int block = (int)(begin >> p.shift) + i0 / p.kv_heads, h = i0 % p.kv_heads;
  int page = block < end ? p.page_of(b, (int64_t)block << p.shift) : -1;
  while (block < end) {
    const int64_t j = (int64_t)block << p.shift;
    const int now = page, head = h;
    h += heads;
    block += blocks + (h >= p.kv_heads ? 1 : 0);
    h -= h >= p.kv_heads ? p.kv_heads : 0;
    if (block < end) page = p.page_of(b, (int64_t)block << p.shift);
    if (now < 0) {
      if (lane == 0) kv_flag(a.err);
      continue;
    }
    const int used = (int)min(n - j, 1ll << p.shift);
    const char* k = reinterpret_cast<const char*>(p.k) + (now * p.k_page + head * p.k_head + (in ? d : 0)) * ES;
    const float* scale = ES == 1 ? p.k_scale + p.scalar_at(now, head, 0) : nullptr;
    float most[N], least[N];
#pragma unroll
    for (int e = 0; e < N; ++e) most[e] = -INFINITY, least[e] = INFINITY;
    for (int r = group; r - group < used; r += groups * KB_AHEAD) {
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
    join_groups<N>(most, a.lanes, most_of);
    join_groups<N>(least, a.lanes, least_of);
    // (lanes of 16 that hold the same: the first of them)
    if (in && (a.lanes >= 16 || (lane & 15) < a.lanes)) {
      O* to = reinterpret_cast<O*>(a.bounds) + ((int64_t)now * p.kv_heads + head) * 2 * p.head_dim + d + (lane >> 5) * (N / 2);
      if (ES == 4 && a.lanes > 16) {
        store_bounds<O, N / 2>(to, most);
        store_bounds<O, N / 2>(to + p.head_dim, least);
      } else {
        to += (lane >> 4 & 1) * (N / 4);
        store_bounds<O, N / 4>(to, most);
        store_bounds<O, N / 4>(to + p.head_dim, least);
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
};

// Ranks: 1 for a block without a page, then by score, NaN above every number.  (0: not a candidate.)
constexpr uint32_t NO_PAGE = 1u, NOT_A_NUMBER = 0xffffffffu;
__device__ __forceinline__ uint32_t rank_of(float score) {
  if (score != score) return NOT_A_NUMBER;
  const uint32_t u = __float_as_uint(score + 0.0f);  // -0 and 0 are equal
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

__device__ __forceinline__ int blocks_of(const SelectArgs& a, int64_t n) {
  return (int)((n + (1ll << a.p.shift) - 1) >> a.p.shift);
}

// The ranks of tiles of 16 blocks, a tile a wavefront.  The sums are in 64 bits, in one order for every form of the launch, and
// rounded to 32 once; those of bf16 products are exact as long as the terms lie within 2^29 of each other.  So neither the
// batch nor the launch decides which blocks are chosen, and another order of sums would not.  v_mfma_f64_4x4x4 multiplies four 4 x 4 tiles: lane 16 g + r takes eight dims
// 8 (4 c + g) .. of the bounds of block r and of the query of head r % 4, and gets the sum of block 4 ((l % 16) / 4) + l / 16
// and head l % 4.  The bounds come from memory into registers; the queries, max(q, 0) and min(q, 0) in 64 bits, are made
// once a workgroup while its first bounds are on their way, into LDS: converted at each use they are half of the work.
// Matrix and vector instructions add up here, from whichever wavefront they come (20 cycles a product of a wavefront, 20 + 17
// with four vector instructions beside it): 64 products and as many unpackings and conversions a tile of 128 dims take 1900.
// DHP: head_dim rounded up to 64; NG: fours of query heads at a time.
template <class O, class Q, int DHP, int NG>
struct Scores {
  static constexpr int NC = DHP / 32, HEADS = 4 * NG;
  static constexpr int LD = DHP + 2;  // of a head in LDS: the four heads of a read are in different banks
  struct Bounds {
    O x[2][NC][8];
  };
  struct Query {
    double x[2][HEADS][LD];
  };

  // query heads i .. of a key head (the last one again where there are no more)
  template <int THREADS>
  static __device__ __forceinline__ void load_query(const SelectArgs& a, Query& to, int64_t b, int h, int i) {
    for (int at = threadIdx.x * 4; at < HEADS * DHP; at += THREADS * 4) {
      const int j = at / DHP, d = at % DHP;
      Q x[4] = {};
      if (d < a.p.head_dim)
        __builtin_memcpy(x, __builtin_assume_aligned(reinterpret_cast<const Q*>(a.q) + b * a.q_sb +
                                                     (int64_t)(h * a.group + min(i + j, a.group - 1)) * a.q_sh + d, 4 * sizeof(Q)), sizeof(x));
#pragma unroll
      for (int e = 0; e < 4; ++e) {  // (a NaN is in the first)
        const float f = to_f32(x[e]);
        to.x[0][j][d + e] = (double)(f < 0.0f ? 0.0f : f);
        to.x[1][j][d + e] = (double)(f < 0.0f ? f : 0.0f);
      }
    }
  }
  static __device__ __forceinline__ void load_bounds(const SelectArgs& a, Bounds& to, int page, int h, int g) {
    const O* src = reinterpret_cast<const O*>(a.bounds) + ((int64_t)max(page, 0) * a.p.kv_heads + h) * 2 * a.p.head_dim;
#pragma unroll
    for (int y = 0; y < 2; ++y)
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int d = 8 * (4 * c + g);
        __builtin_memcpy(to.x[y][c], __builtin_assume_aligned(src + y * a.p.head_dim + (d < a.p.head_dim ? d : 0), 16),
                         sizeof(to.x[y][c]));
      }
  }
  // (the dims behind head_dim, whose query is 0, were loaded from others, which need not be finite)
  static __device__ __forceinline__ void cut(const SelectArgs& a, Bounds& to, int g) {
    if (a.p.head_dim == DHP) return;
#pragma unroll
    for (int c = 0; c < NC; ++c)
      if (8 * (4 * c + g) >= a.p.head_dim) __builtin_memset(to.x[0][c], 0, sizeof(to.x[0][c])), __builtin_memset(to.x[1][c], 0, sizeof(to.x[1][c]));
  }
  // Two values, converted where they are used: all at once, ahead of the products, they would take up to 256 registers.
  static __device__ __forceinline__ void two(const O* x, double (&f)[2]) {
    uint32_t w[sizeof(O) / 2];
    __builtin_memcpy(w, x, 2 * sizeof(O));
#pragma unroll
    for (int i = 0; i < (int)(sizeof(O) / 2); ++i) asm volatile("" : "+v"(w[i]));
    if constexpr (sizeof(O) == 2)
      f[0] = (double)__uint_as_float(w[0] << 16), f[1] = (double)__uint_as_float(w[0] & 0xffff0000u);
    else
      f[0] = (double)__uint_as_float(w[0]), f[1] = (double)__uint_as_float(w[1]);
  }
  // the largest rank over the heads of block 4 (r / 4) + g
  static __device__ __forceinline__ uint32_t rank(const Bounds& k, const Query& q, int r, int g) {
    constexpr int PARTS = NG == 1 ? 4 : 1;  // sums that do not wait for each other (of the heads and halves, too)
    double sum[NG][2][PARTS] = {};
    // the queries of four dims, read a step ahead
    auto read = [&](double2 (&f)[NG][2][2], int step) {
#pragma unroll
      for (int y = 0; y < NG; ++y)
#pragma unroll
        for (int z = 0; z < 2; ++z)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            f[y][z][i] = *reinterpret_cast<const double2*>(&q.x[z][4 * y + (r & 3)][8 * (4 * (step >> 1) + g) + 4 * (step & 1) + 2 * i]);
    };
    double2 f[2][NG][2][2];
    read(f[0], 0);
#pragma unroll
    for (int step = 0; step < 2 * NC; ++step) {
      if (step + 1 < 2 * NC) read(f[(step + 1) & 1], step + 1);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int c = step >> 1, e = 4 * (step & 1) + 2 * i;
        double bound[2][2];
        two(&k.x[0][c][e], bound[0]), two(&k.x[1][c][e], bound[1]);
#pragma unroll
        for (int y = 0; y < NG; ++y)
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            const double2 v = f[step & 1][y][z][i];
            double& s0 = sum[y][z][(2 * i) % PARTS];
            s0 = __builtin_amdgcn_mfma_f64_4x4x4f64(bound[z][0], v.x, s0, 0, 0, 0);
            double& s1 = sum[y][z][(2 * i + 1) % PARTS];
            s1 = __builtin_amdgcn_mfma_f64_4x4x4f64(bound[z][1], v.y, s1, 0, 0, 0);
          }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    uint32_t best = 0;
#pragma unroll
    for (int y = 0; y < NG; ++y) {
      double all = 0.0;
#pragma unroll
      for (int z = 0; z < 2; ++z)
#pragma unroll
        for (int i = 0; i < PARTS; ++i) all += sum[y][z][i];
      best = max(best, rank_of((float)all));
    }
    best = max(best, (uint32_t)__shfl_xor((int)best, 1, 64));
    return max(best, (uint32_t)__shfl_xor((int)best, 2, 64));
  }

  // Ranks of the tiles first, first + step .. up to `tiles` of a (sequence, key head) into rank_out[]: 0 for the blocks that
  // are always kept and, to the end of a tile, for those that are not there.  All threads of the workgroup call it.  ONE: a
  // wavefront has one tile at most (shorter code, fewer registers).
  template <int THREADS, bool ONE>
  static __device__ __forceinline__ void run(const SelectArgs& a, Query& q, int b, int h, int blocks, int first, int step,
                                             int tiles, int lane, uint32_t* rank_out) {
    const int r = lane & 15, g = lane >> 4;
    auto page_at = [&](int t) { return a.p.page_of(b, (int64_t)min(16 * t + r, blocks - 1) << a.p.shift); };
    for (int i = 0; i < a.group; i += HEADS) {
      Bounds now, next;
      int page = page_at(first), next_page = ONE ? 0 : page_at(first + step);
      if (first < tiles) load_bounds(a, now, page, h, g);
      if (i > 0) __syncthreads();
      load_query<THREADS>(a, q, b, h, i);
      __syncthreads();
      if (first >= tiles) continue;
      auto put = [&](int t) {
        cut(a, now, g);
        uint32_t best = rank(now, q, r, g);
        if (page < 0 && g == 0) kv_flag(a.err);
        const int mine = 16 * t + 4 * (r >> 2) + g;
        if (__shfl(page, 4 * (r >> 2) + g, 64) < 0) best = NO_PAGE;
        if (mine < a.first || mine >= blocks - a.recent) best = 0;
        if ((r & 3) == 0) rank_out[mine] = i > 0 ? max(best, rank_out[mine]) : best;
      };
      int t = first;
      for (; !ONE && t + step < tiles; t += step) {  // (the last tile apart: nothing to load beside it)
        const int page_after = page_at(t + 2 * step);
        load_bounds(a, next, next_page, h, g);
        put(t);
        now = next;
        page = next_page;
        next_page = page_after;
      }
      put(t);
    }
  }
};

template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_or_0(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);
}
// Sums over this lane and those before it.
__device__ __forceinline__ int scan64(int v) {
  v += dpp_or_0<0x111, 0xF>(v);
  v += dpp_or_0<0x112, 0xF>(v);
  v += dpp_or_0<0x114, 0xF>(v);
  v += dpp_or_0<0x118, 0xF>(v);
  v += dpp_or_0<0x142, 0xA>(v);  // the last lane of a row of 16 to the row behind it
  v += dpp_or_0<0x143, 0xC>(v);  // and of the first half to the second
  return v;
}
__device__ __forceinline__ uint32_t wave_most(uint32_t x) {
  auto more = [](uint32_t p, int q) { return max(p, (uint32_t)q); };
  x = more(x, dpp_or_0<0x111, 0xF>((int)x));
  x = more(x, dpp_or_0<0x112, 0xF>((int)x));
  x = more(x, dpp_or_0<0x114, 0xF>((int)x));
  x = more(x, dpp_or_0<0x118, 0xF>((int)x));
  x = more(x, dpp_or_0<0x142, 0xA>((int)x));
  x = more(x, dpp_or_0<0x143, 0xC>((int)x));
  return (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
}

constexpr int PK_FEW = 64;  // ranks that are compared with each other

template <int WAVES, int KPT>
struct PickShared {
  int hist[64 * WAVES];
  uint32_t most[WAVES], least[WAVES];
  int part[KPT * WAVES], part2[WAVES];
  int picked[3], few;
  uint2 list[PK_FEW];
};

// How many flags there are before each of this thread's: flag i of thread t is the (i * threads + t)-th.  Returns how many
// there are in all; flags from `rounds` rounds on are not looked at.
template <int WAVES, int N>
__device__ __forceinline__ int before_of(const bool (&flag)[N], int (&before)[N], int rounds, int* part, int lane, int wid) {
  uint64_t m[N];
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < rounds) {
      m[i] = __ballot(flag[i]);
      if (lane == 0) part[i * WAVES + wid] = __popcll(m[i]);
    }
  __syncthreads();
  int sum = 0;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < rounds) {
      before[i] = sum + __popcll(m[i] & ((1ull << lane) - 1));
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        const int v = part[i * WAVES + w];
        if (w < wid) before[i] += v;
        sum += v;
      }
    }
  return sum;
}

// The pages of the a.count blocks to keep, in their order, from the ranks of the blocks tid, tid + threads .. (0: always
// kept, or not there).  The ranks are counted in as many bins as there are threads, even parts of their range; the bin
// that holds the last one kept is found from the counts, and its ranks, where they are few, are compared with each other
// by every wavefront for itself.  Where they are many the bin is cut into bins again.
template <int WAVES, int KPT>
__device__ __forceinline__ void pick(const SelectArgs& a, const uint32_t (&key)[KPT], int blocks, const int32_t (&page)[KPT],
                                     int32_t* out, PickShared<WAVES, KPT>& s) {
  constexpr int BINS = 64 * WAVES;
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int rounds = (blocks + BINS - 1) / BINS;
  int need = a.count - a.first - a.recent;
  bool keep[KPT], open[KPT];  // open: not decided yet
  int before[KPT];
#pragma unroll
  for (int i = 0; i < KPT; ++i) {
    const int at = i * BINS + tid;
    open[i] = need > 0 && key[i] != 0;
    keep[i] = at < blocks && (at < a.first || at >= blocks - a.recent);
  }
  while (need > 0) {  // (the same for all threads)
    uint32_t most = 0, least = 0;  // the largest rank, and of the inverted ranks
#pragma unroll
    for (int i = 0; i < KPT; ++i)
      if (i < rounds && open[i]) most = max(most, key[i]), least = max(least, ~key[i]);
    most = wave_most(most), least = wave_most(least);
    if (lane == 0) s.most[wid] = most, s.least[wid] = least;
    s.hist[tid] = 0;
    if (tid == 0) s.few = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) most = max(most, s.most[w]), least = max(least, s.least[w]);
    const uint32_t low = ~least, range = most - low;
    if (range == 0) {  // one rank for all: the lower blocks
      before_of<WAVES, KPT>(open, before, rounds, s.part, lane, wid);
#pragma unroll
      for (int i = 0; i < KPT; ++i) keep[i] = keep[i] || (i < rounds && open[i] && before[i] < need);
      break;
    }
    // (conversion, product and truncation keep the order)
    const float scale = (float)BINS / ((float)range + 1.0f);
    int bin[KPT];
#pragma unroll
    for (int i = 0; i < KPT; ++i) {
      bin[i] = min((int)((float)(key[i] - low) * scale), BINS - 1);
      if (i < rounds && open[i]) atomicAdd(&s.hist[bin[i]], 1);
    }
    __syncthreads();
    const int mine = s.hist[BINS - 1 - tid], upto = scan64(mine);
    if (lane == 63) s.part2[wid] = upto;
    __syncthreads();
    int above = upto - mine;
#pragma unroll
    for (int w = 0; w < WAVES; ++w)
      if (w < wid) above += s.part2[w];
    if (above < need && above + mine >= need) s.picked[0] = BINS - 1 - tid, s.picked[1] = above, s.picked[2] = mine;
    // (fewer ranks than are needed: lengths that were written to during the call; all of them, so that the rounds end)
    if (tid == BINS - 1 && above + mine < need) s.picked[0] = 0, s.picked[1] = need - mine, s.picked[2] = mine;
    __syncthreads();
    const int last = s.picked[0], many = s.picked[2];
    need -= s.picked[1];
    const bool whole = need == many;
#pragma unroll
    for (int i = 0; i < KPT; ++i) {
      keep[i] = keep[i] || (open[i] && (whole ? bin[i] >= last : bin[i] > last));
      open[i] = open[i] && !whole && bin[i] == last;
    }
    if (whole) break;
    if (many > PK_FEW) continue;
#pragma unroll
    for (int i = 0; i < KPT; ++i)
      if (i < rounds && open[i]) s.list[atomicAdd(&s.few, 1)] = make_uint2(key[i], (uint32_t)(i * BINS + tid));
    __syncthreads();
    const uint2 own = lane < many ? s.list[lane] : make_uint2(0, 0);
    int ahead = 0;  // those before this one: of higher rank, or of the same and a lower block
    for (int i = 0; i < many; ++i) {
      const uint32_t x = (uint32_t)__builtin_amdgcn_readlane((int)own.x, i), y = (uint32_t)__builtin_amdgcn_readlane((int)own.y, i);
      ahead += x > own.x || (x == own.x && y < own.y);
    }
    const int at = __builtin_ctzll(__ballot(lane < many && ahead == need - 1));
    const uint32_t x = (uint32_t)__builtin_amdgcn_readlane((int)own.x, at), y = (uint32_t)__builtin_amdgcn_readlane((int)own.y, at);
#pragma unroll
    for (int i = 0; i < KPT; ++i)
      keep[i] = keep[i] || (open[i] && (key[i] > x || (key[i] == x && (uint32_t)(i * BINS + tid) <= y)));
    break;
  }
  __syncthreads();
  before_of<WAVES, KPT>(keep, before, rounds, s.part, lane, wid);
#pragma unroll
  for (int i = 0; i < KPT; ++i)
    if (i < rounds && keep[i] && before[i] < a.keep) out[before[i]] = page[i];
}

// The pages of this thread's blocks, loaded before it is known which of them are there.
template <int THREADS, int KPT>
__device__ __forceinline__ void load_pages(const SelectArgs& a, const int32_t* pages, int32_t (&page)[KPT]) {
  const int width = (int)(a.p.max_slots >> a.p.shift);
#pragma unroll
  for (int i = 0; i < KPT; ++i) {
    const int at = i * THREADS + threadIdx.x;
    page[i] = at < width ? pages[at] : -1;
  }
}

// What a selection writes beside the pages chosen; true where all blocks are kept and nothing is left to do.
__device__ __forceinline__ bool begin_select(const SelectArgs& a, int b, int h, int64_t n, bool ok, int blocks,
                                             const int32_t* pages, int32_t* out) {
  const int tid = threadIdx.x, kept = min(blocks, a.keep);
  if (h == 0 && tid == 0) {
    if (!ok) kv_flag(a.err);
    a.new_lengths[b] = n - ((int64_t)(blocks - kept) << a.p.shift);
  }
  for (int i = kept + tid; i < a.keep; i += blockDim.x) out[i] = -1;
  if (blocks > a.count) return false;
  for (int i = tid; i < blocks; i += blockDim.x) {
    out[i] = pages[i];
    if ((uint32_t)pages[i] >= (uint32_t)a.p.num_pages) kv_flag(a.err);
  }
  return true;
}

// Ranks and selection in one: a workgroup a (sequence, key head) of up to KPT * THREADS blocks.  32 sequences of 10 .. 501
// blocks, 32 query on 8 key heads x 128 in bf16, 33 MB: 16.4 us; 13.5 with ranks that take no product or conversion (by count
// those are 6.3 us of the longest sequences' CUs, whose wavefronts have four tiles each where the mean is two; the loads beside them
// are not faster), 14.8 without the selection.  The same blocks of int8 pages, 66 MB, 22.6 us; 12 heads of 64 in fp32, 50 MB, 21.9;
// 38 blocks of 8 heads x 64 in bf16 5.0.
template <class O, class Q, int DHP, int NG, int THREADS, int KPT, bool ONE>
__global__ __launch_bounds__(THREADS) void kv_rank_select_kernel(SelectArgs a) {
  constexpr int WAVES = THREADS / 64;
  typedef Scores<O, Q, DHP, NG> S;
  __shared__ __attribute__((aligned(16))) uint32_t rank[THREADS * KPT];
  __shared__ __attribute__((aligned(16))) typename S::Query query;
  __shared__ __attribute__((aligned(16))) PickShared<WAVES, KPT> s;
  const int b = blockIdx.x / a.p.kv_heads, h = blockIdx.x - b * a.p.kv_heads;
  const int tid = threadIdx.x, lane = tid & 63, wid = wave_uniform(tid >> 6);
  bool ok = true;
  const int64_t n = a.p.length_of(a.lengths, b, a.max_length, &ok);
  const int blocks = blocks_of(a, n);
  const int32_t* pages = a.p.table + b * a.p.ld_table;
  int32_t* out = a.table + (int64_t)blockIdx.x * a.keep;
  if (begin_select(a, b, h, n, ok, blocks, pages, out)) return;
  const int tiles = (blocks + 15) >> 4;
  int32_t page[KPT];
  load_pages<THREADS>(a, pages, page);
  S::template run<THREADS, ONE>(a, query, b, h, blocks, wid, WAVES, tiles, lane, rank);
  __syncthreads();
  uint32_t key[KPT];
#pragma unroll
  for (int i = 0; i < KPT; ++i)  // (behind the last tile nothing was written)
    key[i] = i * THREADS + tid < tiles * 16 ? rank[i * THREADS + tid] : 0;
  pick<WAVES, KPT>(a, key, blocks, page, out, s);
}

// Tiles a wavefront where there are few and where there are many, from RK_MANY a CU on (us, 1 / 4: 8 units of 2048 blocks
// 13.7 / 18.6, 128 42.7 / 42.8, 512 158 / 135)
constexpr int RK_MORE = 4, RK_MANY = 64;

// The ranks alone: `per` tiles of a (sequence, key head) a workgroup.  2048 blocks of 32 query on 8 key heads x 128, 8.4 MB: 6.7 us,
// the chain length -> table -> bounds -> products of one tile.
template <class O, class Q, int DHP, int NG, bool ONE>
__global__ __launch_bounds__(256) void kv_rank_kernel(SelectArgs a, int per) {
  typedef Scores<O, Q, DHP, NG> S;
  __shared__ __attribute__((aligned(16))) typename S::Query query;
  const int lane = threadIdx.x & 63, wid = wave_uniform((int)threadIdx.x >> 6);
  const int units = a.B * a.p.kv_heads, chunk = blockIdx.x / units, bh = blockIdx.x - chunk * units;
  const int b = bh / a.p.kv_heads, h = bh - b * a.p.kv_heads;
  bool ok = true;
  const int blocks = blocks_of(a, a.p.length_of(a.lengths, b, a.max_length, &ok));
  const int tiles = min((blocks + 15) >> 4, per * (chunk + 1));
  if (blocks <= a.count || per * chunk >= tiles) return;  // (all of them are kept, or there are none for this workgroup)
  S::template run<256, ONE>(a, query, b, h, blocks, per * chunk + wid, 4, tiles, lane, a.rank + (int64_t)bh * a.ld);
}

// The selection from ranks in the workspace.  2048 blocks: 5.8 us, a launch and the rounds between its barriers.
template <int THREADS, int KPT>
__global__ __launch_bounds__(THREADS) void kv_select_kernel(SelectArgs a) {
  constexpr int WAVES = THREADS / 64;
  __shared__ __attribute__((aligned(16))) PickShared<WAVES, KPT> s;
  const int b = blockIdx.x / a.p.kv_heads, h = blockIdx.x - b * a.p.kv_heads;
  const int tid = threadIdx.x;
  // ranks and pages beside the length that says which of them count
  const uint32_t* rank = a.rank + (int64_t)blockIdx.x * a.ld;
  uint32_t key[KPT];
#pragma unroll
  for (int i = 0; i < KPT; ++i) key[i] = i * THREADS + tid < a.ld ? rank[i * THREADS + tid] : 0;
  const int32_t* pages = a.p.table + b * a.p.ld_table;
  int32_t page[KPT];
  load_pages<THREADS>(a, pages, page);
  bool ok = true;
  const int64_t n = a.p.length_of(a.lengths, b, a.max_length, &ok);
  const int blocks = blocks_of(a, n);
  int32_t* out = a.table + (int64_t)blockIdx.x * a.keep;
  if (begin_select(a, b, h, n, ok, blocks, pages, out)) return;
#pragma unroll
  for (int i = 0; i < KPT; ++i)
    if (i * THREADS + tid >= ((blocks + 15) & ~15)) key[i] = 0;  // (behind the last tile nothing was written)
  pick<WAVES, KPT>(a, key, blocks, page, out, s);
}

constexpr int SL_THREADS = 1024, SL_KEYS = 16;  // of the largest selection that keeps its ranks in registers

// The selection of more blocks than that: a radix selection of a byte a round, the ranks read again in each.  20,000 blocks of 8
// key heads: 53.5 us beside 20.3 for the ranks (82 MB); 8192 by the one above 26.2 beside 10.4.
__global__ __launch_bounds__(SL_THREADS) void kv_select_long_kernel(SelectArgs a) {
  constexpr int WAVES = SL_THREADS / 64;
  __shared__ __attribute__((aligned(16))) int hist[256];
  __shared__ int part[2][WAVES];
  __shared__ int picked[3];
  const KvPages& p = a.p;
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int b = blockIdx.x / p.kv_heads, h = blockIdx.x - b * p.kv_heads;
  bool ok = true;
  const int64_t n = p.length_of(a.lengths, b, a.max_length, &ok);
  const int blocks = blocks_of(a, n);
  const int32_t* pages = p.table + b * p.ld_table;
  int32_t* out = a.table + (int64_t)blockIdx.x * a.keep;
  if (begin_select(a, b, h, n, ok, blocks, pages, out)) return;
  const uint32_t* rank = a.rank + (int64_t)blockIdx.x * a.ld;
  uint32_t found = 0;
  int need = a.count - a.first - a.recent;
  bool whole = need == 0;
  if (whole) found = 0xffffffffu;
  for (int shift = 24; shift >= 0 && !whole; shift -= 8) {
    __syncthreads();
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int i = tid; i < blocks; i += SL_THREADS) {
      const uint32_t x = rank[i];
      if (x != 0 && (shift == 24 || (x >> (shift + 8)) == (found >> (shift + 8)))) atomicAdd(&hist[(x >> shift) & 255], 1);
    }
    __syncthreads();
    if (wid == 0) {  // lane l has the bins 252 - 4 l .. 255 - 4 l
      const int4 c = *reinterpret_cast<const int4*>(&hist[252 - 4 * lane]);
      const int many[4] = {c.w, c.z, c.y, c.x};  // the largest ranks first
      const int sum = (c.x + c.y) + (c.z + c.w);
      int before = scan64(sum) - sum;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (before < need && before + many[i] >= need)  // (one bin of one lane)
          picked[0] = 255 - 4 * lane - i, picked[1] = before, picked[2] = many[i];
        before += many[i];
      }
      // (fewer ranks than are needed: lengths that were written to during the call)
      if (lane == 63 && before < need) picked[0] = 0, picked[1] = need - many[3], picked[2] = many[3];
    }
    __syncthreads();
    found |= (uint32_t)picked[0] << shift;
    need -= picked[1];
    whole = need == picked[2];  // all that share the bytes found are kept
  }
  // ranks above `found`, and of those equal to it the first `need`: in the order of the blocks
  int at = 0, tie = 0;
  const bool none = a.count == a.first + a.recent;
  for (int i0 = 0; i0 < blocks; i0 += SL_THREADS) {
    const int i = i0 + tid;
    const uint32_t x = i < blocks ? rank[i] : 0;
    bool keep[1] = {i < blocks && (i < a.first || i >= blocks - a.recent)}, equal[1] = {!whole && x != 0 && x == found};
    keep[0] = keep[0] || (!none && x != 0 && (whole ? x >= found : x > found));
    int before[1];
    const int ties = before_of<WAVES, 1>(equal, before, 1, part[0], lane, wid);
    keep[0] = keep[0] || (equal[0] && tie + before[0] < need);
    tie += ties;
    const int kept = before_of<WAVES, 1>(keep, before, 1, part[1], lane, wid), to = at + before[0];
    at += kept;
    if (keep[0] && to < a.keep) out[to] = pages[i];
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
  if (B == 0) return OK;
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
  const int64_t need = cdiv(blocks * pages->kv_heads, 4), share = cdiv((int64_t)cu_count() * KB_PER_CU, B);
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

// Ranks and selection in one launch, or in two: one workgroup has all blocks of a (sequence, key head), but two launches
// begin twice.  us in a graph, 64 / 128 / 256 / 512 / 1024 blocks of 32 query on 8 key heads x 128 in bf16:
//               512 threads               256 threads               two launches
//     8 units    6.4  8.0 12.3 17.0 27.5   6.7  9.5 13.0 18.2 30.3   9.0 10.1 10.5 10.8 10.0
//   128 units    6.7  8.4 12.6 18.2 29.3   6.9  9.9 13.4 21.3 34.5   9.3 10.6 12.2 16.2 24.1
//   192 units    6.7  8.5 12.9 18.8 29.9   7.1  9.9 13.5 21.8 34.9   9.4 11.8 13.5 20.7 29.9
//   256 units    6.6  8.7 13.5 20.5 31.7   7.0  9.9 14.2 22.3 35.5   9.5 12.0 16.0 23.7 36.8
//  1024 units   16.0 22.1 48.8 70.6  131  12.0 24.2 37.5 62.3  125  15.7 25.2 38.3 61.5  128
// The rule goes by units and blocks alone.  Where a tile costs less than in this form one launch would go further, where it
// costs more less far (128 / 192 / 256 blocks, 512 threads against two launches):
//   one query head a key head, 64 dims in bf16    8 units  6.0  6.9  8.2 /  8.0  8.6  8.7   128 units  6.2  7.5  8.6 /  8.4  9.9 10.6
//   the same in fp32                             12 units  6.3  7.9  9.4 /  8.5  8.9  9.3   120 units  6.7  8.4  9.9 /  8.7 10.4 10.9
//   eight heads, 128 dims in int8                 8 units 10.6 13.5 17.1 / 11.8 12.1 12.2   128 units 11.3 14.9 18.1 / 12.4 14.7 15.5
//   sixteen, 128 dims in bf16                     8 units 12.4 15.6 18.7 / 12.7 13.2 11.6   128 units 13.0 16.3 19.3 / 13.5 16.4 16.5
constexpr int FUSED_ALWAYS = 192, FUSED_KEYS = 4;  // blocks of any number of units; blocks a thread
enum class Form { two, one_256, one_512 };
Form select_form(int64_t units, int64_t ld) {
  const int64_t cus = cu_count();
  if (ld > 512 * FUSED_KEYS || (ld > FUSED_ALWAYS && 4 * units < 3 * cus)) return Form::two;
  return units > cus && ld <= 256 * FUSED_KEYS ? Form::one_256 : Form::one_512;
}

template <class O, class Q, int DHP, int NG, int THREADS>
void launch_one(const SelectArgs& a, dim3 units, hipStream_t stream) {
  // (the code for one block a thread is shorter: 38 blocks 6.2 -> 5.3 us, up to 501 17.1 -> 16.2)
  if (a.ld <= THREADS / 4)
    hipLaunchKernelGGL((kv_rank_select_kernel<O, Q, DHP, NG, THREADS, 1, true>), units, dim3(THREADS), 0, stream, a);
  else if (a.ld <= THREADS)
    hipLaunchKernelGGL((kv_rank_select_kernel<O, Q, DHP, NG, THREADS, 1, false>), units, dim3(THREADS), 0, stream, a);
  else
    hipLaunchKernelGGL((kv_rank_select_kernel<O, Q, DHP, NG, THREADS, FUSED_KEYS, false>), units, dim3(THREADS), 0, stream, a);
}
template <class O, class Q, int DHP, int NG>
int launch_select(const SelectArgs& a, hipStream_t stream) {
  const int64_t n = (int64_t)a.B * a.p.kv_heads;
  const dim3 units((unsigned)n);
  const Form form = select_form(n, a.ld);
  if (form != Form::two) {
    if (form == Form::one_256)
      launch_one<O, Q, DHP, NG, 256>(a, units, stream);
    else
      launch_one<O, Q, DHP, NG, 512>(a, units, stream);
    CORTEX_CHECK_LAUNCH("kv_rank_select_kernel");
    return OK;
  }
  const int per_wave = n * a.ld / 16 >= RK_MANY * cu_count() ? RK_MORE : 1, chunks = (int)cdiv(a.ld, 64 * per_wave);
  if (per_wave == 1)
    hipLaunchKernelGGL((kv_rank_kernel<O, Q, DHP, NG, true>), dim3((unsigned)(n * chunks)), dim3(256), 0, stream, a, 4);
  else
    hipLaunchKernelGGL((kv_rank_kernel<O, Q, DHP, NG, false>), dim3((unsigned)(n * chunks)), dim3(256), 0, stream, a, 4 * per_wave);
  CORTEX_CHECK_LAUNCH("kv_rank_kernel");
  // The smallest that holds the ranks; the next one instead, ranks and selection of 8 units (us): 1024 blocks 10.1 -> 11.2, 2048
  // 12.4 -> 13.9, 4096 16.7 -> 27.6.  Ranks read again in each round instead of held: 16,384 blocks whose scores differ by
  // little 47.7 -> 72.0, that are all alike 49 -> 93, but with independent bounds 56.1 -> 53.1, and 9000 of those 43.7 -> 34.3
  if (a.ld <= 1024)
    hipLaunchKernelGGL((kv_select_kernel<256, 4>), units, dim3(256), 0, stream, a);
  else if (a.ld <= 2048)
    hipLaunchKernelGGL((kv_select_kernel<512, 4>), units, dim3(512), 0, stream, a);
  else if (a.ld <= 4096)
    hipLaunchKernelGGL((kv_select_kernel<1024, 4>), units, dim3(1024), 0, stream, a);
  else if (a.ld <= SL_THREADS * SL_KEYS)
    hipLaunchKernelGGL((kv_select_kernel<SL_THREADS, SL_KEYS>), units, dim3(SL_THREADS), 0, stream, a);
  else
    hipLaunchKernelGGL(kv_select_long_kernel, units, dim3(SL_THREADS), 0, stream, a);
  CORTEX_CHECK_LAUNCH("kv_select_kernel");
  return OK;
}
// Fours of query heads at a time: as many as there are, up to 16 heads.  (Eight heads as sixteen: 256 blocks 15.1 us instead of
// 11.7, int8 18.8 and 13.3; sixteen as twice eight: the same in bf16, fp32 of 64 dims 13.7 instead of 11.9, fp32 bounds of 128 dims
// 20.0 instead of 19.6 although those spill 47 of 256 registers.)
template <class O, class Q, int DHP>
int launch_select(const SelectArgs& a, hipStream_t stream) {
  if (a.group <= 4) return launch_select<O, Q, DHP, 1>(a, stream);
  return a.group <= 8 ? launch_select<O, Q, DHP, 2>(a, stream) : launch_select<O, Q, DHP, 4>(a, stream);
}
template <class O, class Q>
int launch_select(const SelectArgs& a, hipStream_t stream) {
  return a.p.head_dim <= 64 ? launch_select<O, Q, 64>(a, stream) : launch_select<O, Q, 128>(a, stream);
}

}  // namespace
}  // namespace cortex

extern "C" int64_t cortex_kv_select_workspace_bytes(const cortex_kv_pages* pages, int64_t B, int64_t max_length,
                                                    int64_t count) {
  if (!pages || pages->page_size < 1 || pages->kv_heads < 1 || B < 0 || max_length < 0 || count < 0) return 0;
  const int64_t units = B * pages->kv_heads, ld = rank_ld(pages, max_length, count);
  return select_form(units, ld) == Form::two ? units * ld * 4 : 0;
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
  // (a launch has fewer than 2^32 threads; and the sizes of what the call writes fit 64 bits then)
  CORTEX_CHECK_ARG(B <= 0xffffffffLL / 1024 / pages->kv_heads &&
                       (ld == 0 || B * pages->kv_heads <= 0xffffffffLL / 256 / cdiv(ld, 64)),
                   "%s: %lld sequences of up to %lld blocks are too much for one call", who, (long long)B, (long long)blocks);
  CORTEX_CHECK_ARG(table || keep == 0, "%s: null table", who);
  // what the call writes is read by no workgroup of it, and written once
  struct Rows {  // `n` of `size` bytes, from one to the next `pitch` >= 0
    const char* name;
    __int128 at, n, pitch, size;
  };
  auto whole = [](const char* name, const void* p, __int128 size) {
    return Rows{name, (__int128)(uintptr_t)p, p && size > 0, 0, size};
  };
  auto strided = [](const char* name, __int128 at, int64_t n, __int128 pitch, __int128 size) {
    return pitch < 0 ? Rows{name, at + (n - 1) * pitch, n, -pitch, size} : Rows{name, at, n, pitch, size};
  };
  auto meet = [](const Rows& x, const Rows& one) {
    if (x.n == 0 || one.n == 0) return false;
    const __int128 past = one.at - x.at - x.size;  // the first row that ends behind one's begin
    const __int128 i = past < 0 ? 0 : x.pitch == 0 ? x.n : past / x.pitch + 1;
    return i < x.n && x.at + i * x.pitch < one.at + one.size;
  };
  auto queries = [&] {  // rows of the larger stride; the other one within them
    const __int128 sb = (__int128)q_sb * es, sh = (__int128)q_sh * es, b = sb < 0 ? -sb : sb, h = sh < 0 ? -sh : sh;
    const bool by_b = b >= h;
    const __int128 in = by_b ? (heads - 1) * sh : (B - 1) * sb, dims = pages->head_dim * es;
    return strided("the queries", (__int128)(uintptr_t)q + (in < 0 ? in : 0), by_b ? B : heads, by_b ? sb : sh, (in < 0 ? -in : in) + dims);
  };
  const int64_t need = cortex_kv_select_workspace_bytes(pages, B, a.max_length, count);
  const Rows read[] = {
      whole("lengths", lengths, 8 * B),
      strided("the block table", (uintptr_t)block_table, max_pages ? B : 0, B > 1 ? (__int128)ld_table * 4 : 0, 4 * max_pages), queries(),
      whole("the bounds", pages->bounds, (__int128)pages->num_pages * pages->kv_heads * 2 * pages->head_dim * bound_bytes_of(pages))};
  const Rows made[] = {whole("new_lengths", new_lengths, 8 * B), whole("table", table, 4 * B * pages->kv_heads * keep),
                       whole("the workspace", workspace, need)};
  auto check_apart = [&](int i) {
    for (const Rows& x : read)
      CORTEX_CHECK_ARG(!meet(x, made[i]), "%s: %s may not overlap %s", who, made[i].name, x.name);
    for (int j = 0; j < i; ++j)
      CORTEX_CHECK_ARG(!meet(made[j], made[i]), "%s: %s may not overlap %s", who, made[i].name, made[j].name);
    return OK;
  };
  if (int rc = check_apart(0)) return rc;
  if (int rc = check_apart(1)) return rc;
  CORTEX_CHECK_ARG((workspace || need == 0) && (uintptr_t)workspace % 16 == 0, "%s: null or unaligned workspace", who);
  if (workspace_bytes < need) {
    set_error("%s: workspace of %lld bytes, %lld needed", who, (long long)workspace_bytes, (long long)need);
    return E_WORKSPACE;
  }
  if (int rc = check_apart(2)) return rc;
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
  if (ld == 0) {  // all blocks are kept
    hipLaunchKernelGGL((kv_select_kernel<256, 4>), dim3((unsigned)(B * pages->kv_heads)), dim3(256), 0, stream, a);
    CORTEX_CHECK_LAUNCH("kv_select_kernel");
    return OK;
  }
  if (pages->dtype == DT_F32) return launch_select<float, float>(a, stream);
  if (pages->dtype == DT_BF16) return launch_select<bf16, bf16>(a, stream);
  return launch_select<float, bf16>(a, stream);
}
