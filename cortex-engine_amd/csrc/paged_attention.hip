// Attention of one new token per sequence over its paged keys and values.
//
//   s_j = scale q . k_j   m = max_j s_j   p_j = exp(s_j - m)   l = sum_j p_j   out = sum_j p_j v_j / l
//
// Every key and value row is read once, for all query heads of its key head: a streaming kernel, bound by HBM as long
// as enough bytes are in flight.  The G query heads of a key head are the columns of the matrix products (16 at a time; 16
// are multiplied also where there are fewer, which the matrix cores have the time for).
//
// A wavefront takes tiles of 32 keys.  Both operands come straight from memory into registers, without LDS:
//   scores  S^T = K Q^T: lane (r, g) = (l % 16, l / 16) loads its part of key row key_of(st, r) = 8 (r / 4) + 4 st + r % 4
//           for st 0 and 1; the score registers of group g are then the 8 consecutive keys 8 g .. 8 g + 7;
//   output  O^T += V^T P^T: P^T of those 8 keys is the B operand as it stands.  For V^T lane (r, g) loads the same 8
//           keys at E = DHP / 16 consecutive dims r E .. r E + E - 1, so a row is read whole by 16 lanes; the transpose is
//           one byte permute per register, and product j gives the dims {r E + j}.
// K's registers are free after the scores and V's after the output: the next tile's loads are issued there.
//
// Split over the length: all tiles of all (sequence, key head) units are laid end to end and cut into equal shares, one a
// workgroup, from the lengths on the device (a replayed graph follows them, ragged batches need no plan, and the grid
// is one workgroup per slot of the card).  A unit cut by a share leaves its running (m, l, sum p v) in the workspace, at
// most two a workgroup (the end of a unit and the beginning of another), and a second launch joins them in order.
//
// Measured (bf16, 32 query heads on 8 key heads of 128): one sequence of 131,072 keys, 537 MB, 95 us, 5.7 TB/s; 32 of 150
// .. 8003 keys, 535 MB, 99 us.  Int8, 135 MB, 32 us, 4.2 TB/s: the VALU, widening among others, is busy 58 % of the time (8.4 of
// 28.9 M wavefront cycles, two wavefronts a SIMD), 45 % of a wavefront's is waiting, and two workgroups a CU have half the bytes
// of bf16 in flight.  fp32, 12 heads of 64, 885 MB, 159 us, 5.6 TB/s.  With the weights, 16 of 2048 .. 4160 keys: 47 us, 42
// without storing the scores.
#include <hip/hip_runtime.h>

#include "paged_kv.h"

namespace cortex {
namespace {

constexpr int PA_KT = 32;       // keys of one matrix product
constexpr int PA_WAVES = 4;     // wavefronts of a workgroup that takes a share
constexpr int PA_MORE = 8;      // and of one that has a CU to itself and takes a whole unit
constexpr int PA_ROWS = 16;     // query heads of one matrix product
constexpr int PA_MIN_TILES = PA_WAVES;  // tiles of a share
// Workgroups that a CU holds at once, by the registers of a form that takes shares: 128 dims 168 (int8) to 249, fp32 242 to
// 256 and where head_dim < 128 spills 5, 13 with the weights (not measured apart); 64 dims in fp32 146 to 159, in fewer bits 115
// to 119 and for two products 157 to 163.  (64 sequences of 500 .. 3000 keys x 64 dims, bf16: 2 a CU 55.5 us, 4 54.2; bf16, 128
// dims as 3: 105 -> 110.  Int8 of 128 dims would go in three times; not tried)
__host__ __device__ constexpr int per_cu(int dhp, int es, int rt) { return dhp == 128 ? 2 : es == 4 || rt == 2 ? 3 : 4; }
constexpr int PA_MAX_SHARES = 1024;
// What it costs to begin a unit (fill and drain the loads, sum up), in tiles, where a share may have PA_LONG tiles and
// where it has fewer: without it the shares with many short sequences are the last to end (32 sequences of 150 .. 8003
// keys: 0 118 us, 2 107, 4 107, 8 104.6; 8 of 101 .. 2049 in fp32: 0 22.2, 2 20.6, 4 20.1, 8 21.7; one of 8192: 0 16.8, 2 18)
constexpr int PA_LONG = 16, PA_BEGIN_LONG = 8, PA_BEGIN_SHORT = 2;
// Length up to which a workgroup takes a whole unit, and where there are units for every CU (us, shares against whole units:
// 600 keys, 8 units of 64 dims 14.2 / 10.0; 1000, 64 units of 128 17.3 / 14.6; 2048, 8 units of 128 13.9 / 22.5; 1000 ..
// 2000, 256 units of 64 26.7 / 21.1, 512 of 128 85.8 / 76.8, 128 of 128 27.6 / 28.6; 500 .. 4000, 512 of 128 119 / 121; fp32
// 200 .. 2000, 384 of 64 53.2 / 55.9)
constexpr int PA_ONE_KEYS = 1024, PA_ONE_KEYS_FULL = 2048;
constexpr float PA_RESCALE = 8.0f;  // how far (log2) a maximum may rise before the sums are rescaled: p <= 2^8

struct PagedArgs {
  KvPages p;
  int B, heads, group;  // query heads, and of them to a key head
  int rows;             // query heads of a unit: 16, or 32
  int row_tiles;        // units a key head: ceil(group / rows)
  int units;            // units a sequence: kv_heads * row_tiles
  int shares;
  int begin;            // tiles that beginning a unit counts for
  const void* q;
  int64_t q_sb, q_sh;
  const int64_t* lengths;
  int64_t max_length;
  float scale_log2;
  void* out;
  int64_t o_sb, o_sh;
  int32_t* err;
  // workspace
  float* part;    // (2 shares, rows, DHP + 2): sum p v, then m and l
  float* score;   // (B, heads, score_ld), for accumulate
  float* stats;   // (B, heads, 2): m and 1 / l, for accumulate
  int64_t score_ld;
};

template <class P>
struct Query {
  typedef P type;
};
template <>
struct Query<int8_t> {
  typedef bf16 type;
};

template <int N>
struct Words {
  uint32_t w[N];
};
template <int N>
__device__ __forceinline__ Words<N> load_words(const void* p) {
  Words<N> r;
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) *reinterpret_cast<uint4*>(r.w + i) = reinterpret_cast<const uint4*>(p)[i / 4];
  } else if constexpr (N == 2) {
    *reinterpret_cast<uint2*>(r.w) = *reinterpret_cast<const uint2*>(p);
  } else {
    r.w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
  return r;
}

// max / sum over the four lane groups (lanes l, l ^ 16, l ^ 32, l ^ 48), in every lane
__device__ __forceinline__ float group_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, 64));
  return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float group_sum(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

__device__ __forceinline__ int tiles_of(const PagedArgs& a, int b, bool* ok) {
  return (int)((a.p.length_of(a.lengths, b, a.max_length, ok) + PA_KT - 1) / PA_KT);
}

// What a unit counts for when the shares are cut: its tiles, and what it costs to begin one.
__device__ __forceinline__ int work_of(const PagedArgs& a, int tiles) { return tiles ? tiles + a.begin : 0; }

__device__ __forceinline__ int wave_scan_int(int v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(v, o, 64);
    if (lane >= o) v += u;
  }
  return v;
}
__device__ __forceinline__ int wave_sum_int(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// Tiles of a share, from all tiles; every wavefront computes it for itself.
__device__ __forceinline__ int share_of(const PagedArgs& a, int total) {
  return max(PA_MIN_TILES, (total + a.shares - 1) / a.shares);
}

// ONE: a workgroup takes a whole unit, so that nothing is left to join (short caches); else a share.  RT: products of 16
// query heads that share the rows loaded.
template <class P, int DHP, bool PAD, bool W, int WAVES, bool ONE, int RT>
__global__ __launch_bounds__(64 * WAVES, WAVES == PA_WAVES ? per_cu(DHP, sizeof(P), RT) : 2)
void paged_attention_kernel(PagedArgs a) {
  typedef typename Query<P>::type Q;
  constexpr int ES = sizeof(P);
  constexpr int CE = 16 / ES;           // elements of a 16-byte chunk
  constexpr int NK = DHP / (4 * CE);    // chunks of a key row a lane: d = 4 CE c + CE g
  constexpr int E = DHP / 16;           // dims of a value row a lane: d = E r
  constexpr int VW = E * ES / 4;
  constexpr int LD = DHP + 4;
  constexpr int THREADS = 64 * WAVES, ROWS = PA_ROWS * RT;
  __shared__ __attribute__((aligned(16))) float so[WAVES][ROWS][LD];
  __shared__ float sm[WAVES][ROWS], sl[WAVES][ROWS];
  __shared__ float2 stat[ROWS];
  const KvPages& p = a.p;
  const int tid = threadIdx.x, lane = tid & 63, wid = wave_uniform(tid >> 6);
  const int fr = lane & 15, g = lane >> 4;
  const int Dh = PAD ? p.head_dim : DHP;

  int b = 0, off = 0, t0 = 0, t1 = 1;  // its first sequence, the tile of that sequence's units, and how many tiles
  bool ok = true;
  if constexpr (ONE) {
    b = blockIdx.x / a.units;
  } else {
    int total = 0;
    for (int i = lane; i < a.B; i += 64) {
      total += work_of(a, tiles_of(a, i, &ok));
    }
    if (blockIdx.x == 0 && !ok) kv_flag(a.err);
    total = wave_uniform(wave_sum_int(total)) * a.units;
    const int per = share_of(a, total);
    off = t0 = blockIdx.x * per;
    t1 = min(total, t0 + per);
    if (t0 >= t1) return;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
      const int v = b0 + lane < a.B ? work_of(a, tiles_of(a, b0 + lane, &ok)) * a.units : 0;
      const int inc = wave_scan_int(v, lane);
      const uint64_t past = __ballot(inc > off);
      if (past) {
        const int l = __builtin_ctzll(past);
        b = b0 + l;
        off -= __shfl(inc - v, l, 64);
        break;
      }
      off -= __shfl(inc, 63, 64);
    }
    b = wave_uniform(b);
    off = wave_uniform(off);
  }

  while (t0 < t1 && b < a.B) {
    const int64_t n = p.length_of(a.lengths, b, a.max_length, &ok);
    const int tiles = (int)((n + PA_KT - 1) / PA_KT), work = work_of(a, tiles);
    if (!ONE && off >= work * a.units) {  // done, or empty
      ++b;
      off = 0;
      continue;
    }
    const int u = ONE ? blockIdx.x - b * a.units : off / work, from = off - u * work;
    const int step = ONE ? 0 : min(work - from, t1 - t0);
    const int ta = ONE ? 0 : max(0, from - a.begin), tb = ONE ? tiles : max(0, from + step - a.begin);
    t0 += step;
    off += step;
    if (!ONE && ta == tb) continue;
    const int h = u / a.row_tiles, row0 = (u - h * a.row_tiles) * ROWS;
    const int rows = min(ROWS, a.group - row0);  // query heads of this unit
    const int head0 = h * a.group + row0;

    // query rows as the B operand of the scores
    Q q[RT][NK][CE];
#pragma unroll
    for (int y = 0; y < RT; ++y) {
      const int row = 16 * y + fr;
      const Q* src = reinterpret_cast<const Q*>(a.q) + b * a.q_sb + (head0 + (row < rows ? row : 0)) * a.q_sh;
#pragma unroll
      for (int c = 0; c < NK; ++c) {
        const int d = c * 4 * CE + g * CE;
        const bool in = row < rows && (!PAD || d < Dh);
        Words<CE * sizeof(Q) / 4> w = load_words<CE * sizeof(Q) / 4>(src + (!PAD || d < Dh ? d : 0));
#pragma unroll
        for (int i = 0; i < (int)(CE * sizeof(Q) / 4); ++i) w.w[i] = in ? w.w[i] : 0u;
        __builtin_memcpy(q[y][c], w.w, sizeof(w.w));
      }
    }

    const char* kbase = reinterpret_cast<const char*>(p.k) + h * p.k_head * ES;
    const char* vbase = reinterpret_cast<const char*>(p.v) + h * p.v_head * ES;
    const int mask = (1 << p.shift) - 1;
    const int32_t* table = p.table + b * p.ld_table;
    // the page ids of this lane's 8 keys of a tile: for the key rows (8 (r / 4) ..) and the value rows (8 g ..)
    const int last = (int)p.max_slots - 1;  // (not the last key: the lookups need not wait for the length)
    auto page_at = [&](int j) { return table[min(j, last) >> p.shift]; };
    auto kblock = [&](int t) { return t * PA_KT + 8 * (fr >> 2); };
    auto vblock = [&](int t) { return t * PA_KT + 8 * g; };
    auto in_pool = [&](int page) { return (int64_t)((uint32_t)page < (uint32_t)p.num_pages ? page : 0); };

    struct Ids {
      int k, v;
    };
    auto ids_of = [&](int t) { return Ids{page_at(kblock(t)), page_at(vblock(t))}; };
    Words<4> kr[2][NK];
    Words<VW> vr[8];
    f32x4 ks[2], vs[2];
    auto load_k = [&](int t, const Ids& ids) {
      const int64_t at = in_pool(ids.k) * p.k_page;
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        const int row = (kblock(t) & mask) + 4 * st + (fr & 3);
        const char* src = kbase + (at + row * p.k_slot) * ES;
#pragma unroll
        for (int c = 0; c < NK; ++c) {
          const int d = c * 4 * CE + g * CE;
          kr[st][c] = load_words<4>(src + (!PAD || d < Dh ? d : 0) * ES);
        }
      }
    };
    auto load_v = [&](int t, const Ids& ids) {
      const int64_t page = in_pool(ids.v);
      const int row = vblock(t) & mask;
      const int d = !PAD || fr * E < Dh ? fr * E : 0;
      const char* src = vbase + (page * p.v_page + row * p.v_slot + d) * ES;
#pragma unroll
      for (int i = 0; i < 8; ++i) vr[i] = load_words<VW>(src + i * p.v_slot * ES);
    };
    auto load_scales = [&](int t, const Ids& ids) {
      if constexpr (ES == 1) {
        const int64_t i = p.scalar_at((int)in_pool(ids.v), h, vblock(t) & mask);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          ks[x] = reinterpret_cast<const f32x4*>(p.k_scale + i)[x];
          vs[x] = reinterpret_cast<const f32x4*>(p.v_scale + i)[x];
        }
      }
    };

    float m[RT], l[RT];  // of query 16 y + fr; l: the keys of this lane's group only
    f32x4 o[RT][E];
#pragma unroll
    for (int y = 0; y < RT; ++y) {
      m[y] = -INFINITY, l[y] = 0.0f;
#pragma unroll
      for (int j = 0; j < E; ++j) o[y][j] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    }

    int t = ta + wid;
    Ids id = {};
    if (last >= 0) id = ids_of(t);  // (a table may have no columns)
    if (t < tb) {
      load_k(t, id);
      load_scales(t, id);
      load_v(t, id);
      Ids id1 = ids_of(t + WAVES);
      for (; t < tb; t += WAVES) {
        const Ids id2 = ids_of(t + 2 * WAVES);
        const bool more = t + WAVES < tb;
        // scores of keys 8 g + 4 st + i for query 16 y + fr
        f32x4 x[RT][2];
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          f32x4 s[RT];
#pragma unroll
          for (int y = 0; y < RT; ++y) s[y] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int c = 0; c < NK; ++c) {
            Words<4> kk = kr[st][c];
            // (the query is 0 there, the key maybe not finite)
            if (PAD && c * 4 * CE + g * CE >= Dh) kk = Words<4>{{0u, 0u, 0u, 0u}};
#pragma unroll
            for (int y = 0; y < RT; ++y) {
              if constexpr (ES == 2) {
                bf16x8 qf;
                __builtin_memcpy(&qf, q[y][c], 16);
                s[y] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kk), qf, s[y], 0, 0, 0);
              } else if constexpr (ES == 4) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  s[y] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kk.w[e]), q[y][c][e], s[y], 0, 0, 0);
              } else {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  bf16x8 qf;
                  __builtin_memcpy(&qf, q[y][c] + 8 * e, 16);
                  s[y] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen_i8x8(make_uint2(kk.w[2 * e], kk.w[2 * e + 1])), qf,
                                                                 s[y], 0, 0, 0);
                }
              }
            }
          }
#pragma unroll
          for (int y = 0; y < RT; ++y) {
            x[y][st] = s[y] * a.scale_log2;
            if constexpr (ES == 1) x[y][st] *= ks[st];
          }
        }
        if (more) load_k(t + WAVES, id1);

        // where not all of this lane's 8 keys are there
        const bool page_ok = (uint32_t)id.v < (uint32_t)p.num_pages;
        const int left = page_ok ? (int)n - vblock(t) : 0;
        if (!__all(left >= 8)) {
          if (!page_ok && fr == 0 && vblock(t) < (int)n) kv_flag(a.err);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (i >= left) {  // (what these rows hold is not looked at: 0 times it may be NaN)
#pragma unroll
              for (int y = 0; y < RT; ++y) x[y][i >> 2][i & 3] = -INFINITY;
              vr[i] = Words<VW>{};
              if constexpr (ES == 1) vs[i >> 2][i & 3] = 0.0f;
            }
          }
        }
        if constexpr (W) {
#pragma unroll
          for (int y = 0; y < RT; ++y)
            if (16 * y + fr < rows) {
              float* to = a.score + ((int64_t)b * a.heads + head0 + 16 * y + fr) * a.score_ld + vblock(t);
              reinterpret_cast<f32x4*>(to)[0] = x[y][0];
              reinterpret_cast<f32x4*>(to)[1] = x[y][1];
            }
        }
        float pr[RT][8];
        bf16x8 hi[RT], lo[RT];
#pragma unroll
        for (int y = 0; y < RT; ++y) {
          float top = -INFINITY;
#pragma unroll
          for (int st = 0; st < 2; ++st)
            top = fmaxf(top, fmaxf(fmaxf(x[y][st][0], x[y][st][1]), fmaxf(x[y][st][2], x[y][st][3])));
          top = group_max(top);
          if (__any(top > m[y] + PA_RESCALE)) {  // (m -inf: the first key)
            const float m_new = fmaxf(m[y], top);
            const float alpha = exp2f(m[y] - (m_new == -INFINITY ? 0.0f : m_new));
            l[y] *= alpha;
#pragma unroll
            for (int j = 0; j < E; ++j) o[y][j] *= alpha;
            m[y] = m_new;
          }
          const float ref = m[y] == -INFINITY ? 0.0f : m[y];
          float(&p8)[8] = pr[y];
#pragma unroll
          for (int i = 0; i < 8; ++i) p8[i] = __builtin_amdgcn_exp2f(x[y][i >> 2][i & 3] - ref);
          l[y] += ((p8[0] + p8[1]) + (p8[2] + p8[3])) + ((p8[4] + p8[5]) + (p8[6] + p8[7]));
          if constexpr (ES != 4) {
            if constexpr (ES == 1) {
#pragma unroll
              for (int i = 0; i < 8; ++i) p8[i] *= vs[i >> 2][i & 3];
            }
            // p as two bf16 values: its upper half and what is left.  One product with p rounded to bf16 puts the result
            // 1.4 times as far from 64 bits (2.3e-3 against 1.7e-3, the rounding of the result) and saves nothing.  With
            // bf16 rows the half is that of the number below p, which leaves a rest above 0 of every p from 2^-102 up and
            // of 0 none: 0 times an infinite value would be NaN, and a key without weight adds nothing, however large
            uint32_t bits[8], hw[4];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              bits[i] = __float_as_uint(p8[i]);
              if constexpr (ES == 2) bits[i] = __builtin_elementwise_sub_sat(bits[i], 1u);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) hw[i] = __builtin_amdgcn_perm(bits[2 * i + 1], bits[2 * i], 0x07060302u);
            __builtin_memcpy(&hi[y], hw, 16);
#pragma unroll
            for (int i = 0; i < 8; ++i) lo[y][i] = (bf16)(p8[i] - __uint_as_float(bits[i] & 0xffff0000u));
          }
        }

        // O^T += V^T P^T; product j: dims E (4 g + i) + j of query 16 y + fr
        if constexpr (ES == 4) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < E; ++j)
#pragma unroll
              for (int y = 0; y < RT; ++y)
                o[y][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vr[i].w[j]), pr[y][i], o[y][j], 0, 0, 0);
        } else {
#pragma unroll
          for (int j = 0; j < E; ++j) {
            bf16x8 vf;
            if constexpr (ES == 2) {
              uint32_t w[4];
#pragma unroll
              for (int i = 0; i < 4; ++i)
                w[i] = __builtin_amdgcn_perm(vr[2 * i + 1].w[j >> 1], vr[2 * i].w[j >> 1],
                                             (j & 1) ? 0x07060302u : 0x05040100u);
              __builtin_memcpy(&vf, w, 16);
            } else {
#pragma unroll
              for (int i = 0; i < 8; ++i) vf[i] = (bf16)(float)(int)(int8_t)(vr[i].w[j >> 2] >> (8 * (j & 3)));
            }
#pragma unroll
            for (int y = 0; y < RT; ++y) {
              o[y][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, hi[y], o[y][j], 0, 0, 0);
              o[y][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, lo[y], o[y][j], 0, 0, 0);
            }
          }
        }
        if (more) {
          load_scales(t + WAVES, id1);
          load_v(t + WAVES, id1);
        }
        id = id1;
        id1 = id2;
      }
    }

    // the wavefronts' sums into one
    const int active = min(WAVES, tb - ta);
#pragma unroll
    for (int y = 0; y < RT; ++y) {
      const int row = 16 * y + fr;
      const float sum = group_sum(l[y]);
      if (wid < active && row < rows) {
        if (g == 0) sm[wid][row] = m[y], sl[wid][row] = sum;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < E; j += 4)
            *reinterpret_cast<f32x4*>(&so[wid][row][E * (4 * g + i) + j]) =
                f32x4{o[y][j][i], o[y][j + 1][i], o[y][j + 2][i], o[y][j + 3][i]};
      }
    }
    __syncthreads();
    const bool complete = ONE || (ta == 0 && tb == tiles);
    float* part = a.part + (2 * (int64_t)blockIdx.x + (ta == 0)) * (ROWS * (DHP + 2));
    for (int i = tid; i < rows * DHP; i += THREADS) {
      const int r = i / DHP, d = i - r * DHP;
      float top = -INFINITY;  // (ONE: a sequence without keys has none)
      for (int w = 0; w < active; ++w) top = fmaxf(top, sm[w][r]);
      const float ref = top == -INFINITY ? 0.0f : top;
      float sum = 0.0f, acc = 0.0f;
      for (int w = 0; w < active; ++w) {
        const float f = exp2f(sm[w][r] - ref);
        sum += f * sl[w][r];
        acc += f * so[w][r][d];
      }
      if (complete) {
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        if (d < Dh) reinterpret_cast<Q*>(a.out)[b * a.o_sb + (head0 + r) * a.o_sh + d] = from_f32<Q>(acc * inv);
        if (W && d == 0) {
          if constexpr (ONE)
            stat[r] = make_float2(ref, inv);
          else
            reinterpret_cast<float2*>(a.stats)[(int64_t)b * a.heads + head0 + r] = make_float2(ref, inv);
        }
      } else {
        part[r * DHP + d] = acc;
        if (d == 0) part[ROWS * DHP + r] = top, part[ROWS * (DHP + 1) + r] = sum;
      }
    }
    __syncthreads();
    if constexpr (ONE) {
      if constexpr (W) {  // the weight that its keys received
        const float* score = a.score + ((int64_t)b * a.heads + head0) * a.score_ld;
        for (int j = tid; j < (int)n; j += THREADS) {
          float add = 0.0f;
          for (int r = 0; r < rows; ++r) add += exp2f(score[r * a.score_ld + j] - stat[r].x) * stat[r].y;
          const int page = p.page_of(b, j);
          if (page >= 0) p.weight[p.scalar_at(page, h, p.row_of(j))] += add;
        }
      }
      if (h == 0 && row0 == 0 && tid == 0 && !ok) kv_flag(a.err);
      return;
    }
  }
}

constexpr int PJ_THREADS = 256;
constexpr int PJ_KEYS = 4 * PJ_THREADS;  // keys a workgroup adds the weight of
constexpr int PJ_AHEAD = 8;              // loads issued before the factors that they are multiplied by are known

// The parts of the units that several shares hold, joined in the order of their keys (0 for a sequence without keys),
// and with W the weight that every key received, sum over the query heads of a key head of p_j.  Of a (sequence, key
// head) the first `chunks` workgroups take PJ_KEYS keys' weights each, the others a query head each.  The (m, l) of
// the parts are small: every workgroup that needs them reads them itself.  A chain of round trips (lengths, parts, and
// with W the scores): what does not depend on the one before is loaded beside it.  4 to 6 us, 7 with the weights of 16
// sequences of 2048 .. 4160 keys.
template <class Q, int DHP, bool W>
__global__ __launch_bounds__(PJ_THREADS) void paged_join_kernel(PagedArgs a, int chunks) {
  const int64_t stride = a.rows * (DHP + 2);
  constexpr int GROUPS = PJ_THREADS / DHP;  // parts summed side by side
  __shared__ float share[PA_MAX_SHARES];    // a part's factor
  __shared__ float sums[GROUPS][DHP];
  __shared__ float red[2][PJ_THREADS / 64];
  __shared__ float2 stat[W ? 1024 : 1];
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int per_head = chunks + a.group;
  const int bh = blockIdx.x / per_head, c = blockIdx.x - bh * per_head;
  const int b = bh / a.p.kv_heads, h = bh - b * a.p.kv_heads;
  bool ok;
  const int64_t n = a.p.length_of(a.lengths, b, a.max_length, &ok);
  if (W && c < chunks && (int64_t)c * PJ_KEYS >= n) return;
  int total = 0, before = 0;
  for (int i = lane; i < a.B; i += 64) {
    const int x = work_of(a, tiles_of(a, i, &ok));
    total += x;
    before += i < b ? x : 0;
  }
  total = wave_uniform(wave_sum_int(total)) * a.units;
  before = wave_uniform(wave_sum_int(before)) * a.units;
  const int tiles = (int)((n + PA_KT - 1) / PA_KT);
  const int per = share_of(a, total);
  // the shares w0 .. w1 that hold the unit of query head i
  auto unit_of = [&](int i, int* w0, int* w1) {
    const int s = before + (h * a.row_tiles + i / a.rows) * (tiles + a.begin);
    *w0 = min((s + a.begin) / per, a.shares - 1);
    *w1 = min((s + a.begin + tiles - 1) / per, a.shares - 1);  // (in the workspace, whatever becomes of the lengths meanwhile)
  };
  auto slot = [&](int w, int w0) { return a.part + (2 * (int64_t)w + (w == w0)) * stride; };

  if (!W || c >= chunks) {
    const int i = c - chunks, r = i % a.rows;
    Q* out = reinterpret_cast<Q*>(a.out) + b * a.o_sb + (int64_t)(h * a.group + i) * a.o_sh;
    if (tiles == 0) {
      if (tid < a.p.head_dim) out[tid] = from_f32<Q>(0.0f);
      return;
    }
    int w0, w1;
    unit_of(i, &w0, &w1);
    if (w0 == w1) return;  // written by its one workgroup
    const int parts = w1 - w0 + 1;
    const int d = tid % DHP, group = tid / DHP;
    float ahead[PJ_AHEAD];
#pragma unroll
    for (int x = 0; x < PJ_AHEAD; ++x) {
      const int w = group + x * GROUPS;
      ahead[x] = w < parts ? slot(w0 + w, w0)[r * DHP + d] : 0.0f;
    }
    float top = -INFINITY, l0 = 0.0f;
    for (int w = tid; w < parts; w += PJ_THREADS) {
      const float* x = slot(w0 + w, w0) + a.rows * DHP + r;
      share[w] = x[0];
      top = fmaxf(top, x[0]);
      if (w == tid) l0 = x[a.rows];
    }
    top = wave_max(top);
    if (lane == 0) red[0][wid] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    const float ref = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
    for (int w = tid; w < parts; w += PJ_THREADS) {
      const float f = exp2f(share[w] - ref);
      share[w] = f;
      sum += f * (w == tid ? l0 : slot(w0 + w, w0)[a.rows * (DHP + 1) + r]);
    }
    sum = wave_sum(sum);
    if (lane == 0) red[1][wid] = sum;
    __syncthreads();
    sum = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
    float acc = 0.0f;
#pragma unroll
    for (int x = 0; x < PJ_AHEAD; ++x)
      if (group + x * GROUPS < parts) acc += share[group + x * GROUPS] * ahead[x];
#pragma unroll 8
    for (int w = group + PJ_AHEAD * GROUPS; w < parts; w += GROUPS) acc += share[w] * slot(w0 + w, w0)[r * DHP + d];
    sums[group][d] = acc;
    __syncthreads();
    if (tid < a.p.head_dim) {
      acc = sums[0][tid];
#pragma unroll
      for (int x = 1; x < GROUPS; ++x) acc += sums[x][tid];
      out[tid] = from_f32<Q>(acc * (sum == 0.0f ? 0.0f : 1.0f / sum));
    }
    return;
  }

  if constexpr (W) {
    const int64_t j = (int64_t)c * PJ_KEYS + 4 * tid, at = j < n ? j : 0;
    const float* score = a.score + ((int64_t)b * a.heads + h * a.group) * a.score_ld + at;
    f32x4 ahead[PJ_AHEAD];
#pragma unroll
    for (int i = 0; i < PJ_AHEAD; ++i)
      ahead[i] = *reinterpret_cast<const f32x4*>(score + (i < a.group ? i : 0) * a.score_ld);
    const int page = a.p.page_of(b, at);  // (four keys of one page)
    f32x4* weight = reinterpret_cast<f32x4*>(a.p.weight + a.p.scalar_at(page < 0 ? 0 : page, h, a.p.row_of(at)));
    const f32x4 old = *weight;
    // m and 1 / l of the query heads, a wavefront each
    for (int i = wid; i < a.group; i += PJ_THREADS / 64) {
      int w0, w1;
      unit_of(i, &w0, &w1);
      if (w0 == w1) {
        if (lane == 0) stat[i] = reinterpret_cast<const float2*>(a.stats)[(int64_t)b * a.heads + h * a.group + i];
        continue;
      }
      const int r = i % a.rows;
      float top = -INFINITY, sum = 0.0f;
      for (int w = w0 + lane; w <= w1; w += 64) top = fmaxf(top, slot(w, w0)[a.rows * DHP + r]);
      top = wave_max(top);
      const float ref = top == -INFINITY ? 0.0f : top;
      for (int w = w0 + lane; w <= w1; w += 64) {
        const float* x = slot(w, w0) + a.rows * DHP + r;
        sum += exp2f(x[0] - ref) * x[a.rows];
      }
      sum = wave_sum(sum);
      if (lane == 0) stat[i] = make_float2(ref, sum == 0.0f ? 0.0f : 1.0f / sum);
    }
    __syncthreads();
    f32x4 add = {0.0f, 0.0f, 0.0f, 0.0f};
    auto head = [&](const f32x4& x, const float2 s) {
#pragma unroll
      for (int e = 0; e < 4; ++e) add[e] += exp2f(x[e] - s.x) * s.y;
    };
#pragma unroll
    for (int i = 0; i < PJ_AHEAD; ++i)
      if (i < a.group) head(ahead[i], stat[i]);
#pragma unroll 4
    for (int i = PJ_AHEAD; i < a.group; ++i) head(*reinterpret_cast<const f32x4*>(score + i * a.score_ld), stat[i]);
    if (j >= n || page < 0) return;
    if (j + 4 <= n) {
      *weight = old + add;
    } else {
      for (int e = 0; j + e < n; ++e) reinterpret_cast<float*>(weight)[e] = old[e] + add[e];
    }
  }
}

// How a call is laid out: shares, and the parts of its workspace in bytes.
struct Layout {
  int rows, row_tiles, units, shares, begin, dhp;
  int waves;  // of a workgroup that takes a whole unit; 0: shares
  int64_t score_ld, part, score, stats;
};
Layout layout_of(const cortex_kv_pages* p, int64_t B, int64_t heads, int64_t most, int accumulate) {
  Layout y;
  const int64_t group = heads / p->kv_heads, cus = cu_count();
  const int es = p->dtype == DT_F32 ? 4 : p->dtype == DT_BF16 ? 2 : 1;
  y.dhp = p->head_dim <= 64 ? 64 : 128;
  // whole units take 16 query heads (what more there are read short caches again), shares up to 32 at once where their
  // registers hold them (32 sequences of 8000 .. 16000 keys, one key head of 128: 32 heads 73.5 -> 64.7 us, 64 130 -> 90)
  y.rows = PA_ROWS;
  y.row_tiles = (int)cdiv(group, y.rows);
  const bool full = B * p->kv_heads * y.row_tiles >= cus && es < 4;
  y.waves = 0;
  if (most <= (full ? PA_ONE_KEYS_FULL : PA_ONE_KEYS) && (!accumulate || y.row_tiles == 1))
    y.waves = B * p->kv_heads * y.row_tiles > cus ? PA_WAVES : PA_MORE;
  else if (group > PA_ROWS && es < 4)
    y.row_tiles = (int)cdiv(group, y.rows = 2 * PA_ROWS);
  y.units = (int)(p->kv_heads * y.row_tiles);
  const int64_t tiles = B * y.units * cdiv(most, PA_KT), shares = cdiv(tiles, PA_MIN_TILES);
  const int64_t pcu = per_cu(y.dhp, es, y.rows / PA_ROWS);
  const int64_t slots = cus * pcu < PA_MAX_SHARES ? cus * pcu : PA_MAX_SHARES;
  y.shares = (int)(shares < 1 ? 1 : shares < slots ? shares : slots);
  y.begin = tiles / y.shares >= PA_LONG ? PA_BEGIN_LONG : PA_BEGIN_SHORT;
  y.score_ld = cdiv(most, PA_KT) * PA_KT;
  y.part = y.waves ? 0 : 2ll * y.shares * y.rows * (y.dhp + 2) * 4;
  y.score = accumulate ? B * heads * y.score_ld * 4 : 0;
  y.stats = accumulate && !y.waves ? cdiv(B * heads * 2 * 4, 16) * 16 : 0;
  return y;
}

template <class P, int DHP, bool W, int WAVES, bool ONE, int RT>
void launch_main(const PagedArgs& a, unsigned grid, hipStream_t stream) {
  const dim3 block(64 * WAVES);
  if (a.p.head_dim == DHP)
    hipLaunchKernelGGL((paged_attention_kernel<P, DHP, false, W, WAVES, ONE, RT>), dim3(grid), block, 0, stream, a);
  else
    hipLaunchKernelGGL((paged_attention_kernel<P, DHP, true, W, WAVES, ONE, RT>), dim3(grid), block, 0, stream, a);
}
template <class P, int DHP, bool W>
int launch(const PagedArgs& a, int waves, hipStream_t stream) {
  if (waves) {
    const unsigned units = (unsigned)a.B * (unsigned)a.units;
    if (waves == PA_WAVES)
      launch_main<P, DHP, W, PA_WAVES, true, 1>(a, units, stream);
    else
      launch_main<P, DHP, W, PA_MORE, true, 1>(a, units, stream);
    CORTEX_CHECK_LAUNCH("paged_attention_kernel");
    return OK;
  }
  if constexpr (sizeof(P) < 4) {
    if (a.rows > PA_ROWS)
      launch_main<P, DHP, W, PA_WAVES, false, 2>(a, (unsigned)a.shares, stream);
    else
      launch_main<P, DHP, W, PA_WAVES, false, 1>(a, (unsigned)a.shares, stream);
  } else {
    launch_main<P, DHP, W, PA_WAVES, false, 1>(a, (unsigned)a.shares, stream);
  }
  CORTEX_CHECK_LAUNCH("paged_attention_kernel");
  const int64_t chunks = W ? cdiv(a.max_length, PJ_KEYS) : 0;
  hipLaunchKernelGGL((paged_join_kernel<typename Query<P>::type, DHP, W>),
                     dim3((unsigned)((chunks + a.group) * a.B * a.p.kv_heads)), dim3(PJ_THREADS), 0, stream, a, (int)chunks);
  CORTEX_CHECK_LAUNCH("paged_join_kernel");
  return OK;
}
template <class P>
int launch_type(const PagedArgs& a, int waves, int accumulate, hipStream_t stream) {
  if (a.p.head_dim <= 64) return accumulate ? launch<P, 64, true>(a, waves, stream) : launch<P, 64, false>(a, waves, stream);
  return accumulate ? launch<P, 128, true>(a, waves, stream) : launch<P, 128, false>(a, waves, stream);
}

// The length that a call expects at most: max_length, or the table's width where that is negative.
int64_t expected_length(int64_t max_length, int64_t max_slots) {
  return max_length < 0 || max_length > max_slots ? max_slots : max_length;
}

int check_heads(const char* who, const cortex_kv_pages* pages, int64_t B, int64_t heads, int64_t most) {
  CORTEX_CHECK_ARG(heads >= 1 && pages->kv_heads >= 1 && heads % pages->kv_heads == 0 && heads / pages->kv_heads <= 1024,
                   "%s: %lld query heads are not a multiple (up to 1024) of %lld key heads", who, (long long)heads,
                   (long long)pages->kv_heads);
  CORTEX_CHECK_ARG(B >= 0 && B <= 4096, "%s: %lld sequences (at most 4096)", who, (long long)B);
  const int64_t units = pages->kv_heads * cdiv(heads / pages->kv_heads, PA_ROWS);
  CORTEX_CHECK_ARG(most < 0 || B * units <= 0x3fffffffLL / (cdiv(most, PA_KT) + PA_BEGIN_LONG),
                   "%s: %lld sequences of up to %lld keys are too much for one call", who, (long long)B, (long long)most);
  // (a launch has fewer than 2^32 threads: whole units of up to 512, a joining workgroup of 256 a query head and 1024 keys)
  CORTEX_CHECK_ARG(B * units <= 0xffffffffLL / 512 &&
                       (most < 0 || B * pages->kv_heads <= 0xffffffffLL / PJ_THREADS / (cdiv(most, PJ_KEYS) + heads / pages->kv_heads)),
                   "%s: %lld sequences of %lld heads are too much for one call", who, (long long)B, (long long)heads);
  return OK;
}

}  // namespace
}  // namespace cortex

using namespace cortex;

extern "C" int64_t cortex_paged_attention_workspace_bytes(const cortex_kv_pages* pages, int64_t B, int64_t heads,
                                                          int64_t max_length, int accumulate) {
  if (!pages || check_heads("cortex_paged_attention_workspace_bytes", pages, B, heads, max_length) || max_length < 0) return 0;
  const Layout y = layout_of(pages, B, heads, max_length, accumulate);
  return y.part + y.score + y.stats;
}

extern "C" int cortex_paged_attention(const cortex_kv_pages* pages, int64_t B, int64_t heads, const void* q,
                                      int64_t q_sb, int64_t q_sh, const int32_t* block_table, int64_t ld_table,
                                      int64_t max_pages, const int64_t* lengths, int64_t max_length, float scale,
                                      int accumulate, void* out, int64_t o_sb, int64_t o_sh, void* workspace,
                                      int64_t workspace_bytes, int32_t* err, hipStream_t stream) {
  const char* who = "cortex_paged_attention";
  PagedArgs a = {};
  if (int rc = kv_check(who, pages, B, block_table, ld_table, max_pages, &a.p)) return rc;
  a.max_length = expected_length(max_length, a.p.max_slots);
  if (int rc = check_heads(who, pages, B, heads, a.max_length)) return rc;
  CORTEX_CHECK_ARG(!accumulate || pages->weight, "%s: accumulate needs pages with weight", who);
  if (B == 0) return OK;
  CORTEX_CHECK_ARG(q && out && lengths, "%s: null q, out or lengths", who);
  const int64_t es = pages->dtype == DT_F32 ? 4 : 2;
  CORTEX_CHECK_ARG((uintptr_t)q % 16 == 0 && (q_sb * es) % 16 == 0 && (q_sh * es) % 16 == 0,
                   "%s: query rows must be 16-byte aligned", who);
  const Layout y = layout_of(pages, B, heads, a.max_length, accumulate);
  CORTEX_CHECK_ARG((workspace || y.part + y.score + y.stats == 0) && (uintptr_t)workspace % 16 == 0,
                   "%s: null or unaligned workspace", who);
  if (workspace_bytes < y.part + y.score + y.stats) {
    set_error("%s: workspace of %lld bytes, %lld needed", who, (long long)workspace_bytes,
              (long long)(y.part + y.score + y.stats));
    return E_WORKSPACE;
  }
  a.B = (int)B;
  a.heads = (int)heads;
  a.group = (int)(heads / pages->kv_heads);
  a.rows = y.rows;
  a.row_tiles = y.row_tiles;
  a.units = y.units;
  a.shares = y.shares;
  a.begin = y.begin;
  a.q = q;
  a.q_sb = q_sb;
  a.q_sh = q_sh;
  a.lengths = lengths;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.out = out;
  a.o_sb = o_sb;
  a.o_sh = o_sh;
  a.err = err;
  a.score_ld = y.score_ld;
  a.part = reinterpret_cast<float*>(workspace);
  a.score = a.part + y.part / 4;
  a.stats = a.score + y.score / 4;
  if (pages->dtype == DT_F32) return launch_type<float>(a, y.waves, accumulate, stream);
  if (pages->dtype == DT_BF16) return launch_type<bf16>(a, y.waves, accumulate, stream);
  return launch_type<int8_t>(a, y.waves, accumulate, stream);
}
