// Attention of one new token per sequence over its paged keys and values.
#include <hip/hip_runtime.h>

#include "paged_kv.h"

namespace cortex {
namespace {

struct PagedArgs {
  KvPages p;
  int64_t B;
  int heads, group;  // query heads, and of them to a key head
  const void* q;
  int64_t q_sb, q_sh;
  const int64_t* lengths;
  int64_t max_length;
  float scale_log2;
  int accumulate;
  void* out;
  int64_t o_sb, o_sh;
  int32_t* err;
};

template <class P>
struct Query {
  typedef P type;
};
template <>
struct Query<int8_t> {
  typedef bf16 type;
};

// One workgroup a (sequence, key head): its query heads one after the other, 256 keys at a time.
template <class P>
__global__ __launch_bounds__(256) void paged_attention_kernel(PagedArgs a) {
  typedef typename Query<P>::type Q;
  __shared__ float q[128], prob[256], red[4], stats[2][1024];
  const KvPages& p = a.p;
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int64_t b = blockIdx.x / p.kv_heads;
  const int h = blockIdx.x - (int)b * p.kv_heads;
  bool ok = true;
  const int64_t n = p.length_of(a.lengths, b, a.max_length, &ok);
  if (!ok && tid == 0) kv_flag(a.err);
  const P* k = reinterpret_cast<const P*>(p.k) + h * p.k_head;
  const P* v = reinterpret_cast<const P*>(p.v) + h * p.v_head;
  auto score = [&](int64_t j) {
    const int page = p.page_of(b, j);
    if (page < 0) {
      kv_flag(a.err);
      return -INFINITY;
    }
    const P* row = k + page * p.k_page + p.row_of(j) * p.k_slot;
    float s = 0.0f;
    for (int d = 0; d < p.head_dim; ++d) s = fmaf(q[d], to_f32(row[d]), s);
    if (sizeof(P) == 1) s *= p.k_scale[p.scalar_at(page, h, p.row_of(j))];
    return s * a.scale_log2;
  };
  auto load_q = [&](int g) {
    __syncthreads();
    if (tid < p.head_dim) q[tid] = to_f32(reinterpret_cast<const Q*>(a.q)[b * a.q_sb + (h * a.group + g) * a.q_sh + tid]);
    __syncthreads();
  };
  for (int g = 0; g < a.group; ++g) {
    load_q(g);
    float m = -INFINITY, l = 0.0f, acc = 0.0f;
    for (int64_t j0 = 0; j0 < n; j0 += 256) {
      const int64_t j = j0 + tid;
      const float s = j < n ? score(j) : -INFINITY;
      float t = wave_max(s);
      if (lane == 0) red[wid] = t;
      __syncthreads();
      const float m_new = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
      const float ref = m_new == -INFINITY ? 0.0f : m_new;
      const float pr = j < n ? exp2f(s - ref) : 0.0f;
      prob[tid] = pr;
      t = wave_sum(pr);
      __syncthreads();
      if (lane == 0) red[wid] = t;
      __syncthreads();
      const float alpha = exp2f(m - ref);
      l = l * alpha + ((red[0] + red[1]) + (red[2] + red[3]));
      acc *= alpha;
      if (tid < p.head_dim)
        for (int i = 0; i < 256 && j0 + i < n; ++i) {
          const int page = p.page_of(b, j0 + i);
          if (page < 0) continue;
          float x = to_f32(v[page * p.v_page + p.row_of(j0 + i) * p.v_slot + tid]);
          if (sizeof(P) == 1) x *= p.v_scale[p.scalar_at(page, h, p.row_of(j0 + i))];
          acc = fmaf(prob[i], x, acc);
        }
      m = m_new;
      __syncthreads();
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (tid < p.head_dim)
      reinterpret_cast<Q*>(a.out)[b * a.o_sb + (h * a.group + g) * a.o_sh + tid] = from_f32<Q>(acc * inv);
    if (tid == 0) stats[0][g] = m == -INFINITY ? 0.0f : m, stats[1][g] = inv;
  }
  if (!a.accumulate) return;
  for (int g = 0; g < a.group; ++g) {
    load_q(g);
    for (int64_t j = tid; j < n; j += 256) {
      const int page = p.page_of(b, j);
      if (page >= 0) p.weight[p.scalar_at(page, h, p.row_of(j))] += exp2f(score(j) - stats[0][g]) * stats[1][g];
    }
  }
}

}  // namespace
}  // namespace cortex

using namespace cortex;

static int64_t expected_length(int64_t max_length, int64_t max_slots) {
  return max_length < 0 || max_length > max_slots ? max_slots : max_length;
}

extern "C" int64_t cortex_paged_attention_workspace_bytes(const cortex_kv_pages* pages, int64_t B, int64_t heads,
                                                          int64_t max_length, int accumulate) {
  (void)pages, (void)B, (void)heads, (void)max_length, (void)accumulate;
  return 0;
}

extern "C" int cortex_paged_attention(const cortex_kv_pages* pages, int64_t B, int64_t heads, const void* q,
                                      int64_t q_sb, int64_t q_sh, const int32_t* block_table, int64_t ld_table,
                                      int64_t max_pages, const int64_t* lengths, int64_t max_length, float scale,
                                      int accumulate, void* out, int64_t o_sb, int64_t o_sh, void* workspace,
                                      int64_t workspace_bytes, int32_t* err, hipStream_t stream) {
  const char* who = "cortex_paged_attention";
  PagedArgs a = {};
  if (int rc = kv_check(who, pages, B, block_table, ld_table, max_pages, &a.p)) return rc;
  CORTEX_CHECK_ARG(heads >= 1 && heads % pages->kv_heads == 0 && heads / pages->kv_heads <= 1024,
                   "%s: %lld query heads are not a multiple (up to 1024) of %lld key heads", who, (long long)heads,
                   (long long)pages->kv_heads);
  CORTEX_CHECK_ARG(B <= 4096, "%s: %lld sequences (at most 4096)", who, (long long)B);
  CORTEX_CHECK_ARG(!accumulate || pages->weight, "%s: accumulate needs pages with weight", who);
  if (B == 0) return OK;
  CORTEX_CHECK_ARG(q && out && lengths, "%s: null q, out or lengths", who);
  a.B = B;
  a.heads = (int)heads;
  a.group = (int)(heads / pages->kv_heads);
  a.q = q;
  a.q_sb = q_sb;
  a.q_sh = q_sh;
  a.lengths = lengths;
  a.max_length = expected_length(max_length, a.p.max_slots);
  a.scale_log2 = scale * 1.4426950408889634f;
  a.accumulate = accumulate;
  a.out = out;
  a.o_sb = o_sb;
  a.o_sh = o_sh;
  a.err = err;
  (void)workspace, (void)workspace_bytes;
  const dim3 grid((unsigned)(B * pages->kv_heads));
  if (pages->dtype == DT_F32)
    hipLaunchKernelGGL(paged_attention_kernel<float>, grid, dim3(256), 0, stream, a);
  else if (pages->dtype == DT_BF16)
    hipLaunchKernelGGL(paged_attention_kernel<bf16>, grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL(paged_attention_kernel<int8_t>, grid, dim3(256), 0, stream, a);
  CORTEX_CHECK_LAUNCH("paged_attention_kernel");
  return OK;
}
