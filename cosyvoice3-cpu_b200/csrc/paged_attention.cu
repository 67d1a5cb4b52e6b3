// Attention of one new token per request over its paged key/value cache.
//
// out[b][h] = sum_j p_j V[j], p = softmax(scale * q[b][h] . K[j]) over the request's cached keys j
// in [max(0, len - window), len); a request without keys gives zeros and a log-sum of -inf.
#include <algorithm>

#include "paged.cuh"

namespace {

struct AttnArgs {
  const void* q;
  int q_type;
  int64_t qsb, qsh;
  const void *k, *v;
  int64_t ksp, ksh, kst, vsp, vsh, vst, pages, ps;
  const int* tables;
  int64_t ld, max_blocks;
  const int* lens;
  int heads, kv_heads;
  int64_t window;
  float scale;
  void* out;
  int64_t osb, osh;
  float* lse;
  int* bad;
};

constexpr int AW = 8;  // warps: each takes every AW-th key

// One CTA per (request, query head); a warp's lanes hold D / 32 dimensions of the head.
template <typename KT, int D>
__global__ void __launch_bounds__(AW * 32) paged_attention_kernel(const AttnArgs a) {
  constexpr int E = D / 32;
  __shared__ float part[AW][D], pm[AW], pl[AW];
  dep_wait();
  dep_release();
  const int h = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t b = blockIdx.y;
  const int g = h / (a.heads / a.kv_heads);
  const int64_t len = min((int64_t)max(a.lens[b], 0), a.max_blocks * a.ps);
  const int64_t lo = a.window > 0 ? max(len - a.window, (int64_t)0) : 0;
  float q[E], acc[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = cv3p::load_any(a.q, a.q_type, b * a.qsb + h * a.qsh + lane * E + e) * a.scale;
    acc[e] = 0.f;
  }
  for (int64_t j = lo + warp; j < len; j += AW) {
    const int64_t blk = j / a.ps, r = j - blk * a.ps;
    const int page = a.tables[b * a.ld + blk];
    if (page < 0 || page >= a.pages) {
      if (a.bad && h == 0 && lane == 0 && (r == 0 || j == lo)) atomicAdd(a.bad, 1);
      continue;
    }
    const KT* kr = static_cast<const KT*>(a.k) + page * a.ksp + g * a.ksh + r * a.kst + lane * E;
    const KT* vr = static_cast<const KT*>(a.v) + page * a.vsp + g * a.vsh + r * a.vst + lane * E;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s = fmaf(q[e], cv3p::to_f32<KT>(kr[e]), s);
    s = warp_sum(s);
    const float mn = fmaxf(m, s);
    const float c = m == -INFINITY ? 0.f : expf(m - mn), p = s == -INFINITY ? 0.f : expf(s - mn);
    m = mn;
    l = l * c + p;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = acc[e] * c + p * cv3p::to_f32<KT>(vr[e]);
  }
#pragma unroll
  for (int e = 0; e < E; ++e) part[warp][lane * E + e] = acc[e];
  if (lane == 0) { pm[warp] = m; pl[warp] = l; }
  __syncthreads();
  float M = -INFINITY, L = 0.f;
  for (int w = 0; w < AW; ++w) M = fmaxf(M, pm[w]);
  for (int w = 0; w < AW; ++w) L += pl[w] == 0.f ? 0.f : pl[w] * expf(pm[w] - M);  // (a NaN score: l is NaN)
  for (int e = threadIdx.x; e < D; e += AW * 32) {
    float o = 0.f;
    for (int w = 0; w < AW; ++w) o += pl[w] == 0.f ? 0.f : part[w][e] * expf(pm[w] - M);
    cv3p::store_any(a.out, a.q_type, b * a.osb + h * a.osh + e, L == 0.f ? 0.f : o / L);
  }
  if (a.lse && threadIdx.x == 0) a.lse[b * a.heads + h] = L == 0.f ? -INFINITY : M + logf(L);
}

template <typename KT>
void (*pick(int64_t d))(const AttnArgs) {
  switch (d) {
    case 32: return paged_attention_kernel<KT, 32>;
    case 64: return paged_attention_kernel<KT, 64>;
    case 96: return paged_attention_kernel<KT, 96>;
    default: return paged_attention_kernel<KT, 128>;
  }
}

}  // namespace

extern "C" int64_t cv3_paged_attention_workspace(int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                                 int64_t max_len) {
  return 0;
}

extern "C" int cv3_paged_attention(const void* q, int q_type, int64_t qsb, int64_t qsh, const void* k_pages,
                                   const void* v_pages, int kv_type, int64_t ksp, int64_t ksh, int64_t kst, int64_t vsp,
                                   int64_t vsh, int64_t vst, int64_t num_pages, int64_t page_size,
                                   const int* block_tables, int64_t table_ld, int64_t max_blocks, const int* lens,
                                   int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t window,
                                   float scale, void* out, int64_t osb, int64_t osh, float* lse, int* bad,
                                   float* workspace, int64_t workspace_floats, void* stream) {
  CV3_REQUIRE(batch >= 0 && heads > 0 && kv_heads > 0 && num_pages >= 0 && page_size > 0 && max_blocks >= 0 &&
                  table_ld >= max_blocks && window >= 0,
              CV3_ERR_VALUE, "paged_attention: bad shape");
  CV3_REQUIRE(heads % kv_heads == 0, CV3_ERR_VALUE, "%lld query heads is not a multiple of %lld kv heads",
              (long long)heads, (long long)kv_heads);
  CV3_REQUIRE(head_dim == 32 || head_dim == 64 || head_dim == 96 || head_dim == 128, CV3_ERR_UNSUPPORTED,
              "paged_attention: head_dim %lld (built for 32, 64, 96 and 128)", (long long)head_dim);
  CV3_REQUIRE(cv3p::type_ok(q_type) && cv3p::type_ok(kv_type), CV3_ERR_VALUE, "paged_attention: unknown element type");
  const int ce = 16 / cv3p::type_size(kv_type);
  CV3_REQUIRE(cv3p::aligned16(k_pages) && cv3p::aligned16(v_pages) && (ksp | ksh | kst | vsp | vsh | vst) % ce == 0,
              CV3_ERR_VALUE, "paged_attention: cache rows must start on 16-byte boundaries");
  CV3_REQUIRE(max_blocks * page_size <= INT32_MAX, CV3_ERR_VALUE, "paged_attention: positions are 32-bit numbers");
  if (batch == 0) return CV3_OK;
  const AttnArgs a = {q, q_type, qsb, qsh, k_pages, v_pages, ksp, ksh, kst, vsp, vsh, vst, num_pages, page_size,
                      block_tables, table_ld, max_blocks, lens, (int)heads, (int)kv_heads, window, scale, out, osb, osh,
                      lse, bad};
  const auto fn = kv_type == CV3_TYPE_F32 ? pick<float>(head_dim)
                  : kv_type == CV3_TYPE_F16 ? pick<__half>(head_dim) : pick<__nv_bfloat16>(head_dim);
  return cv3::check_launch("paged_attention", cv3::launch_dep(fn, dim3((unsigned)heads, (unsigned)batch), dim3(AW * 32), 0,
                                                              cv3::as_stream(stream), a));
}
