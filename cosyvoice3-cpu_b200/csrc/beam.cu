// Beam search's choice: the best K of a group's K x V continuations.
//
// key(k, v) = (score_k + log_softmax(x_k)_v) / (count_k + 1)^alpha; a finished hypothesis offers
// itself, unchanged, as its one candidate.  Equal keys go to the lowest k * V + v.
#include <algorithm>

#include "paged.cuh"

namespace {

struct BeamArgs {
  const void* logits;
  int type;
  int64_t ld;
  int64_t groups;
  int beams;
  int64_t vocab;
  const float* scores;
  const int *counts, *done;
  int64_t stop_lo, stop_hi;
  const int* min_len;
  double alpha;
  int64_t* tokens;
  int* parents;
  float* scores_out;
  int *counts_out, *done_out;
  int64_t chunks;
  // workspace: per (row, chunk) the largest logit, the sum of exp against it, and the best candidates
  double* sum;
  float* top;
  unsigned long long* cand;  // [row][chunk][beams]: ordered logit << 32 | ~token; 0: none
};

constexpr int BT = 256, BE = 16;  // threads, logits per thread: a chunk has BT * BE

// floats in an order that unsigned comparison follows; -0 and +0 are one value
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t u) {
  return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u);
}
__device__ __forceinline__ unsigned long long ordered(double x) {
  const unsigned long long u = __double_as_longlong(x + 0.0);
  return u >> 63 ? ~u : u | (1ull << 63);
}

// A hypothesis that nothing can continue: no (or NaN) score.
__device__ __forceinline__ bool dead(float score) { return !(score > -INFINITY); }

// The warp's list of the n largest keys, lane i the i-th: puts in `key` of every lane that beats the n-th.
__device__ __forceinline__ void list_add(unsigned long long key, unsigned long long& list, int n) {
  const int lane = threadIdx.x & 31;
  unsigned long long last = __shfl_sync(0xffffffffu, list, n - 1);
  unsigned wins = __ballot_sync(0xffffffffu, key > last);
  while (wins) {
    const int src = __ffs(wins) - 1;
    const unsigned long long x = __shfl_sync(0xffffffffu, key, src);
    const int at = __popc(__ballot_sync(0xffffffffu, list > x));
    const unsigned long long up = __shfl_up_sync(0xffffffffu, list, 1);
    list = lane < at ? list : lane == at ? x : up;
    if (lane >= n) list = 0;
    last = __shfl_sync(0xffffffffu, list, n - 1);
    if (lane == src) key = 0;
    wins = __ballot_sync(0xffffffffu, key > last);
  }
}

__global__ void __launch_bounds__(BT) beam_scan_kernel(const BeamArgs a) {
  __shared__ float redf[32];
  __shared__ double redd[BT / 32];
  __shared__ unsigned long long lists[BT / 32][32];
  dep_wait();
  dep_release();
  const int64_t row = blockIdx.y, chunk = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (a.done[row]) return;
  const int64_t v0 = chunk * BT * BE;
  const bool none = dead(a.scores[row]);
  const bool early = a.min_len && a.counts[row] < a.min_len[row / a.beams];
  float x[BE], m = -INFINITY;
#pragma unroll
  for (int e = 0; e < BE; ++e) {
    const int64_t v = v0 + e * BT + threadIdx.x;
    x[e] = v < a.vocab ? cv3p::load_any(a.logits, a.type, row * a.ld + v) : -INFINITY;
    if (x[e] != x[e]) x[e] = -INFINITY;  // NaN: no candidate
    m = fmaxf(m, x[e]);
  }
  m = block_max(m, redf);
  double s = 0.0;
#pragma unroll
  for (int e = 0; e < BE; ++e)
    if (x[e] > -INFINITY) s += x[e] == m ? 1.0 : exp((double)x[e] - (double)m);
  s = warp_sum_d(s);
  if (lane == 0) redd[warp] = s;
  unsigned long long list = 0;
#pragma unroll 1
  for (int e = 0; e < BE; ++e) {
    const int64_t v = v0 + e * BT + threadIdx.x;
    const bool out = none || (early && v >= a.stop_lo && v < a.stop_hi);
    const unsigned long long key =
        v < a.vocab ? (unsigned long long)ordered(out ? -INFINITY : x[e]) << 32 | (uint32_t)~(uint32_t)v : 0ull;
    list_add(key, list, a.beams);
  }
  lists[warp][lane] = list;
  __syncthreads();
  if (warp == 0) {
    for (int w = 1; w < BT / 32; ++w) list_add(lists[w][lane], list, a.beams);
    const int64_t at = row * a.chunks + chunk;
    if (lane < a.beams) a.cand[at * a.beams + lane] = list;
    if (lane == 0) {
      double t = 0.0;
      for (int w = 0; w < BT / 32; ++w) t += redd[w];
      a.sum[at] = t;
      a.top[at] = m;
    }
  }
}

// a candidate: ordered key, then lowest k * V + v
struct Cand {
  unsigned long long key;
  unsigned long long tie;  // ~(k * V + v)
};

__device__ __forceinline__ bool better(const Cand& x, const Cand& y) {
  return x.key > y.key || (x.key == y.key && x.tie > y.tie);
}

__device__ __forceinline__ void list_add(Cand c, Cand& list, int n) {
  const int lane = threadIdx.x & 31;
  for (;;) {
    Cand last = {__shfl_sync(0xffffffffu, list.key, n - 1), __shfl_sync(0xffffffffu, list.tie, n - 1)};
    const unsigned wins = __ballot_sync(0xffffffffu, better(c, last));
    if (!wins) return;
    const int src = __ffs(wins) - 1;
    const Cand x = {__shfl_sync(0xffffffffu, c.key, src), __shfl_sync(0xffffffffu, c.tie, src)};
    const int at = __popc(__ballot_sync(0xffffffffu, better(list, x)));
    const Cand up = {__shfl_up_sync(0xffffffffu, list.key, 1), __shfl_up_sync(0xffffffffu, list.tie, 1)};
    list = lane < at ? list : lane == at ? x : up;
    if (lane >= n) list = Cand{0, 0};
    if (lane == src) c = Cand{0, 0};
  }
}

// score + log-probability of a token, from its logit, its row's largest and log(sum of exp against it)
__device__ __forceinline__ double continued(double base, float x, float top, double lsum) {
  if (!(x > -INFINITY)) return -(double)INFINITY;
  const double c = base + ((x == top ? 0.0 : (double)x - (double)top) - lsum);
  return c == c ? c : -(double)INFINITY;  // (an infinite score and an impossible token)
}

__global__ void __launch_bounds__(BT) beam_pick_kernel(const BeamArgs a) {
  __shared__ double lsum[CV3_MAX_BEAMS], base[CV3_MAX_BEAMS], norm[CV3_MAX_BEAMS];
  __shared__ float tops[CV3_MAX_BEAMS];
  __shared__ Cand lists[BT / 32][32];
  dep_wait();
  dep_release();
  const int64_t g = blockIdx.x;
  const int K = a.beams, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int k = warp; k < K; k += BT / 32) {
    const int64_t row = g * K + k;
    const bool fin = a.done[row] != 0;
    float m = -INFINITY;
    double s = 0.0;
    if (!fin) {
      for (int64_t c = lane; c < a.chunks; c += 32) m = fmaxf(m, a.top[row * a.chunks + c]);
      m = warp_max(m);
      for (int64_t c = lane; c < a.chunks; c += 32) {
        const float t = a.top[row * a.chunks + c];
        if (t > -INFINITY) s += a.sum[row * a.chunks + c] * (t == m ? 1.0 : exp((double)t - (double)m));
      }
      s = warp_sum_d(s);
    }
    if (lane == 0) {
      const float sc = a.scores[row];
      const int n = max(a.counts[row], 0) + (fin ? 0 : 1);
      tops[k] = m;
      lsum[k] = log(s);
      base[k] = dead(sc) ? -INFINITY : (double)sc;
      norm[k] = a.alpha == 0.0 ? 1.0 : pow((double)max(n, 1), a.alpha);
    }
  }
  __syncthreads();
  Cand list = {0, 0};
  const int64_t per = a.chunks * K, all = per * K;
  for (int64_t i0 = warp * 32; i0 < all; i0 += BT) {
    const int64_t i = i0 + lane;
    Cand c = {0, 0};
    if (i < all) {
      const int k = (int)(i / per);
      const int64_t row = g * K + k;
      if (a.done[row]) {
        const int64_t v = i - (int64_t)k * per;  // itself, then what stands in where nothing is left
        if (v < K && v < a.vocab)
          c = Cand{ordered(v == 0 ? base[k] / norm[k] : -(double)INFINITY), ~(unsigned long long)(k * a.vocab + v)};
      } else {
        const unsigned long long u = a.cand[row * per + (i - (int64_t)k * per)];
        if (u) {
          const float x = unordered((uint32_t)(u >> 32));
          const uint32_t v = ~(uint32_t)u;
          c = Cand{ordered(continued(base[k], x, tops[k], lsum[k]) / norm[k]), ~(unsigned long long)(k * a.vocab + v)};
        }
      }
    }
    list_add(c, list, K);
  }
  lists[warp][lane] = list;
  __syncthreads();
  if (warp) return;
  for (int w = 1; w < BT / 32; ++w) list_add(lists[w][lane], list, K);
  if (lane >= K) return;
  const int64_t id = (int64_t)~list.tie;
  const int k = (int)(id / a.vocab);
  const int64_t v = id - (int64_t)k * a.vocab, row = g * K + k, to = g * K + lane;
  const bool fin = a.done[row] != 0;
  double cum = -(double)INFINITY;
  if (list.key > ordered(-(double)INFINITY)) {
    cum = fin ? base[k] : continued(base[k], cv3p::load_any(a.logits, a.type, row * a.ld + v), tops[k], lsum[k]);
  }
  const int count = a.counts[row] + (fin ? 0 : 1);
  __syncwarp(0xffffffffu >> (32 - K));  // the outputs may be the inputs' own buffers
  a.tokens[to] = fin ? 0 : v;
  a.parents[to] = k;
  a.scores_out[to] = (float)cum;
  a.counts_out[to] = count;
  a.done_out[to] = fin || (v >= a.stop_lo && v < a.stop_hi) ? 1 : 0;
}

int64_t chunks_of(int64_t vocab) { return (vocab + BT * BE - 1) / (BT * BE); }

}  // namespace

extern "C" int64_t cv3_beam_workspace(int64_t groups, int64_t beams, int64_t vocab) {
  return groups * beams * chunks_of(vocab) * (16 + 8 * beams);
}

extern "C" int cv3_beam_select(const cv3_beam_params* p, void* stream) {
  CV3_REQUIRE(p && p->size == (int64_t)sizeof(*p), CV3_ERR_VALUE, "beam_select: bad parameter block");
  CV3_REQUIRE(p->groups >= 0 && p->vocab > 0 && p->vocab <= INT32_MAX && p->ld >= p->vocab && p->stop_lo <= p->stop_hi,
              CV3_ERR_VALUE, "beam_select: bad shape");
  CV3_REQUIRE(p->beams > 0 && p->beams <= CV3_MAX_BEAMS, CV3_ERR_UNSUPPORTED, "beam_select: %lld beams (1 to %d)",
              (long long)p->beams, CV3_MAX_BEAMS);
  CV3_REQUIRE(cv3p::type_ok(p->type), CV3_ERR_VALUE, "beam_select: unknown element type");
  CV3_REQUIRE(p->groups <= 65535 && p->groups * p->beams <= 65535, CV3_ERR_UNSUPPORTED,
              "beam_select: more than 65535 hypotheses");
  if (p->groups == 0) return CV3_OK;
  const int64_t chunks = chunks_of(p->vocab), n = p->groups * p->beams * chunks;
  CV3_REQUIRE(p->workspace && p->workspace_bytes >= cv3_beam_workspace(p->groups, p->beams, p->vocab) &&
                  ((uintptr_t)p->workspace & 7) == 0,
              CV3_ERR_VALUE, "beam_select: the workspace must hold cv3_beam_workspace() bytes");
  char* w = static_cast<char*>(p->workspace);
  const BeamArgs a = {p->logits, (int)p->type, p->ld, p->groups, (int)p->beams, p->vocab, p->scores, p->counts, p->done,
                      p->stop_lo, p->stop_hi, p->min_len, p->length_penalty, p->tokens, p->parents, p->scores_out,
                      p->counts_out, p->done_out, chunks, reinterpret_cast<double*>(w), reinterpret_cast<float*>(w + 8 * n),
                      reinterpret_cast<unsigned long long*>(w + 16 * n)};
  cudaStream_t st = cv3::as_stream(stream);
  int rc = cv3::check_launch("beam_scan", cv3::launch_dep(beam_scan_kernel, dim3((unsigned)chunks, (unsigned)(p->groups * p->beams)),
                                                          dim3(BT), 0, st, a));
  if (rc) return rc;
  return cv3::check_launch("beam_pick", cv3::launch_dep(beam_pick_kernel, dim3((unsigned)p->groups), dim3(BT), 0, st, a));
}
