// Beam search's choice: the best K of a group's K x V continuations.
//
// key(k, v) = (score_k + log_softmax(x_k)_v) / (count_k + 1)^alpha; a finished hypothesis offers
// itself, unchanged, as its one candidate.  Equal keys go to the lower hypothesis, its larger logit (the 64
// bits of a key may have no room for it under a huge score), the lower token.
//
// Bound by the logits' bytes.  Within a hypothesis the key grows with the logit, so a row gives its K
// largest logits (lowest token on ties) and its log-sum-exp; the K * K candidates are then ordered by
// keys in 64 bits.  A CTA reads its chunk of a row in tiles of 512 logits, once for the sum and the
// tiles' maxima; the K-th largest of these maxima (with fewer than K tiles: of the lanes') bounds the K-th logit from
// below, so only the tiles that reach it -- at most K, but for ties -- are read again (from L2) for candidates.  (Lists kept
// while reading cost more than all the rest.)  32 x 8 rows over 151936 tokens take 58 us (156 MB, 2.7 TB/s), with a
// seventh of them finished, which are not read, 46 us (133 MB, 2.9 TB/s): the sum's 21 instructions a logit (their issue slots are
// half full, waits on one another fill the rest) and the waits of the two readings bound it.
//
// Precision: candidates of different hypotheses may lie closer than fp32 resolves, so the log-sum-exp
// is held to 2e-8 whatever the logits are: a term e^(x - m) is 2^(k + j/32) (1 + q), the power of two a 64-bit number
// put together from a table and added up in 64 bits, q -- at most 0.022 -- a cubic in fp32 (see Terms).
#include <algorithm>

#include "paged.cuh"

namespace {

struct BeamArgs {
  const void* logits;
  int64_t ld;
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
  int chunks;      // of a row
  int64_t tiles;   // of a chunk
  char* work;      // the tasks' results of all groups (two launches)
};

typedef unsigned long long u64;

constexpr int BW = 8, BT = BW * 32;
constexpr int TILE = 512;      // logits of a warp's step, 16 a lane
constexpr int TILES_MOST = 1024;  // of a task (a multiple of the warps)

// A task's (row's chunk's) result: sum of exp against the largest logit, that logit, then `beams`
// candidates: ordered logit << 32 | ~token, 0 for none.
__host__ __device__ constexpr int64_t task_bytes(int64_t beams) { return 16 + 8 * beams; }

// floats in an order that unsigned comparison follows; -0 and +0 are one value
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t u) {
  return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u);
}
__device__ __forceinline__ u64 ordered(double x) {
  const u64 u = __double_as_longlong(x + 0.0);
  return u >> 63 ? ~u : u | (1ull << 63);
}

__device__ __forceinline__ double unordered(u64 u) {
  return __longlong_as_double(u >> 63 ? u & ~(1ull << 63) : ~u);
}

// A hypothesis that nothing can continue: no (or NaN) score.
__device__ __forceinline__ bool dead(float score) { return !(score > -INFINITY); }


// A candidate of the choice: ordered key, then lowest hypothesis, largest logit, lowest token.
struct Cand {
  u64 key;
  u64 place;
};
constexpr int TOKEN_BITS = 27;  // 5 bits of the hypothesis, 32 of the ordered logit, these
constexpr uint32_t TOKENS = 1u << TOKEN_BITS;

__device__ __forceinline__ u64 place_of(int k, uint32_t logit, uint32_t token) {
  return (u64)(CV3_MAX_BEAMS - 1 - k) << (TOKEN_BITS + 32) | (u64)logit << TOKEN_BITS | (TOKENS - 1 - token);
}
static_assert(CV3_MAX_BEAMS <= 32, "a hypothesis's number takes 5 bits");

__device__ __forceinline__ bool better(u64 x, u64 y) { return x > y; }
__device__ __forceinline__ bool better(const Cand& x, const Cand& y) {
  return x.key > y.key || (x.key == y.key && x.place > y.place);
}
__device__ __forceinline__ u64 from_lane(u64 x, int lane) { return __shfl_sync(0xffffffffu, x, lane); }
__device__ __forceinline__ Cand from_lane(const Cand& x, int lane) { return {from_lane(x.key, lane), from_lane(x.place, lane)}; }
__device__ __forceinline__ u64 across(u64 x, int j) { return __shfl_xor_sync(0xffffffffu, x, j); }
__device__ __forceinline__ Cand across(const Cand& x, int j) { return {across(x.key, j), across(x.place, j)}; }

// The warp's lists: lane i holds the i-th best, zeros behind the last.  A bitonic network sorts 32
// entries in 15 exchanges; two sorted lists give the 32 best of both in 5.
template <typename X>
__device__ __forceinline__ X exchange(X x, int j, bool keep_better) {
  const X y = across(x, j);
  return better(x, y) == keep_better ? x : y;
}
template <typename X>
__device__ __forceinline__ X sorted(X x) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) x = exchange(x, j, ((lane & j) == 0) == ((lane & k) == 0));
  return x;
}
template <typename X>
__device__ __forceinline__ X merged(X x, const X& other) {
  const int lane = threadIdx.x & 31;
  const X y = from_lane(other, 31 - lane);
  x = better(x, y) ? x : y;
#pragma unroll
  for (int j = 16; j > 0; j >>= 1) x = exchange(x, j, (lane & j) == 0);
  return x;
}

// e^(x - m) = 2^n (1 + q), n the multiple of 1/32 that x log2(e) - R rounds to, R the one that m log2(e) rounds to.  Adding
// 1.5 * 2^18 to a number rounds it to such a multiple and leaves it in the low bits of the sum; n + R is exact, and what is
// left of x log2(e) (log2(e) in two parts) comes out of one fused product.  Taking off what is left of m log2(e), the term
// of m itself is 1, exactly, and what is left of x is within 2^-5: 2^f - 1 = f (C1 + C2 f + C3 f^2), whose f^4 term
// is spread over the others as the Chebyshev polynomial has it (2.3e-9 off at most).  x is taken no lower than m - 80, which
// adds less than 1e-29 to any sum (NaN goes there too).
constexpr float LOG2E_HI = 1.442695022f, LOG2E_LO = 1.925963033e-8f;  // the nearest fp32 number and the rest's
constexpr float STEPS = 393216.f;
constexpr float MOST = 65536.f;  // |m| up to which R + n stays a number of the sum's kind
constexpr double LN2 = 0.693147180559945309;
constexpr float C1 = (float)LN2, C3 = (float)(LN2 * LN2 * LN2 / 6),
                C2 = (float)(LN2 * LN2 / 2 + LN2 * LN2 * LN2 * LN2 / 24 * 0.75 / 1024);

// two fp32 numbers in one instruction
struct Two {
  u64 v;
};
__device__ __forceinline__ Two two(float x, float y) {
  Two r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ Two fma(Two x, Two y, Two z) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(x.v), "l"(y.v), "l"(z.v));
  return r;
}
__device__ __forceinline__ Two add(Two x, Two y) {
  Two r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(x.v), "l"(y.v));
  return r;
}
__device__ __forceinline__ Two mul(Two x, Two y) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(x.v), "l"(y.v));
  return r;
}
__device__ __forceinline__ void apart(Two x, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x.v)); }

struct Reference {  // what the terms need of m
  float least, start, rest;
  __device__ __forceinline__ explicit Reference(float m) {
    const float r = fmaf(m, LOG2E_HI, STEPS) - STEPS;
    least = m - 80.f;
    start = STEPS - r;
    rest = fmaf(m, LOG2E_LO, fmaf(m, LOG2E_HI, -r));
  }
};

__device__ __forceinline__ float warp_top(float x) {  // of values that are not NaN
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}

// The CTA's shared memory for a task.
struct Scratch {
  u64 held[BW][64];  // candidates on their way into a warp's list
  u64 lists[BW][32];
  double ss[BW];
  float ms[BW];
  uint32_t tops[TILES_MOST];  // ordered maxima of the tiles (stop ids left out where they are none)
  uint32_t bar;
  uint32_t power_hi[32], power_lo[32];  // 2^(j/32) in 64 bits, the upper word less j << 15 (what j adds to it in a sum)

  __device__ __forceinline__ void fill() {
    if (threadIdx.x < 32) {
      const u64 p = __double_as_longlong(exp2(threadIdx.x / 32.0));
      power_hi[threadIdx.x] = (uint32_t)(p >> 32) - (threadIdx.x << 15);
      power_lo[threadIdx.x] = (uint32_t)p;
    }
  }
};

// One task by the whole CTA; false for rows whose logits do not count (finished hypotheses and those that
// do not exist).  A lane takes every 32nd logit of a tile, so rows may begin anywhere and alike rows give
// the same bits wherever they lie; nothing depends on the warps' timing either.
// The result is in warp 0: list, and in every lane m and s.
template <typename T>
__device__ bool scan(const BeamArgs& a, int64_t row, int64_t chunk, Scratch& sh, u64& list, float& m, double& s) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, K = a.beams;
  const T* logits = static_cast<const T*>(a.logits) + row * a.ld;
  const int begin = (int)(chunk * a.tiles * TILE);
  const int tiles = (int)((min((chunk + 1) * a.tiles * TILE, a.vocab) - begin + TILE - 1) / TILE);
  float x[16];
  int v0 = 0;  // token of the lane's first logit; the others follow in steps of 32
  auto inside = [&](int e) -> bool { return v0 + e * 32 < a.vocab; };
  auto stopped = [&](int e) -> bool { return v0 + e * 32 >= a.stop_lo && v0 + e * 32 < a.stop_hi; };
  T raw[16];
  auto fetch = [&](int tile) {
    const int at = begin + tile * TILE + lane;
    const T* p = logits + at;
    if (at - lane + TILE <= a.vocab) {
#pragma unroll
      for (int e = 0; e < 16; ++e) raw[e] = p[e * 32];
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) raw[e] = at + e * 32 < a.vocab ? p[e * 32] : cv3p::from_f32<T>(-INFINITY);
    }
  };
  auto take = [&](int tile) {
    v0 = begin + tile * TILE + lane;
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = cv3p::to_f32<T>(raw[e]);
  };
  auto no_nan = [&]() {  // a NaN logit is no term, and as good as -inf
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = fmaxf(x[e], -INFINITY);
  };
  auto maximum = [&]() -> float {  // (fmaxf passes over NaN)
    float top = -INFINITY;
#pragma unroll
    for (int e = 0; e < 16; ++e) top = fmaxf(top, x[e]);
    return top;
  };

  // the first tile and the row's state on their way together
  if (warp < tiles) fetch(warp);
  const bool fin = a.done[row] != 0;
  const float score = a.scores[row];
  const int count_so_far = a.counts[row], least_count = a.min_len ? a.min_len[row / K] : 0;
  if (fin || dead(score)) return false;
  const bool early = a.min_len && count_so_far < least_count && a.stop_lo < a.stop_hi;

  // first reading: the sum of exp against a running maximum that begins with the first BW tiles', and
  // the tiles' maxima
  float mine = -INFINITY, wtop = -INFINITY;  // the tile's maximum in this lane and in the warp
  if (warp < tiles) {
    take(warp);
    mine = maximum();
    wtop = warp_top(mine);
  }
  u64* held = sh.held[warp];
  int count = 0;
  __syncthreads();  // (the last task's shared memory is done with)
  if (lane == 0) sh.ms[warp] = wtop;
  __syncthreads();
  m = -INFINITY;
  s = 0.0;
#pragma unroll
  for (int w = 0; w < BW; ++w) m = fmaxf(m, sh.ms[w]);
  Reference ref(m);
  // a tile's terms against m
  auto add_terms = [&]() {
    double powers[2] = {0.0, 0.0};
    Two rests = two(0.f, 0.f);
    const Two start = two(ref.start, ref.start), rest = two(-ref.rest, -ref.rest), log_hi = two(LOG2E_HI, LOG2E_HI),
              log_lo = two(LOG2E_LO, LOG2E_LO);
#pragma unroll
    for (int e = 0; e < 16; e += 2) {
      const Two y = two(fmaxf(x[e], ref.least), fmaxf(x[e + 1], ref.least)), n = fma(y, log_hi, start);
      Two f = fma(y, log_hi, fma(n, two(-1.f, -1.f), start));
      f = add(fma(y, log_lo, f), rest);
      const Two q = mul(f, fma(fma(two(C3, C3), f, two(C2, C2)), f, two(C1, C1)));
      float at[2], power[2];
      apart(n, at[0], at[1]);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t bits = __float_as_uint(at[i]), hi = sh.power_hi[bits & 31u] + (bits << 15), lo = sh.power_lo[bits & 31u];
        powers[i] += __hiloint2double((int)hi, (int)lo);
        // the same power in fp32, cut off: 2^-23 of 0.022
        power[i] = __uint_as_float(__funnelshift_l(lo, hi, 3) + ((127u - 1023u) << 23));
      }
      rests = fma(two(power[0], power[1]), q, rests);
    }
    float even, odd;
    apart(rests, even, odd);
    s += (powers[0] + powers[1]) + (double)(even + odd);
  };
  // the same where m is infinite or beyond what n holds: one by one in 64 bits (terms below e^-64 left out)
  auto add_terms_far = [&]() {
#pragma unroll 1
    for (int e = 0; e < 16; ++e) {
      float y = 0.f;
#pragma unroll
      for (int f = 0; f < 16; ++f) y = f == e ? x[f] : y;
      if (y == m) s += 1.0;
      else if (y > m - 64.f) s += exp((double)y - (double)m);
    }
  };
  // too few maxima to bound the K-th logit: the lanes' serve (32 x 32 rows of 6761 tokens: 62 us instead of 120, where
  // all were candidates)
  const bool few = tiles < K;
  u64 best = 0;
  for (int tile = warp; tile < tiles;) {
    if (tile + BW < tiles) fetch(tile + BW);  // on its way while this one is worked on
    if (wtop > m) {
      if (s != 0.0) s *= exp((double)m - (double)wtop);
      m = wtop;
      ref = Reference(m);
    }
    float mine_allowed = mine, allowed = wtop;
    if (early && v0 - lane < a.stop_hi && v0 - lane + TILE > a.stop_lo) {
      mine_allowed = -INFINITY;
#pragma unroll
      for (int e = 0; e < 16; ++e) mine_allowed = stopped(e) ? mine_allowed : fmaxf(mine_allowed, x[e]);
      allowed = warp_top(mine_allowed);
    }
    if (lane == 0) sh.tops[tile] = ordered(allowed);
    if (few) {
      const u64 key = ordered(mine_allowed);
      best = tile == warp ? sorted(key) : merged(best, sorted(key));
    }
    if (m > -INFINITY) {
      if (fabsf(m) < MOST) add_terms();
      else add_terms_far();
    }
    tile += BW;
    if (tile < tiles) {
      take(tile);
      mine = maximum();
      wtop = warp_top(mine);
    }
  }
  if (few) sh.lists[warp][lane] = best;
  __syncthreads();

  // the bar: the K-th largest of the tiles' maxima, or of the lanes'
  if (warp == 0) {
    if (few) {
      for (int w = 1; w < min(tiles, BW); ++w) best = merged(best, sh.lists[w][lane]);
    } else {
      for (int i = 0; i < tiles; i += 32) {
        const u64 key = i + lane < tiles ? (u64)sh.tops[i + lane] : 0ull;
        if (__any_sync(0xffffffffu, key > from_lane(best, K - 1))) best = i ? merged(best, sorted(key)) : sorted(key);
      }
    }
    const uint32_t bar = (uint32_t)from_lane(best, K - 1);
    if (lane == 0) sh.bar = bar;
  }
  __syncthreads();

  // second reading: what reaches the bar, merged into the warp's list 32 at a time
  const uint32_t bar = sh.bar;
  const float least = bar ? unordered(bar) : -INFINITY;
  int turn = 0;
  count = 0;
  bool listed = false;
  list = 0;
  auto flush = [&]() {
    __syncwarp();
    const u64 key = lane < count ? held[lane] : 0ull, rest = lane + 32 < count ? held[lane + 32] : 0ull;
    __syncwarp();
    held[lane] = rest;
    __syncwarp();
    count = max(count - 32, 0);
    list = listed ? merged(list, sorted(key)) : sorted(key);
    listed = true;
    if (lane >= K) list = 0;
  };
  for (int t0 = 0; t0 < tiles; t0 += 32) {
    unsigned reach = __ballot_sync(0xffffffffu, t0 + lane < tiles && sh.tops[t0 + lane] >= bar);
    for (; reach; reach &= reach - 1) {
      if (turn++ % BW != warp) continue;
      fetch(t0 + __ffs(reach) - 1);
      take(t0 + __ffs(reach) - 1);
      no_nan();
      unsigned fits = 0;
#pragma unroll
      for (int e = 0; e < 16; ++e) fits |= (x[e] >= least && inside(e) ? 1u : 0u) << e;
      for (unsigned left = __reduce_or_sync(0xffffffffu, fits); left; left &= left - 1) {
        const int e = __ffs(left) - 1;
        float y = 0.f;
#pragma unroll
        for (int f = 0; f < 16; ++f) y = f == e ? x[f] : y;
        if (early && stopped(e)) y = -INFINITY;
        const u64 key = (u64)ordered(y) << 32 | (uint32_t)~(uint32_t)(v0 + e * 32);
        const u64 last = from_lane(list, K - 1);  // (by all lanes: not within a condition)
        const bool pass = (fits >> e & 1u) && y >= least && key > last;
        const unsigned who = __ballot_sync(0xffffffffu, pass);
        if (pass) held[count + __popc(who & ((1u << lane) - 1u))] = key;
        count += __popc(who);
        if (count >= 32) flush();
      }
    }
  }
  if (count) flush();
  s = warp_sum_d(s);
  sh.lists[warp][lane] = list;
  if (lane == 0) { sh.ms[warp] = m; sh.ss[warp] = s; }
  __syncthreads();
#pragma unroll
  for (int w = BW / 2; w > 0; w >>= 1) {
    if (warp < w) {
      list = merged(list, sh.lists[warp + w][lane]);
      if (lane >= K) list = 0;
      sh.lists[warp][lane] = list;
    }
    __syncthreads();
  }
  if (warp == 0) {
    const float top = lane < BW ? sh.ms[lane] : -INFINITY;
    m = warp_max(top);
    s = warp_sum_d(top == -INFINITY ? 0.0 : sh.ss[lane] * (top == m ? 1.0 : exp((double)top - (double)m)));
  }
  return true;
}

// score + log-probability of a token, from its logit, its row's largest and log(sum of exp against it)
__device__ __forceinline__ double continued(double base, float x, float top, double lsum) {
  if (!(x > -INFINITY)) return -(double)INFINITY;
  const double c = base + ((x == top ? 0.0 : (double)x - (double)top) - lsum);
  return c == c ? c : -(double)INFINITY;  // (an infinite score and an impossible token)
}

// What the choice needs of a group's hypotheses, read while the logits are on their way.
struct Group {
  double base[CV3_MAX_BEAMS], norm[CV3_MAX_BEAMS], lsum[CV3_MAX_BEAMS];  // score, length's power, log of the sum
  float tops[CV3_MAX_BEAMS];
  int fins[CV3_MAX_BEAMS], lengths[CV3_MAX_BEAMS];  // 2: finished, 1: does not exist; length of a continuation
};

__device__ void prepare(const BeamArgs& a, int64_t g, Group& w) {
  const int k = threadIdx.x;
  if (k >= a.beams) return;
  const int64_t row = g * a.beams + k;
  const bool fin = a.done[row] != 0;
  const float score = a.scores[row];
  const int length = a.counts[row] + (fin ? 0 : 1);
  w.base[k] = dead(score) ? -INFINITY : (double)score;
  w.norm[k] = a.alpha == 0.0 ? 1.0 : pow((double)max(length, 1), a.alpha);
  w.fins[k] = fin ? 2 : dead(score);
  w.lengths[k] = length;
}

// The group's choice by one CTA, from its tasks' results (global or shared memory).
__device__ void choose(const BeamArgs& a, int64_t g, const char* work, Group& w) {
  __shared__ Cand lists[BW][32];
  const int K = a.beams, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t tb = task_bytes(K);
  for (int k = warp; k < K; k += BW) {
    if (w.fins[k]) continue;
    const char* from = work + (int64_t)k * a.chunks * tb;
    float m = -INFINITY;
    double s = 0.0;
    for (int c = lane; c < a.chunks; c += 32) m = fmaxf(m, *reinterpret_cast<const float*>(from + c * tb + 8));
    m = warp_max(m);
    for (int c = lane; c < a.chunks; c += 32) {
      const float t = *reinterpret_cast<const float*>(from + c * tb + 8);
      if (t > -INFINITY) s += *reinterpret_cast<const double*>(from + c * tb) * (t == m ? 1.0 : exp((double)t - (double)m));
    }
    s = warp_sum_d(s);
    if (lane == 0) {
      w.tops[k] = m;
      w.lsum[k] = log(s);
    }
  }
  __syncthreads();
  // A task's candidates are in descending order, so a warp takes its tasks' first ones before the next ones and
  // stops when none is among its best K: `ranks` of every task at a time, as many as 256 lanes hold.
  Cand list = {0, 0};
  const int tasks = a.chunks * K, ranks = max(1, min(K, BT / tasks)), all = tasks * ranks;
  bool first = true;
  for (int i0 = warp * 32; i0 < all; i0 += BT) {
    const int task = (i0 + lane) / ranks, k = min(task / a.chunks, K - 1);
    const int fin = w.fins[k];
    const bool scanned = task < tasks && !fin, alone = task < tasks && fin && task == k * a.chunks;
    const u64* from = reinterpret_cast<const u64*>(work + (int64_t)task * tb + 16);
    int r = (i0 + lane) % ranks;
    u64 u = scanned && r < K ? from[r] : 0ull;
    for (int r0 = 0; r0 < K; r0 += ranks) {
      const u64 next = scanned && r + ranks < K ? from[r + ranks] : 0ull;
      Cand c = {0, 0};
      if (u) {
        const uint32_t logit = (uint32_t)(u >> 32), token = ~(uint32_t)u;
        c.key = ordered(continued(w.base[k], unordered(logit), w.tops[k], w.lsum[k]) / w.norm[k]);
        c.place = place_of(k, c.key > ordered(-(double)INFINITY) ? logit : ordered(-INFINITY), token);
      } else if (alone && r < K && r < a.vocab) {  // a finished one itself, then what stands in where nothing is left
        c.key = ordered(r == 0 && fin == 2 ? w.base[k] / w.norm[k] : -(double)INFINITY);
        c.place = place_of(k, ordered(-INFINITY), r);
      }
      u = next;
      r += ranks;
      const Cand last = from_lane(list, K - 1);
      if (!__any_sync(0xffffffffu, better(c, last))) break;
      list = first ? sorted(c) : merged(list, sorted(c));
      first = false;
      if (lane >= K) list = Cand{0, 0};
    }
  }
  lists[warp][lane] = list;
  __syncthreads();
#pragma unroll
  for (int half = BW / 2; half > 0; half >>= 1) {
    if (warp < half && half * 32 < all) {  // (warps beyond the candidates have empty lists)
      list = merged(list, lists[warp + half][lane]);
      if (lane >= K) list = Cand{0, 0};
      lists[warp][lane] = list;
    }
    __syncthreads();
  }
  if (warp || lane >= K) return;
  const int k = CV3_MAX_BEAMS - 1 - (int)(list.place >> (TOKEN_BITS + 32));
  const int64_t v = TOKENS - 1 - (uint32_t)(list.place & (TOKENS - 1)), to = g * K + lane;
  const bool fin = w.fins[k] == 2;
  // the key times the length's power is the score again (to the last bits of 64); the outputs may be
  // the inputs' own buffers, of which nothing is read any more
  const double cum = list.key > ordered(-(double)INFINITY) ? (fin ? w.base[k] : unordered(list.key) * w.norm[k]) : -(double)INFINITY;
  a.tokens[to] = fin ? 0 : v;
  a.parents[to] = k;
  a.scores_out[to] = (float)cum;
  a.counts_out[to] = w.lengths[k];
  a.done_out[to] = fin || (v >= a.stop_lo && v < a.stop_hi) ? 1 : 0;
}

// two launches: a CTA per task, then one per group
template <typename T>
__global__ void __launch_bounds__(BT, 3) beam_scan_kernel(const BeamArgs a) {
  __shared__ Scratch sh;
  sh.fill();
  dep_wait();
  dep_release();
  const int64_t row = blockIdx.y;
  u64 list;
  float m;
  double s;
  if (scan<T>(a, row, blockIdx.x, sh, list, m, s) && threadIdx.x < 32) {
    char* w = a.work + (row * a.chunks + blockIdx.x) * task_bytes(a.beams);
    if (threadIdx.x < a.beams) reinterpret_cast<u64*>(w + 16)[threadIdx.x] = list;
    if (threadIdx.x == 0) {
      *reinterpret_cast<double*>(w) = s;
      *reinterpret_cast<float*>(w + 8) = m;
    }
  }
}

__global__ void __launch_bounds__(BT) beam_pick_kernel(const BeamArgs a) {
  __shared__ Group w;
  dep_wait();
  dep_release();
  const int64_t g = blockIdx.x;
  prepare(a, g, w);
  __syncthreads();
  choose(a, g, a.work + g * a.beams * a.chunks * task_bytes(a.beams), w);
}

__device__ __forceinline__ void put8(uint32_t at, u64 x) {
  asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(at), "l"(x) : "memory");
}

// one launch: a cluster per group shares its tasks; the results go to the first CTA's shared memory
template <typename T>
__global__ void __launch_bounds__(BT) beam_cluster_kernel(const BeamArgs a, int cluster) {
  extern __shared__ __align__(16) char work[];
  __shared__ Scratch sh;
  __shared__ Group w;
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  sh.fill();
  dep_wait();
  dep_release();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // every CTA of the cluster runs
  const int64_t g = blockIdx.x / cluster;
  const int rank = blockIdx.x % cluster;
  uint32_t first;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(first) : "r"((uint32_t)__cvta_generic_to_shared(work)));
  if (rank == 0) prepare(a, g, w);
  for (int i = rank; i < a.beams * a.chunks; i += cluster) {
    u64 list;
    float m;
    double s;
    if (scan<T>(a, g * a.beams + i / a.chunks, i % a.chunks, sh, list, m, s) && threadIdx.x < 32) {
      const uint32_t at = first + (uint32_t)(i * task_bytes(a.beams));
      if (threadIdx.x < a.beams) put8(at + 16 + threadIdx.x * 8, list);
      if (threadIdx.x == 0) {
        put8(at, __double_as_longlong(s));
        put8(at + 8, __float_as_uint(m));
      }
    }
  }
  cv3p::cluster_sync();
  if (rank == 0) choose(a, g, work, w);
}

// How a call is cut.  One launch with a cluster per group where each of its CTAs has one task, every warp then walks
// at most 4 tiles for every hypothesis that a CTA stands for, and the clusters take at most three CTAs for two SMs; else two,
// measured (one / two, fp32, us): 1 x 4 hypotheses of 6761 tokens 9.0 / 9.9, 16 x 8 of them 11.4 / 11.3, 100 x 1 9.1 / 10.2;
// 1 x 16 21.5 / 14.8 (two tasks a CTA), 32 x 8 13.2 / 12.8 and 100 x 4 21.9 / 13.1 (more CTAs), 4 x 8 of 20000 13.7 / 13.8, 1 x 4
// of 151936 27.2 / 11.7.
//
// Two launches: as many chunks as one wave of three CTAs on every SM takes, or one more that overshoots it by
// at most a third of a chunk's share: with every row live that costs nothing on average, and as soon as some are finished, whose CTAs
// leave early, it is faster.  Rows of 151936, the wave's chunks / one more, none finished and a seventh finished: 112 rows
// 33.8 / 33.5 and 33.3 / 28.7 us, 120 33.9 / 35.7 and 33.6 / 29.2, 152 43.4 / 42.0 and 42.3 / 34.1, 224 57.3 / 55.4 and 56.6 / 44.7,
// 256 57.2 / 56.3 and 56.7 / 44.8; past that third 128 rows 33.9 / 38.3 and 33.8 / 29.3, 144 34.6 / 39.6 and 34.0 / 38.1.
// But a chunk has 8 + 2 K tiles: the bar takes K maxima, and every chunk gives the second
// launch K candidates (151936 tokens, half as many tiles / such chunks / 16 + 3 K: 4 hypotheses 10.8 / 11.4 / 13.1 us, 8 of them 15.5
// / 14.4 / 15.8, 16 26.5 / 23.4 / 22.0, 32 34.9 / 31.9 / 38.1).
struct Plan {
  int64_t cluster, chunks, tiles, bytes;  // cluster 0: two launches; bytes of results
};
constexpr int64_t TILES_LEAST = 8, TILES_BEAM = 2;
constexpr int64_t CLUSTER = 8, CLUSTER_TILES = 4;

Plan plan_of(int64_t groups, int64_t beams, int64_t vocab) {
  Plan p = {};
  const int64_t row = (vocab + TILE - 1) / TILE;  // tiles of a row
  auto cut = [&](int64_t chunks) {
    chunks = std::max(chunks, (row + TILES_MOST - 1) / TILES_MOST);
    p.tiles = (std::max<int64_t>(1, (row + chunks - 1) / chunks) + BW - 1) / BW * BW;
    p.chunks = (row + p.tiles - 1) / p.tiles;
  };
  if (beams <= CLUSTER && beams * ((row + BW - 1) / BW) <= CLUSTER * CLUSTER_TILES) {
    cut(CLUSTER / beams);
    p.cluster = beams * p.chunks;
    while (p.cluster & (p.cluster - 1)) ++p.cluster;  // a power of two
    if (2 * groups * p.cluster > 3 * cv3::sm_count()) p.cluster = 0;
  }
  if (!p.cluster) {
    const int64_t rows = groups * beams, wave = 3 * cv3::sm_count();
    int64_t chunks = std::max<int64_t>(1, wave / rows);
    if (rows * (chunks + 1) <= wave + wave / (3 * (chunks + 1))) ++chunks;
    cut(std::max<int64_t>(1, std::min(chunks, row / (TILES_LEAST + TILES_BEAM * beams))));
  }
  p.bytes = (p.cluster ? 1 : groups) * beams * p.chunks * task_bytes(beams);
  return p;
}

template <typename T>
int launch(const BeamArgs& a, const Plan& plan, int64_t groups, cudaStream_t st) {
  if (plan.cluster) {
    int rc = cv3::allow_smem((const void*)beam_cluster_kernel<T>, (int)plan.bytes);
    if (rc) return rc;
    return cv3::check_launch("beam_select",
                             cv3p::launch_cluster(beam_cluster_kernel<T>, dim3((unsigned)(groups * plan.cluster)), dim3(BT),
                                                  (size_t)plan.bytes, (unsigned)plan.cluster, st, a, (int)plan.cluster));
  }
  int rc = cv3::check_launch("beam_scan", cv3::launch_dep(beam_scan_kernel<T>, dim3((unsigned)plan.chunks, (unsigned)(groups * a.beams)),
                                                          dim3(BT), 0, st, a));
  if (rc) return rc;
  return cv3::check_launch("beam_pick", cv3::launch_dep(beam_pick_kernel, dim3((unsigned)groups), dim3(BT), 0, st, a));
}

}  // namespace

extern "C" int64_t cv3_beam_workspace(int64_t groups, int64_t beams, int64_t vocab) {
  if (groups <= 0 || beams <= 0 || beams > CV3_MAX_BEAMS || vocab <= 0) return 0;
  const Plan p = plan_of(groups, beams, vocab);
  return p.cluster ? 0 : p.bytes;
}

extern "C" int cv3_beam_select(const cv3_beam_params* p, void* stream) {
  CV3_REQUIRE(p && p->size == (int64_t)sizeof(*p), CV3_ERR_VALUE, "beam_select: bad parameter block");
  CV3_REQUIRE(p->groups >= 0 && p->vocab > 0 && p->ld >= p->vocab && p->stop_lo <= p->stop_hi,
              CV3_ERR_VALUE, "beam_select: bad shape");
  CV3_REQUIRE(p->beams > 0 && p->beams <= CV3_MAX_BEAMS, CV3_ERR_UNSUPPORTED, "beam_select: %lld beams (1 to %d)",
              (long long)p->beams, CV3_MAX_BEAMS);
  CV3_REQUIRE(p->vocab <= TOKENS, CV3_ERR_UNSUPPORTED, "beam_select: %lld tokens (up to 2^27)", (long long)p->vocab);
  CV3_REQUIRE(cv3p::type_ok(p->type), CV3_ERR_VALUE, "beam_select: unknown element type");
  // (lengths to that power stay finite and above 0 in 64 bits)
  CV3_REQUIRE(p->length_penalty >= -16.0 && p->length_penalty <= 16.0, CV3_ERR_VALUE,
              "beam_select: length penalty %g (-16 to 16)", p->length_penalty);
  CV3_REQUIRE(p->groups <= 65535 && p->groups * p->beams <= 65535, CV3_ERR_UNSUPPORTED,
              "beam_select: more than 65535 hypotheses");
  CV3_REQUIRE((uintptr_t)p->logits % cv3p::type_size(p->type) == 0, CV3_ERR_VALUE, "beam_select: misaligned logits");
  if (p->groups == 0) return CV3_OK;
  const Plan plan = plan_of(p->groups, p->beams, p->vocab);
  CV3_REQUIRE(plan.cluster || (p->workspace && p->workspace_bytes >= plan.bytes && ((uintptr_t)p->workspace & 7) == 0),
              CV3_ERR_VALUE, "beam_select: the workspace must hold cv3_beam_workspace() bytes");
  const BeamArgs a = {p->logits, p->ld, (int)p->beams, p->vocab, p->scores, p->counts, p->done, p->stop_lo, p->stop_hi,
                      p->min_len, p->length_penalty, p->tokens, p->parents, p->scores_out, p->counts_out, p->done_out,
                      (int)plan.chunks, plan.tiles, static_cast<char*>(p->workspace)};
  cudaStream_t st = cv3::as_stream(stream);
  if (p->type == CV3_TYPE_F32) return launch<float>(a, plan, p->groups, st);
  if (p->type == CV3_TYPE_F16) return launch<__half>(a, plan, p->groups, st);
  return launch<__nv_bfloat16>(a, plan, p->groups, st);
}
