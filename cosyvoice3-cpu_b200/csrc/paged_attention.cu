// Attention of one new token per request over its paged key/value cache.
//
// out[b][h] = sum_j p_j V[j], p = softmax(scale * q[b][h] . K[j]) over the request's cached keys j
// in [max(0, len - window), len); a request without keys gives zeros and a log-sum of -inf.
//
// Bound by the cache's bytes: every key and value is read once for the up to 8 query heads that share
// it.  Three choices follow.
//
// 1. Work is cut evenly, whatever the lengths.  A pair (request, group of up to 8 heads of a kv head)
//    has ceil(keys / TK) tiles; all pairs' tiles in order form one line, of which the grid's CTAs take
//    equal pieces (found from the lengths on the device, so a captured launch follows them).  A CTA meets at most two pairs that it does not hold whole -- the one that began before
//    its piece and the one that goes on behind it -- and leaves their partial results (running
//    maximum, sum, unnormalised output) in two slots; a second launch joins the slots of every pair
//    that was cut, in CTA order, so the result does not depend on timing.  Short caches, whose cost
//    is latency, take one launch instead: a cluster of CTAs per pair, joined through shared memory.
// 2. One pass, nothing staged.  A warp takes KI keys of each tile with matrix instructions whose
//    operands come straight from global memory into registers: the keys' and values' 16-byte pieces
//    land in the lanes that need them because the order in which head dimensions (for q.k) and the
//    order in which output columns (for p.v) enter a product is free.
// 3. fp32 arithmetic on the tf32 matrix pipe.  fp16 and bf16 keys and values are tf32 numbers
//    exactly; fp32 ones are split into two (the low 13 bits apart).  The products have 16 rows and at
//    most 8 heads, so rows 0..7 hold the upper tf32 part of q (then of p) and rows 8..15 the lower
//    part: 22 bits of both at no cost.  The matrix pipe truncates when it adds, so only one tile's
//    p.v is summed there; tiles are added in fp32 registers, the softmax's rescaling on the way.
//    Queries of the cache's own 16-bit type need less: 16-bit products, exact for q.k, and p in two
//    16-bit parts, whose 2^-16 (bf16) or 2^-22 (fp16) is far below the result's rounding (64 ragged requests: 377 instead of
//    404 us).
//
// Measured: 64 requests of 1 to 16384 keys, 32 / 8 heads of 128, bf16 (2.15 GB): 346 us, 6.2 TB/s (390 us
// when it runs on and on and the card's power limit lowers its clock; fp16 355 us); 32 of 64 to 1650 keys, 14 / 2
// heads of 64, fp32 (28 MB): 14.8 us, up to four steps of the longest request, each its loads' latency and its
// products, behind the chain length -> table -> keys; one of 325 keys: 6.0 us.
#include <algorithm>
#include <type_traits>

#include "paged.cuh"

namespace {

struct AttnArgs {
  const void* q;
  int q_type;
  int64_t qsb, qsh;
  const void *k, *v;
  int64_t ksp, ksh, kst, vsp, vsh, vst, pages;
  int ps;
  uint32_t ps_mul, ps_shift;  // n / ps = (n * ps_mul) >> ps_shift for 0 <= n < 2^31 (64-bit product)
  const int* tables;
  int64_t ld;
  int max_keys;  // columns * page size
  const int* lens;
  int batch, heads, kv_heads, group, groups;  // group: heads per kv head; groups: of up to 8 of them
  int window;
  float scale;
  void* out;
  int64_t osb, osh;
  float* lse;
  int* bad;
  float* part;  // [CTA][2][8][D] unnormalised outputs
  float* stat;  // [CTA][2][8][2] maximum (base 2) and sum
  int2* cut;    // [pair] first CTA and number of CTAs (0: nothing to join)
};

constexpr int NW = 8;                  // warps of a CTA, each with KI keys of every tile
constexpr int HT = 8;                  // query heads of a CTA (rows of a product that are not lower parts)
constexpr float LOG2E = 1.4426950408889634f;
constexpr float TINY = 1e-37f;         // stands for a lower part of 0, so that 0 * inf does not arise

// Keys of a warp's step: 4 to 8 KB of keys and values for the warp, which with two CTAs per SM (128
// registers a thread; one CTA with more: 438 instead of 366 us for 64 ragged requests) keeps enough
// loads in flight.  (32 keys of 128 bytes, 8 KB too, spill: one 38399-key bf16 context took 20.4
// instead of 16.7 us.)
template <typename KT, int D>
constexpr int keys_per_step() {
  return D * (int)sizeof(KT) <= 64 ? 32 : D * (int)sizeof(KT) <= 256 ? 16 : 8;
}

__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename KT>
__device__ __forceinline__ void mma_16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<KT, __nv_bfloat16>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Two probabilities as 16-bit parts: the upper ones, and what these leave (never 0, so that 0 * inf does not
// arise).  bf16 has fp32's exponents: 16 bits of any probability, TINY where nothing is left.  fp16 begins at 6e-8, and
// many keys behind a dominating one may have less each: the upper parts are those of p * P16, the lower ones are raised by
// R16 once more, both powers of two that go out of the sums again.  22 bits of p down to 2^-28, 2^-50 below; 2^-49 for 0.
template <typename KT>
constexpr float P16 = std::is_same<KT, __half>::value ? 16384.f : 1.f;
template <typename KT>
constexpr float R16 = std::is_same<KT, __half>::value ? 2048.f : 1.f;

template <typename KT>
__device__ __forceinline__ void split_16(float x, float y, uint32_t& hi, uint32_t& lo) {
  if constexpr (std::is_same<KT, __nv_bfloat16>::value) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    const float rx = x - __uint_as_float(hi << 16), ry = y - __uint_as_float(hi & 0xFFFF0000u);
    const __nv_bfloat162 l = __floats2bfloat162_rn(rx == 0.f ? TINY : rx, ry == 0.f ? TINY : ry);
    lo = *reinterpret_cast<const uint32_t*>(&l);
  } else {
    x *= P16<KT>;
    y *= P16<KT>;
    const __half2 h = __floats2half2_rn(x, y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    const float2 back = __half22float2(h);
    const __half2 l = __floats2half2_rn((x - back.x) * R16<KT>, (y - back.y) * R16<KT>);
    lo = *reinterpret_cast<const uint32_t*>(&l);
    lo |= (lo & 0x7FFFu ? 0u : 1u) | (lo & 0x7FFF0000u ? 0u : 0x10000u);
  }
}

__device__ __forceinline__ uint32_t tf32_hi(uint32_t x) { return x & 0xFFFFE000u; }

__device__ __forceinline__ float exp2_fast(float x) {  // relative error 2^-22
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <int BYTES>
struct Raw;
template <>
struct Raw<16> { uint32_t r[4]; };
template <>
struct Raw<32> { uint32_t r[8]; };
template <>
struct Raw<8> { uint32_t r[2]; };

__device__ __forceinline__ void fetch(Raw<32>& x, const void* p, bool ok) {
#pragma unroll
  for (int i = 0; i < 8; ++i) x.r[i] = 0u;
  if (ok)
    asm volatile("ld.global.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(x.r[0]), "=r"(x.r[1]), "=r"(x.r[2]), "=r"(x.r[3]), "=r"(x.r[4]), "=r"(x.r[5]), "=r"(x.r[6]),
                   "=r"(x.r[7])
                 : "l"(p));
}

__device__ __forceinline__ void fetch(Raw<16>& x, const void* p, bool ok) {
  x.r[0] = x.r[1] = x.r[2] = x.r[3] = 0u;
  if (ok)
    asm volatile("ld.global.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(x.r[0]), "=r"(x.r[1]), "=r"(x.r[2]), "=r"(x.r[3]) : "l"(p));
}
__device__ __forceinline__ void fetch(Raw<8>& x, const void* p, bool ok) {
  x.r[0] = x.r[1] = 0u;
  if (ok) asm volatile("ld.global.L1::no_allocate.v2.b32 {%0,%1}, [%2];" : "=r"(x.r[0]), "=r"(x.r[1]) : "l"(p));
}

// element e of a piece as fp32 bits
template <typename KT, int B>
__device__ __forceinline__ uint32_t element(const Raw<B>& x, int e) {
  if constexpr (sizeof(KT) == 4) {
    return x.r[e];
  } else if constexpr (std::is_same<KT, __nv_bfloat16>::value) {
    return e & 1 ? x.r[e >> 1] & 0xFFFF0000u : x.r[e >> 1] << 16;
  } else {
    const __half h = __ushort_as_half((unsigned short)(e & 1 ? x.r[e >> 1] >> 16 : x.r[e >> 1] & 0xFFFFu));
    return __float_as_uint(__half2float(h));
  }
}

// what the upper tf32 part leaves of x (NaN of an infinity: sums of such products count as 0)
__device__ __forceinline__ uint32_t tf32_rest(uint32_t x) {
  return __float_as_uint(__uint_as_float(x) - __uint_as_float(tf32_hi(x)));
}
// the same, rounded to the nearest tf32 by the pipe, which drops the low 13 bits (of an infinity: 0): at most 2^-22
// of a key, value, query or probability is lost.  The plain rest loses up to 3 * 2^-23, always towards 0: with it
// the worst relative error of 325 to 30000 keys was 1.5e-6 (values only: 5.1e-7) instead of 4.7e-7, fp32's own being
// 0.5 to 2.6e-6; the values' rounding costs 1% (one utterance 6.6 instead of 6.5 us, 32 of them 15.4 instead of 15.3).
__device__ __forceinline__ uint32_t tf32_near(uint32_t x) { return tf32_rest(x) + 0x1000u; }
__device__ __forceinline__ float or_zero(float x) { return x == x ? x : 0.f; }

__device__ __forceinline__ int page_index(const AttnArgs& a, int key) {
  return (int)(((uint64_t)(uint32_t)key * a.ps_mul) >> a.ps_shift);
}

// first visible key and end of request b
__device__ __forceinline__ void visible(const AttnArgs& a, int b, int& lo, int& hi) {
  hi = min(max(a.lens[b], 0), a.max_keys);
  lo = a.window > 0 ? max(hi - a.window, 0) : 0;
}

// UNI: page_size is a multiple of 16, so 16 (or 8) keys from a multiple of 16 share a page.
// H16: the queries have the cache's 16-bit type.
// CL: clusters of gridDim / pairs CTAs, one per pair, instead of even pieces of the line.
template <typename KT, int D, bool UNI, bool H16, bool CL>
__global__ void __launch_bounds__(NW * 32, 2) paged_attention_kernel(const AttnArgs a) {
  constexpr int KI = keys_per_step<KT, D>(), NT = KI / 8, TK = NW * KI;
  constexpr bool WIDE = sizeof(KT) == 4;          // keys and values need a lower part
  // a key piece: 32 bytes where 4 lanes' pieces fill whole rows (a 128-byte line per key and load), else 16
  constexpr int KB = D * (int)sizeof(KT) % 128 == 0 ? 32 : 16;
  constexpr int KE = KB / (int)sizeof(KT);        // its elements; 4 lanes cover 4 * KE dimensions
  constexpr int KC = D / (4 * KE);
  constexpr int VE = sizeof(KT) == 2 && D % 64 == 0 ? 8 : 4;  // of a value piece; 8 lanes cover 8 * VE
  constexpr int VC = D / (8 * VE);
  constexpr int VB = VE * (int)sizeof(KT);
  constexpr int GK = UNI ? (KI >= 16 ? KI / 16 : 1) : NT;  // page lookups of a step: per 16 keys, or per 8 and row
  constexpr int QS = H16 ? D / 16 : D / 8, QW = H16 ? 2 : 4;  // steps of q.k, words of a lane's operand
  __shared__ __align__(16) uint32_t sq[QS][32][QW];  // q as product operands; H16: rows 0..7, else lower parts in 8..15
  __shared__ float so[NW][HT][D + 1];  // (rows apart by 1 bank: the 8 heads of a store fall into different ones)
  __shared__ float sm[NW][HT], sl[NW][HT];
  dep_wait();
  dep_release();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, n = lane >> 2, t = lane & 3;
  const int per = a.kv_heads * a.groups;  // pairs of a request
  const int c = blockIdx.x;

  // a pair's queries as product operands in shared memory
  auto queries = [&](int b, int h0, int nh) {
    for (int i = tid; i < QS * 32; i += NW * 32) {
      const int s = i >> 5, ln = i & 31, row = ln >> 2;
      const int64_t at = b * a.qsb + (h0 + row) * a.qsh;
      if constexpr (H16) {  // four dimensions of a key piece per step, two in a word
        const int d = s / (KE / 4) * 4 * KE + (ln & 3) * KE + s % (KE / 4) * 4;
        const unsigned short* q = static_cast<const unsigned short*>(a.q) + at + d;
#pragma unroll
        for (int e = 0; e < 2; ++e) sq[s][ln][e] = row < nh ? q[2 * e] | (uint32_t)q[2 * e + 1] << 16 : 0u;
      } else {
        const int d = s / (KE / 2) * 4 * KE + (ln & 3) * KE + s % (KE / 2) * 2;
        uint32_t v[4] = {0u, 0u, 0u, 0u};
        if (row < nh) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float x = cv3p::load_any(a.q, a.q_type, at + d + e) * (a.scale * LOG2E);
            const uint32_t r = __float_as_uint(or_zero(__uint_as_float(tf32_near(__float_as_uint(x)))));
            v[2 * e] = tf32_hi(__float_as_uint(x));
            v[2 * e + 1] = (r & 0x7FFFE000u) ? r : __float_as_uint(copysignf(TINY, x));
          }
        }
        *reinterpret_cast<uint4*>(&sq[s][ln][0]) = make_uint4(v[0], v[1], v[2], v[3]);
      }
    }
  };

  // Table entries that a step's lookups need: UNI: of its 16-key groups; else of the rows that this lane
  // reads: key n, values 2t and 2t + 1 of each 8 keys.  Only the table's own bounds are looked at, so the
  // first step's entries may be fetched before the request's length is known.
  int ent[GK][UNI ? 1 : 3];
  auto peek = [&](const int* table, int key0) {
    auto entry = [&](int key) -> int { return key < a.max_keys ? table[page_index(a, key)] : -1; };
#pragma unroll
    for (int i = 0; i < GK; ++i) {
      if constexpr (UNI) {
        ent[i][0] = entry(key0 + i * 16);
      } else {
        ent[i][0] = entry(key0 + i * 8 + n);
        ent[i][1] = entry(key0 + i * 8 + 2 * t);
        ent[i][2] = entry(key0 + i * 8 + 2 * t + 1);
      }
    }
  };

  // Tiles t0, t0 + every, ... below t1 of a pair (the first's entries peeked at): the warps' maxima, sums and
  // unnormalised outputs to shared memory.  The queries are there, but for the barrier.
  auto attend = [&](int b, int pair, int lo, int hi, int g, int t0, int t1, int every) {
    const KT* kb = static_cast<const KT*>(a.k) + g * a.ksh + t * KE + (UNI ? n * a.kst : 0);
    const KT* vb = static_cast<const KT*>(a.v) + g * a.vsh + n * VE + (UNI ? 2 * t * a.vst : 0);
    const int* table = a.tables + b * a.ld;
    const bool counts = a.bad && pair == 0;
    float o[D / 8][2], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = 0.f;

    Raw<KB> kr[NT][KC];
    Raw<VB> vr[NT][2][VC];
    const int base = lo & -KI, first = base + t0 * TK + warp * KI, end = min(hi, base + t1 * TK), ahead = every * TK;
    // the pages of a step from its table entries, -1 for none
    int pg[GK][UNI ? 1 : 3];
    auto settle = [&](int key0) {
      // key: the first that this lookup stands for; mine: this lane counts a bad entry
      auto page = [&](int entry, int key, bool mine) -> int {
        if (key < lo || key >= hi) return -1;
        const bool ok = (unsigned)entry < (unsigned)a.pages;
        if (!ok && counts && mine && (key == lo || key == page_index(a, key) * a.ps)) atomicAdd(a.bad, 1);
        return ok ? entry : -1;
      };
#pragma unroll
      for (int i = 0; i < GK; ++i) {
        if constexpr (UNI) {
          const int k0 = key0 + i * 16;
          pg[i][0] = k0 + min(KI, 16) > lo ? page(ent[i][0], max(k0, lo), lane == 0) : -1;
        } else {
          pg[i][0] = page(ent[i][0], key0 + i * 8 + n, false);
          pg[i][1] = page(ent[i][1], key0 + i * 8 + 2 * t, n == 0);
          pg[i][2] = page(ent[i][2], key0 + i * 8 + 2 * t + 1, n == 0);
        }
      }
    };
    auto row_of = [&](int key) -> int { return key - page_index(a, key) * a.ps; };
    // UNI: kb and vb point at this lane's first row and piece of a 16-key group, which lies in one page
    auto load_k = [&](int key0) {
      if constexpr (UNI) {
#pragma unroll
        for (int x = 0; x < GK; ++x) {
          const KT* src = kb + (int64_t)pg[x][0] * a.ksp + (int64_t)row_of(key0 + x * 16) * a.kst;
#pragma unroll
          for (int i = 0; i < (NT < 2 ? NT : 2); ++i) {
            const int key = key0 + x * 16 + i * 8 + n;
            const bool ok = pg[x][0] >= 0 && key >= lo && key < hi;
#pragma unroll
            for (int c = 0; c < KC; ++c) fetch(kr[2 * x + i][c], src + i * 8 * a.kst + c * 4 * KE, ok);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          const int key = key0 + i * 8 + n;
          const KT* src = kb + (int64_t)pg[i][0] * a.ksp + (int64_t)row_of(key) * a.kst;
#pragma unroll
          for (int c = 0; c < KC; ++c) fetch(kr[i][c], src + c * 4 * KE, pg[i][0] >= 0);
        }
      }
    };
    auto load_v = [&](int key0) {
      if constexpr (UNI) {
#pragma unroll
        for (int x = 0; x < GK; ++x) {
          const KT* src = vb + (int64_t)pg[x][0] * a.vsp + (int64_t)row_of(key0 + x * 16) * a.vst;
#pragma unroll
          for (int i = 0; i < (NT < 2 ? NT : 2); ++i)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const int key = key0 + x * 16 + i * 8 + 2 * t + r;
              const bool ok = pg[x][0] >= 0 && key >= lo && key < hi;
#pragma unroll
              for (int c = 0; c < VC; ++c) fetch(vr[2 * x + i][r][c], src + (i * 8 + r) * a.vst + c * 8 * VE, ok);
            }
        }
      } else {
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int key = key0 + i * 8 + 2 * t + r;
            const KT* src = vb + (int64_t)pg[i][1 + r] * a.vsp + (int64_t)row_of(key) * a.vst;
#pragma unroll
            for (int c = 0; c < VC; ++c) fetch(vr[i][r][c], src + c * 8 * VE, pg[i][1 + r] >= 0);
          }
      }
    };

    if (first < end) {
      settle(first);
      load_k(first);
    }
    __syncthreads();  // the queries are in shared memory; what it held before is done with
    for (int key0 = first; key0 < end; key0 += ahead) {
      load_v(key0);
      const int next = key0 + ahead;
      if (next < end) peek(table, next);
      float s0[NT][4], s1[NT][4];  // two chains: even and odd steps, or upper and lower parts of the keys
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) s0[i][e] = s1[i][e] = 0.f;
      if constexpr (H16) {
#pragma unroll
        for (int s = 0; s < QS; ++s) {
          const uint2 q2 = *reinterpret_cast<const uint2*>(&sq[s][lane][0]);
          const uint32_t qa[4] = {q2.x, 0u, q2.y, 0u};
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            const auto& piece = kr[i][s / (KE / 4)];
            mma_16<KT>(s & 1 ? s1[i] : s0[i], qa, piece.r[s % (KE / 4) * 2], piece.r[s % (KE / 4) * 2 + 1]);
          }
        }
      } else {
#pragma unroll
        for (int s = 0; s < D / 8; ++s) {
          const uint4 q4 = *reinterpret_cast<const uint4*>(&sq[s][lane][0]);
          const uint32_t qa[4] = {q4.x, q4.y, q4.z, q4.w};
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            const uint32_t b0 = element<KT>(kr[i][s / (KE / 2)], s % (KE / 2) * 2);
            const uint32_t b1 = element<KT>(kr[i][s / (KE / 2)], s % (KE / 2) * 2 + 1);
            if constexpr (WIDE) {
              mma_tf32(s0[i], qa, tf32_hi(b0), tf32_hi(b1));
              mma_tf32(s1[i], qa, tf32_near(b0), tf32_near(b1));
            } else {
              mma_tf32(s & 1 ? s1[i] : s0[i], qa, b0, b1);
            }
          }
        }
      }
      float top = m, sc[NT][2];  // this lane's scores: keys 2t, 2t + 1 of each 8
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float rest = s1[i][r] + s1[i][2 + r];
          const float x = H16 ? (s0[i][r] + s1[i][r]) * (a.scale * LOG2E)
                              : (s0[i][r] + s0[i][2 + r]) + (WIDE ? or_zero(rest) : rest);
          const int key = key0 + i * 8 + 2 * t + r;
          const bool seen = (UNI ? pg[i / 2][0] : pg[i][1 + r]) >= 0 && key >= lo && key < hi;
          sc[i][r] = seen ? x : -INFINITY;
          top = fmaxf(top, sc[i][r]);
        }
      if (next < end) {
        settle(next);
        load_k(next);
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const float ref = top == -INFINITY ? 0.f : top;
      const float fade = exp2_fast(m - ref);
      m = top;
      l *= fade;
      float pr[NT][2];
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          pr[i][r] = exp2_fast(sc[i][r] - ref);
          l += pr[i][r];
        }
      if constexpr (H16) {
        uint32_t p[NT / 2][4];
#pragma unroll
        for (int i = 0; i < NT; ++i) split_16<KT>(pr[i][0], pr[i][1], p[i / 2][i % 2 * 2], p[i / 2][i % 2 * 2 + 1]);
#pragma unroll
        for (int j = 0; j < D / 8; ++j) {
          float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < NT; i += 2) {
            const int x = j / VE, w = j % VE / 2;
            const uint32_t half = j % 2 ? 0x7632u : 0x5410u;  // a column's values of two keys in a word
            mma_16<KT>(acc, p[i / 2], __byte_perm(vr[i][0][x].r[w], vr[i][1][x].r[w], half),
                       __byte_perm(vr[i + 1][0][x].r[w], vr[i + 1][1][x].r[w], half));
          }
          o[j][0] = fmaf(o[j][0], fade, fmaf(acc[2], 1.f / R16<KT>, acc[0]));
          o[j][1] = fmaf(o[j][1], fade, fmaf(acc[3], 1.f / R16<KT>, acc[1]));
        }
      } else {
        uint32_t p[NT][4];
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            p[i][2 * r] = tf32_hi(__float_as_uint(pr[i][r]));
            p[i][2 * r + 1] = __float_as_uint(fmaxf(pr[i][r] - __uint_as_float(p[i][2 * r]), TINY)) + 0x1000u;
          }
#pragma unroll
        for (int j = 0; j < D / 8; ++j) {
          float acc[4] = {0.f, 0.f, 0.f, 0.f}, low[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            const uint32_t b0 = element<KT>(vr[i][0][j / VE], j % VE), b1 = element<KT>(vr[i][1][j / VE], j % VE);
            if constexpr (WIDE) {
              mma_tf32(acc, p[i], tf32_hi(b0), tf32_hi(b1));
              mma_tf32(low, p[i], tf32_near(b0), tf32_near(b1));
            } else {
              mma_tf32(acc, p[i], b0, b1);
            }
          }
          float y0 = acc[0] + acc[2], y1 = acc[1] + acc[3];
          if constexpr (WIDE) {
            y0 += or_zero(low[0] + low[2]);
            y1 += or_zero(low[1] + low[3]);
          }
          o[j][0] = fmaf(o[j][0], fade, y0);
          o[j][1] = fmaf(o[j][1], fade, y1);
        }
      }
    }

    // the warps' shares of the pair
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if (t == 0) { sm[warp][n] = m; sl[warp][n] = l; }
    constexpr float BACK = H16 ? 1.f / P16<KT> : 1.f;
#pragma unroll
    for (int x = 0; x < VC; ++x)
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        so[warp][n][x * 8 * VE + 2 * t * VE + e] = o[x * VE + e][0] * BACK;
        so[warp][n][x * 8 * VE + (2 * t + 1) * VE + e] = o[x * VE + e][1] * BACK;
      }
    __syncthreads();
  };
  // Warp w puts head w's shares together: the lane's D / 32 outputs (every 32nd), in every lane M and L.
  constexpr int E = D / 32;
  auto gather = [&](float& M, float& L, float (&x)[E]) {
    const int h = warp;
    const float m = sm[lane % NW][h], l = sl[lane % NW][h];  // (a warp's sum is NaN where it met a NaN score)
    M = m;
#pragma unroll
    for (int o = NW / 2; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    const float f = l == 0.f ? 0.f : exp2_fast(m - M);
    L = l * f;
#pragma unroll
    for (int o = NW / 2; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float fw = __shfl_sync(0xffffffffu, f, w);
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = fmaf(so[w][h][e * 32 + lane], fw, x[e]);
    }
  };
  auto finish = [&](int b, int h, float M, float L, const float (&x)[E]) {
#pragma unroll
    for (int e = 0; e < E; ++e)
      cv3p::store_any(a.out, a.q_type, b * a.osb + h * a.osh + e * 32 + lane, L == 0.f ? 0.f : x[e] / L);
    if (a.lse && lane == 0) a.lse[(int64_t)b * a.heads + h] = L == 0.f ? -INFINITY : (M + log2f(L)) / LOG2E;
  };
  auto heads_of = [&](int pair, int& g, int& h0, int& nh) {
    g = pair / a.groups;
    h0 = g * a.group + (pair - g * a.groups) * HT;
    nh = min(HT, (g + 1) * a.group - h0);
  };
  auto tiles_of = [&](int b) -> int {
    int lo, hi;
    visible(a, b, lo, hi);
    return hi > lo ? (hi - (lo & -KI) + TK - 1) / TK : 0;
  };

  if constexpr (CL) {
    const int S = gridDim.x / (a.batch * per), rank = c % S;
    const int b = c / S / per, pair = c / S - b * per;
    int lo, hi, g, h0, nh;
    heads_of(pair, g, h0, nh);
    // CTA `rank` has the tiles rank, rank + S, ...: without a window the first one's entries and the queries are
    // on their way before the length is known
    const int* table = a.tables + b * a.ld;
    if (a.window == 0) peek(table, rank * TK + warp * KI);
    queries(b, h0, nh);
    visible(a, b, lo, hi);
    if (a.window != 0) peek(table, (lo & -KI) + rank * TK + warp * KI);
    attend(b, pair, lo, hi, g, rank, tiles_of(b), S);
    float M, L, x[E];
    gather(M, L, x);
    if (S == 1) {
      if (warp < nh) finish(b, h0 + warp, M, L, x);
      return;
    }
    __shared__ float stat[HT][2];
#pragma unroll
    for (int e = 0; e < E; ++e) so[0][warp][e * 32 + lane] = x[e];  // (read by this lane alone so far)
    if (lane == 0) { stat[warp][0] = M; stat[warp][1] = L; }
    cv3p::cluster_sync();
    if (warp % S == rank && warp < nh) {  // the heads are dealt to the CTAs
      const bool there = lane < S;
      const float m = there ? cv3p::cluster_load(&stat[warp][0], lane) : -INFINITY;
      const float l = there ? cv3p::cluster_load(&stat[warp][1], lane) : 0.f;
      float o[8][E];
#pragma unroll
      for (int r = 0; r < 8; ++r)
#pragma unroll
        for (int e = 0; e < E; ++e) o[r][e] = r < S ? cv3p::cluster_load(&so[0][warp][e * 32 + lane], r) : 0.f;
      M = warp_max(m);
      const float f = l == 0.f ? 0.f : exp2_fast(m - M);
      L = warp_sum(l * f);
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = 0.f;
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const float fr = __shfl_sync(0xffffffffu, f, r);
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = fmaf(o[r][e], fr, x[e]);
      }
      finish(b, h0 + warp, M, L, x);
    }
    cv3p::cluster_sync();  // no CTA leaves while another reads its shared memory
    return;
  } else {

  // requests without keys: zeros, nothing to join
  for (int b = c; b < a.batch; b += gridDim.x) {
    if (tiles_of(b)) continue;
    const float zero[E] = {};
    for (int h = warp; h < a.heads; h += NW) finish(b, h, -INFINITY, 0.f, zero);
    for (int i = tid; i < per; i += NW * 32) a.cut[(int64_t)b * per + i] = make_int2(0, 0);
  }

  // the whole line and this CTA's piece of it; every warp finds it by itself
  int64_t W = 0;
  for (int b = lane; b < a.batch; b += 32) W += tiles_of(b);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) W += __shfl_xor_sync(0xffffffffu, W, o);
  W *= per;
  const int64_t share = (W + gridDim.x - 1) / gridDim.x;
  int64_t u = c * share;
  const int64_t u_end = min(u + share, W);
  if (u >= u_end) return;
  int b = 0;
  int64_t before = 0;  // tiles of the requests before b (one pair each)
  for (int b0 = 0;; b0 += 32) {
    const int64_t mine = b0 + lane < a.batch ? tiles_of(b0 + lane) : 0;
    int64_t sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += x;
    }
    const unsigned past = __ballot_sync(0xffffffffu, (before + sum) * per > u);
    if (past) {
      const int at = __ffs(past) - 1;
      b = b0 + at;
      before += __shfl_sync(0xffffffffu, sum - mine, at);
      break;
    }
    before += __shfl_sync(0xffffffffu, sum, 31);
  }

  // (the walk's state waits in shared memory while the registers serve a pair)
  __shared__ struct { int64_t u, before; int b; } walk;
  __shared__ struct { int b, h0, nh, slot; } now;  // slot -1: a whole pair
  if (tid == 0) { walk.u = u; walk.before = before; walk.b = b; }
  for (;;) {
    __syncthreads();  // the last pair's shared memory is done with
    u = walk.u;
    if (u >= u_end) break;
    before = walk.before;
    b = walk.b;
    int lo, hi, g, h0, nh, pair, tiles;
    for (;;) {  // the pair that u lies in
      tiles = tiles_of(b);
      const int64_t past = u - before * per;
      if (tiles && past < (int64_t)tiles * per) {
        pair = (int)(past / tiles);
        break;
      }
      before += tiles;
      ++b;
    }
    visible(a, b, lo, hi);
    heads_of(pair, g, h0, nh);
    const int64_t u0 = before * per + (int64_t)pair * tiles;
    const int t0 = (int)(u - u0), t1 = (int)min((int64_t)tiles, u_end - u0);
    peek(a.tables + b * a.ld, (lo & -KI) + t0 * TK + warp * KI);
    queries(b, h0, nh);
    __syncthreads();  // everyone has read the walk's state
    if (tid == 0) {
      const bool whole = t0 == 0 && t1 == tiles;
      walk = {u0 + t1, before, b};
      now = {b, h0, nh, whole ? -1 : t0 > 0 ? 0 : 1};
      if (t0 == 0)  // who holds the pair: CTA x has the tiles from x * share on
        a.cut[(int64_t)b * per + pair] = whole ? make_int2(0, 0) : make_int2(c, (int)((u0 + tiles - 1) / share) - c + 1);
    }
    attend(b, pair, lo, hi, g, t0, t1, 1);
    float M, L, x[E];
    gather(M, L, x);
    if (warp < now.nh) {
      if (now.slot < 0) {
        finish(now.b, now.h0 + warp, M, L, x);
      } else {
        const int64_t at = ((int64_t)c * 2 + now.slot) * HT + warp;
#pragma unroll
        for (int e = 0; e < E; ++e) a.part[at * D + e * 32 + lane] = x[e];
        if (lane == 0) { a.stat[at * 2] = M; a.stat[at * 2 + 1] = L; }
      }
    }
  }
  }
}

// Joins the parts of every pair that was cut.  WPH warps share a head: one where there are pairs
// enough to fill the GPU, all of them where few long pairs have many parts each.
template <int D, int WPH>
__global__ void __launch_bounds__(NW * 32) paged_join_kernel(const AttnArgs a) {
  constexpr int E = D / 32;
  __shared__ float so[NW][D], sm[NW], sl[NW];
  dep_wait();
  dep_release();
  const int pair = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = blockIdx.y * (NW / WPH) + warp / WPH;
  const int2 cut = a.cut[pair];
  if (cut.y == 0) return;
  const int per = a.kv_heads * a.groups, b = pair / per, r = pair - b * per;
  const int g = r / a.groups, h0 = g * a.group + (r - g * a.groups) * HT;
  const int nh = min(HT, (g + 1) * a.group - h0);
  float M = -INFINITY, L = 0.f, x[E];
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] = 0.f;
  if (h < nh) {
    // part i: the pair's first CTA left it in slot 1, the others in slot 0
    for (int i0 = warp % WPH; i0 < cut.y; i0 += 4 * WPH) {
      float pm[4], pl[4], px[4][E];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + u * WPH;
        pm[u] = -INFINITY;
        pl[u] = 0.f;
        if (i < cut.y) {
          const int64_t at = ((int64_t)(cut.x + i) * 2 + (i == 0)) * HT + h;
          pm[u] = a.stat[at * 2];
          pl[u] = a.stat[at * 2 + 1];
#pragma unroll
          for (int e = 0; e < E; ++e) px[u][e] = a.part[at * D + e * 32 + lane];
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (pl[u] == 0.f) continue;
        const float top = fmaxf(M, pm[u]), f = L == 0.f ? 0.f : exp2_fast(M - top), w = exp2_fast(pm[u] - top);
        M = top;
        L = L * f + pl[u] * w;
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = x[e] * f + px[u][e] * w;
      }
    }
  }
  if constexpr (WPH > 1) {
#pragma unroll
    for (int e = 0; e < E; ++e) so[warp][e * 32 + lane] = x[e];
    if (lane == 0) { sm[warp] = M; sl[warp] = L; }
    __syncthreads();
    if (warp % WPH) return;
    for (int w = 1; w < WPH; ++w) {
      if (sl[warp + w] == 0.f) continue;
      const float top = fmaxf(M, sm[warp + w]), f = L == 0.f ? 0.f : exp2_fast(M - top), y = exp2_fast(sm[warp + w] - top);
      M = top;
      L = L * f + sl[warp + w] * y;
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = x[e] * f + so[warp + w][e * 32 + lane] * y;
    }
  }
  if (h >= nh) return;
#pragma unroll
  for (int e = 0; e < E; ++e)
    cv3p::store_any(a.out, a.q_type, b * a.osb + (h0 + h) * a.osh + e * 32 + lane, L == 0.f ? 0.f : x[e] / L);
  if (a.lse && lane == 0) a.lse[(int64_t)b * a.heads + h0 + h] = L == 0.f ? -INFINITY : (M + log2f(L)) / LOG2E;
}

using Fn = void (*)(const AttnArgs);

template <typename KT, int D, bool UNI, bool H16>
Fn pick(bool cl) {
  return cl ? paged_attention_kernel<KT, D, UNI, H16, true> : paged_attention_kernel<KT, D, UNI, H16, false>;
}

template <typename KT, int D>
Fn pick(bool uni, bool h16, bool cl) {
  if constexpr (sizeof(KT) == 2)
    if (h16) return uni ? pick<KT, D, true, true>(cl) : pick<KT, D, false, true>(cl);
  return uni ? pick<KT, D, true, false>(cl) : pick<KT, D, false, false>(cl);
}

template <typename KT>
Fn pick(int64_t d, bool uni, bool h16, bool cl) {
  switch (d) {
    case 32: return pick<KT, 32>(uni, h16, cl);
    case 64: return pick<KT, 64>(uni, h16, cl);
    case 96: return pick<KT, 96>(uni, h16, cl);
    default: return pick<KT, 128>(uni, h16, cl);
  }
}

Fn pick_join(int64_t d, bool wide) {
  switch (d) {
    case 32: return wide ? paged_join_kernel<32, NW> : paged_join_kernel<32, 1>;
    case 64: return wide ? paged_join_kernel<64, NW> : paged_join_kernel<64, 1>;
    case 96: return wide ? paged_join_kernel<96, NW> : paged_join_kernel<96, 1>;
    default: return wide ? paged_join_kernel<128, NW> : paged_join_kernel<128, 1>;
  }
}

// Keys of a CTA's tile (keys_per_step of the type and head dimension).
int64_t tile_of(int64_t d, int64_t size) { return NW * (d * size <= 64 ? 32 : d * size <= 256 ? 16 : 8); }

struct Plan {
  int64_t pairs, grid, cluster, floats;  // cluster 0: even pieces and a join
};

// A cluster per pair (as many CTAs as tiles, up to 8 and one wave of two CTAs per SM), or one wave that
// cuts the line into even pieces and a join.  The host knows the table's width only: `steps` is what a
// CTA of a cluster has to do for the longest request, `even` what one of the wave has if all are that
// long.  The join costs about two steps, and only even pieces gain from shorter requests, so clusters
// take up to even + 2 steps and 8 at most.  Measured, cluster / even pieces (fp32, head dim 64, us): one
// request of 325 keys 6.0 / 7.8, of 800 6.1 / 8.3, of 1600 8.0 / 8.3, of 3200 11.6 / 8.4; 8 requests of up to 1650
// 8.6 / 9.6, 32 of them 14.8 / 15.5, 32 of up to 6000 38 / 31.
constexpr int64_t CLUSTER_STEPS = 8, JOIN_STEPS = 2;

Plan plan_of(int64_t batch, int64_t heads, int64_t kv_heads, int64_t d, int64_t size, int64_t max_len) {
  Plan p = {};
  p.pairs = batch * kv_heads * ((heads / kv_heads + HT - 1) / HT);
  const int64_t wave = 2 * cv3::sm_count(), tk = tile_of(d, size);
  const int64_t tiles = max_len / tk + 2;  // (a window's first tile may begin before its first key)
  int64_t s = 1;
  while (s < 8 && s < tiles - 1 && p.pairs * s * 2 <= wave) s *= 2;
  const int64_t steps = (tiles + s - 1) / s * ((p.pairs * s + wave - 1) / wave), even = (p.pairs * tiles + wave - 1) / wave;
  if (steps <= CLUSTER_STEPS && steps <= even + JOIN_STEPS) {
    p.cluster = s;
    p.grid = p.pairs * s;
  } else {
    p.grid = std::min(wave, p.pairs * tiles);
    p.floats = 2 * p.pairs + p.grid * 2 * HT * (d + 2);
  }
  return p;
}

}  // namespace

extern "C" int64_t cv3_paged_attention_workspace(int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                                 int kv_type, int64_t max_len) {
  if (batch <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || max_len < 0) return 0;
  return plan_of(batch, heads, kv_heads, head_dim, cv3p::type_size(kv_type), max_len).floats;
}

extern "C" int cv3_paged_attention(const cv3_paged_attention_params* p, void* stream) {
  CV3_REQUIRE(p && p->size == (int64_t)sizeof(*p), CV3_ERR_VALUE, "paged_attention: bad parameter block");
  CV3_REQUIRE(p->batch >= 0 && p->heads > 0 && p->kv_heads > 0 && p->num_pages >= 0 && p->page_size > 0 &&
                  p->max_blocks >= 0 && p->table_ld >= p->max_blocks && p->window >= 0,
              CV3_ERR_VALUE, "paged_attention: bad shape");
  CV3_REQUIRE(p->heads % p->kv_heads == 0, CV3_ERR_VALUE, "%lld query heads is not a multiple of %lld kv heads",
              (long long)p->heads, (long long)p->kv_heads);
  const int64_t d = p->head_dim;
  CV3_REQUIRE(d == 32 || d == 64 || d == 96 || d == 128, CV3_ERR_UNSUPPORTED,
              "paged_attention: head_dim %lld (built for 32, 64, 96 and 128)", (long long)d);
  CV3_REQUIRE(cv3p::type_ok(p->q_type) && cv3p::type_ok(p->kv_type), CV3_ERR_VALUE,
              "paged_attention: unknown element type");
  const int es = cv3p::type_size(p->kv_type), ce = 32 / es;
  CV3_REQUIRE(((uintptr_t)p->k_pages & 31) == 0 && ((uintptr_t)p->v_pages & 31) == 0 &&
                  (p->ksp | p->ksh | p->kst | p->vsp | p->vsh | p->vst) % ce == 0,
              CV3_ERR_VALUE, "paged_attention: cache rows must start on 32-byte boundaries");
  // (a tile behind the last key must not pass 2^31 either)
  CV3_REQUIRE(p->page_size <= INT32_MAX && p->max_blocks <= INT32_MAX &&
                  p->max_blocks * p->page_size <= INT32_MAX - 4096 && p->num_pages <= INT32_MAX &&
                  p->batch <= 1 << 24 && p->heads <= 1 << 16,
              CV3_ERR_VALUE, "paged_attention: positions, pages and pairs are 32-bit numbers");
  if (p->batch == 0) return CV3_OK;
  const int64_t max_len = p->max_blocks * p->page_size;
  const Plan plan = plan_of(p->batch, p->heads, p->kv_heads, d, es, max_len);
  CV3_REQUIRE(plan.grid <= INT32_MAX && plan.pairs <= INT32_MAX, CV3_ERR_VALUE, "paged_attention: too many requests and heads");
  CV3_REQUIRE(plan.floats == 0 || (p->workspace && p->workspace_floats >= plan.floats && ((uintptr_t)p->workspace & 7) == 0),
              CV3_ERR_VALUE, "paged_attention: the workspace must hold cv3_paged_attention_workspace() floats");
  // n / page_size by a product: with 2^(sh-1) < page_size <= 2^sh and mul = ceil(2^(31+sh) / page_size), the excess
  // mul * page_size - 2^(31+sh) is below 2^sh, so n < 2^31 times it stays below 2^(31+sh): the quotient is exact
  int sh = 0;
  while ((int64_t)1 << sh < p->page_size) ++sh;
  const uint32_t mul = (uint32_t)((((uint64_t)1 << (31 + sh)) + p->page_size - 1) / p->page_size);
  float* stat = p->workspace + 2 * plan.pairs;
  const int group = (int)(p->heads / p->kv_heads);
  const AttnArgs a = {p->q, (int)p->q_type, p->qsb, p->qsh, p->k_pages, p->v_pages, p->ksp, p->ksh, p->kst, p->vsp,
                      p->vsh, p->vst, p->num_pages, (int)p->page_size, mul, (uint32_t)(31 + sh), p->block_tables,
                      p->table_ld, (int)max_len, p->lens, (int)p->batch, (int)p->heads, (int)p->kv_heads, group,
                      (group + HT - 1) / HT, (int)std::min<int64_t>(p->window, INT32_MAX), (float)p->scale, p->out,
                      p->osb, p->osh, p->lse, p->bad, stat + plan.grid * 2 * HT * 2, stat,
                      reinterpret_cast<int2*>(p->workspace)};
  const bool uni = p->page_size % 16 == 0, h16 = es == 2 && p->q_type == p->kv_type, cl = plan.cluster > 0;
  const Fn fn = p->kv_type == CV3_TYPE_F32   ? pick<float>(d, uni, h16, cl)
                : p->kv_type == CV3_TYPE_F16 ? pick<__half>(d, uni, h16, cl) : pick<__nv_bfloat16>(d, uni, h16, cl);
  cudaStream_t st = cv3::as_stream(stream);
  const dim3 grid((unsigned)plan.grid), block(NW * 32);
  if (cl)
    return cv3::check_launch("paged_attention", plan.cluster == 1
                                                    ? cv3::launch_dep(fn, grid, block, 0, st, a)
                                                    : cv3p::launch_cluster(fn, grid, block, 0, (unsigned)plan.cluster, st, a));
  int rc = cv3::check_launch("paged_attention", cv3::launch_dep(fn, grid, block, 0, st, a));
  if (rc) return rc;
  // (one request of 38399 keys, 2 pairs: 18 us wide, 39 us not; 64 of up to 4096, 512 pairs: 113 and 109.5 us)
  const bool wide = plan.pairs <= 64;
  return cv3::check_launch("paged_join", cv3::launch_dep(pick_join(d, wide), dim3((unsigned)plan.pairs, wide ? HT : 1),
                                                         block, 0, st, a));
}
