// The paged key/value cache's bookkeeping and writes: block tables and slot maps from request
// lengths (paged_extend), RoPE + store by slot (paged_append), beams following their parents
// (paged_reorder), pages that several rows name (paged_give_back).
//
// A cache is a pool of pages [page][kv_head][page_size][head_dim] (any strides with contiguous
// rows); a request owns the pages its block-table row names, token t at row t % page_size of page
// table[t / page_size].  A slot is page * page_size + row: one number that says where a token lives.
#include <algorithm>

#include "paged.cuh"

namespace {

using cv3p::load_vec;
using cv3p::store_vec;

// ---------------------------------------------------------------------------
// block tables and slots
// ---------------------------------------------------------------------------

struct ExtendArgs {
  const int *lens, *fresh, *release;
  int64_t batch;
  int* tables;
  int64_t ld, max_blocks, ps;
  int* stack;  // free pages, popped from the end
  int64_t cap;
  const int* count;
  int64_t rows;
  int64_t* slots;
  int *seq, *pos, *offsets, *lens_out, *count_out;
  int wide;       // slots, seq and pos are 16-byte aligned
  int* page_off;  // [batch + 1] scratch: pages taken before request b; [batch]: pages on the stack before the first was taken
};

constexpr int ET = 1024;

__device__ __forceinline__ int64_t blocks_of(int64_t n, int64_t ps) { return (n + ps - 1) / ps; }

struct Sum2 {
  int64_t x, y;
};

// inclusive sums over the block's threads; `total` the whole sums
__device__ __forceinline__ Sum2 block_scan(Sum2 v, Sum2* red, Sum2& total) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, warps = blockDim.x >> 5;
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, v.x, o), y = __shfl_up_sync(0xffffffffu, v.y, o);
    if (lane >= o) { v.x += x; v.y += y; }
  }
  __syncthreads();
  if (lane == 31) red[wid] = v;
  __syncthreads();
  Sum2 w = lane < warps ? red[lane] : Sum2{0, 0};  // every warp sums the warps' totals by itself
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, w.x, o), y = __shfl_up_sync(0xffffffffu, w.y, o);
    if (lane >= o) { w.x += x; w.y += y; }
  }
  total = {__shfl_sync(0xffffffffu, w.x, 31), __shfl_sync(0xffffffffu, w.y, 31)};
  const int64_t bx = __shfl_sync(0xffffffffu, w.x, max(wid - 1, 0)), by = __shfl_sync(0xffffffffu, w.y, max(wid - 1, 0));
  v.x += wid ? bx : 0;
  v.y += wid ? by : 0;
  return v;
}

// Rows [i, i + n) of the token outputs, n <= RV, i a multiple of RV.  The page of a token: an old page
// stands in the table; a page taken by this call comes from the stack, and the token that begins it
// writes it into the table.
constexpr int RV = 4;

__device__ __forceinline__ void extend_rows(const ExtendArgs& a, int i, int n) {
  const int total = a.offsets[a.batch], ps = (int)a.ps;
  int64_t slot[RV];
  int seq[RV], pos[RV];
#pragma unroll
  for (int u = 0; u < RV; ++u) {  // rows behind the last token: no slot
    slot[u] = -1;
    seq[u] = -1;
    pos[u] = 0;
  }
  if (i < total) {
    int lo = 0, hi = (int)a.batch - 1;  // the last request whose first row is <= i; it has row i
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (a.offsets[mid] <= i) lo = mid;
      else hi = mid - 1;
    }
    int b = lo - 1, end = i, p = 0, j = -1, r = 0, first = 0, page = 0;
#pragma unroll
    for (int u = 0; u < RV; ++u) {
      if (u >= n || i + u >= total) break;
      if (i + u >= end) {  // the next request that has rows
        int begin;
        do {
          ++b;
          begin = a.offsets[b];
          end = a.offsets[b + 1];
        } while (end <= i + u);
        const int base = a.lens_out[b] - (end - begin);
        first = (int)(((unsigned)base + (unsigned)ps - 1u) / (unsigned)ps);
        p = base + (i + u - begin);
        j = p / ps;
        r = p - j * ps;
        page = -1;
      } else {
        ++p;
        if (++r == ps) {
          r = 0;
          ++j;
          page = -1;
        }
      }
      if (page < 0) {
        if (j < first) {
          page = a.tables[b * a.ld + j];
        } else {
          page = a.stack[a.page_off[a.batch] - 1 - (a.page_off[b] + (j - first))];
          if (r == 0) a.tables[b * a.ld + j] = page;
        }
      }
      slot[u] = (int64_t)page * ps + r;
      seq[u] = b;
      pos[u] = p;
    }
  }
  if (n == RV && a.wide) {
    reinterpret_cast<longlong2*>(a.slots + i)[0] = make_longlong2(slot[0], slot[1]);
    reinterpret_cast<longlong2*>(a.slots + i)[1] = make_longlong2(slot[2], slot[3]);
    *reinterpret_cast<int4*>(a.seq + i) = make_int4(seq[0], seq[1], seq[2], seq[3]);
    *reinterpret_cast<int4*>(a.pos + i) = make_int4(pos[0], pos[1], pos[2], pos[3]);
  } else {
#pragma unroll
    for (int u = 0; u < RV; ++u)
      if (u < n) {
        a.slots[i + u] = slot[u];
        a.seq[i + u] = seq[u];
        a.pos[i + u] = pos[u];
      }
  }
}

// Pages given back, sums over the requests, lengths and counts (and, fused, the rows) by one CTA.  Many
// requests' pages are given back by a cluster of them (a third of 32, 64 and 512 requests done: 5.5, 5.6
// and 6.9 us; by one CTA 6.8, 10.0 and 12.3 us).
constexpr int OWN = 4;  // new tokens up to which a request's thread writes its rows itself

__global__ void __launch_bounds__(ET) extend_scan_kernel(const ExtendArgs a, int fused) {
  __shared__ Sum2 red[ET / 32];
  __shared__ long long first_out;
  __shared__ Sum2 cut;
  dep_wait();
  dep_release();
  const int tid = threadIdx.x, T = blockDim.x;
  if (tid == 0) first_out = a.batch;
  int64_t have = min((int64_t)max(*a.count, 0), a.cap);
  if (a.release) {
    __shared__ int give[ET], place[ET];
    const int lane = tid & 31, ranks = gridDim.x, warps = ranks * (T >> 5), warp = blockIdx.x * (T >> 5) + (tid >> 5);
    int64_t carry = 0;
    for (int64_t b0 = 0; b0 < a.batch; b0 += T) {
      const int64_t b = b0 + tid;
      const bool gives = b < a.batch && a.release[b] != 0;
      const int64_t n = gives ? min(blocks_of(max(a.lens[b], 0), a.ps), a.max_blocks) : 0;
      Sum2 total;
      const int64_t at = min(have + carry + block_scan(Sum2{n, 0}, red, total).x - n, a.cap);
      give[tid] = (int)min(n, a.cap - at);
      place[tid] = (int)at;
      __syncthreads();
      // a warp per request, four requests' first 64 pages on the way at a time
      const int most = (int)min((int64_t)T, a.batch - b0);
      for (int q = warp; q < most; q += 4 * warps) {
        int x[4][2];
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            const int i = q + u * warps, j = v * 32 + lane;
            x[u][v] = i < most && j < give[i] ? a.tables[(b0 + i) * a.ld + j] : 0;
          }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int i = q + u * warps;
          if (i >= most) break;
#pragma unroll
          for (int v = 0; v < 2; ++v)
            if (v * 32 + lane < give[i]) a.stack[place[i] + v * 32 + lane] = x[u][v];
          for (int j = 64 + lane; j < give[i]; j += 32) a.stack[place[i] + j] = a.tables[(b0 + i) * a.ld + j];
        }
      }
      carry += total.x;
      __syncthreads();
    }
    have = min(have + carry, a.cap);
    if (ranks > 1) {
      cv3p::cluster_sync();
      if (blockIdx.x) return;
    }
  }
  Sum2 asked = {0, 0};  // pages and rows asked for by the requests before this tile
  int64_t taken = 0;    // pages of the requests that are served
  bool own = fused != 0;
  for (int64_t b0 = 0; b0 < a.batch; b0 += T) {
    const int64_t b = b0 + tid;
    int64_t base = 0, n = 0, need = 0;
    if (b < a.batch) {
      base = a.release && a.release[b] ? 0 : max(a.lens[b], 0);
      n = max(a.fresh[b], 0);
      need = blocks_of(base + n, a.ps) - blocks_of(base, a.ps);
    }
    Sum2 total;
    Sum2 upto = block_scan(Sum2{need, n}, red, total);
    upto.x += asked.x;
    upto.y += asked.y;
    if (b < a.batch && (upto.x > have || upto.y > a.rows || base + n > a.max_blocks * a.ps))
      atomicMin(&first_out, (long long)b);
    own = __syncthreads_and(own && n <= OWN);
    const int64_t stop = first_out;
    if (b < a.batch) {
      const bool served = b < stop;
      a.lens_out[b] = (int)(served ? base + n : base);
      a.page_off[b] = (int)(upto.x - need);
      if (served) {
        a.offsets[b + 1] = (int)upto.y;
        if (own && n) {  // few new tokens: their rows at once
          const int64_t first = blocks_of(base, a.ps);
          int64_t j = base / a.ps, r = base - j * a.ps;
          int page = -1;
          for (int64_t i = 0; i < n; ++i) {
            if (i == 0 || r == 0) {
              page = j < first ? a.tables[b * a.ld + j] : a.stack[have - 1 - (upto.x - need + (j - first))];
              if (j >= first) a.tables[b * a.ld + j] = page;
            }
            const int64_t row = upto.y - n + i;
            a.slots[row] = (int64_t)page * a.ps + r;
            a.seq[row] = (int)b;
            a.pos[row] = (int)(base + i);
            if (++r == a.ps) { r = 0; ++j; }
          }
        }
      }
    }
    // the sums of what is served: all of the tile, or the requests before the first that is not
    if (stop >= b0 + T || stop >= a.batch) {
      taken = asked.x + total.x;
      asked = {asked.x + total.x, asked.y + total.y};
      continue;
    }
    if (b == stop) cut = {upto.x - need, upto.y - n};
    __syncthreads();
    taken = cut.x;
    asked = cut;
    for (int64_t c = b; c < a.batch; c += T) {
      if (c >= stop) {
        a.offsets[c + 1] = (int)cut.y;
        if (c >= b0 + T) a.lens_out[c] = a.release && a.release[c] ? 0 : max(a.lens[c], 0);
      }
    }
    break;
  }
  if (tid == 0) {
    a.offsets[0] = 0;
    a.page_off[a.batch] = (int)have;
    *a.count_out = (int)(have - taken);
  }
  if (!fused) return;
  if (own) {  // what is left are the rows behind the last token
    for (int64_t i = asked.y + tid; i < a.rows; i += T) {
      a.slots[i] = -1;
      a.seq[i] = -1;
      a.pos[i] = 0;
    }
    return;
  }
  __syncthreads();
  for (int i = tid * RV; i < a.rows; i += T * RV) extend_rows(a, i, (int)min((int64_t)RV, a.rows - i));
}

__global__ void __launch_bounds__(256) extend_rows_kernel(const ExtendArgs a) {
  dep_wait();
  dep_release();
  const int64_t i = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) * RV;
  if (i < a.rows) extend_rows(a, (int)i, (int)min((int64_t)RV, a.rows - i));
}

// ---------------------------------------------------------------------------
// RoPE and store by slot
// ---------------------------------------------------------------------------

struct AppendArgs {
  const void* qkv;
  int64_t rows, ld;
  const float *cosT, *sinT;
  int64_t positions;
  const int64_t* slots;
  const int* pos;
  int heads, kv_heads, d;
  void* q;
  void *k, *v;
  int64_t ksp, ksh, kst, vsp, vsh, vst, pages, ps;
  int* bad;
  int lanes;  // threads that share a row's heads at one place
};

// A thread holds one row's place -- VEC elements of a head's first half and the VEC that face them in
// the second, which the half-split rotation mixes -- and walks every `lanes`-th head there: the two
// table pieces are loaded once for all of them, and HU heads are on the way at a time (16384 bf16 rows
// of 48 heads of 128, 407 MB: 68 us at 6 heads twice; 75 us at 4, 132 us at one head a thread).
constexpr int HU = 6;

template <typename AT, typename CT, int VEC>
__global__ void __launch_bounds__(256) append_kernel(const AppendArgs a) {
  dep_wait();
  dep_release();
  const int half = a.d / 2, per = half / VEC, all = a.heads + 2 * a.kv_heads, turned = a.heads + a.kv_heads;
  const int64_t id = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
  const int64_t r = id / (per * a.lanes);
  if (r >= a.rows) return;
  const int w = (int)(id - r * (per * a.lanes)), lane = w / per, e = (w - lane * per) * VEC;
  const int64_t slot = a.slots[r];
  int64_t p = a.pos ? a.pos[r] : 0;
  const AT* x = static_cast<const AT*>(a.qkv) + r * a.ld + e;
  const bool in_table = !a.cosT || (p >= 0 && p < a.positions);
  const bool stored = slot >= 0 && slot < a.pages * a.ps && in_table;
  if (!stored && slot != -1 && a.bad && w == 0) atomicAdd(a.bad, 1);
  if (!in_table) p = 0;
  int64_t page = 0, row = 0;
  if (stored) {
    page = (slot >> 31) == 0 ? (int64_t)((uint32_t)slot / (uint32_t)a.ps) : slot / a.ps;
    row = slot - page * a.ps;
  }
  float cl[VEC], ch[VEC], sl[VEC], sh[VEC];
  if (a.cosT) {
    const float* c = a.cosT + p * a.d + e;
    const float* s = a.sinT + p * a.d + e;
    load_vec<float, VEC>(c, cl);
    load_vec<float, VEC>(c + half, ch);
    load_vec<float, VEC>(s, sl);
    load_vec<float, VEC>(s + half, sh);
  }
  const int end = stored ? all : a.heads;  // what is not stored is not read
  for (int h0 = lane; h0 < end; h0 += HU * a.lanes) {
    cv3p::Vec<AT, VEC> first[HU], second[HU];
#pragma unroll
    for (int u = 0; u < HU; ++u) {
      const int h = min(h0 + u * a.lanes, end - 1);  // (a head past the last: the last again)
      first[u] = *reinterpret_cast<const cv3p::Vec<AT, VEC>*>(x + h * a.d);
      second[u] = *reinterpret_cast<const cv3p::Vec<AT, VEC>*>(x + h * a.d + half);
    }
#pragma unroll
    for (int u = 0; u < HU; ++u) {
      const int h = h0 + u * a.lanes;
      if (h >= end) break;
      float lo[VEC], hi[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        lo[j] = cv3p::to_f32<AT>(first[u].v[j]);
        hi[j] = cv3p::to_f32<AT>(second[u].v[j]);
      }
      if (h < turned && a.cosT) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {  // x * cos + rotate_half(x) * sin, each product rounded
          const float y = lo[j], z = hi[j];
          lo[j] = __fadd_rn(__fmul_rn(y, cl[j]), __fmul_rn(-z, sl[j]));
          hi[j] = __fadd_rn(__fmul_rn(z, ch[j]), __fmul_rn(y, sh[j]));
        }
      }
      if (h < a.heads) {
        AT* y = static_cast<AT*>(a.q) + (r * a.heads + h) * a.d + e;
        store_vec<AT, VEC>(y, lo);
        store_vec<AT, VEC>(y + half, hi);
      } else {
        const int g = h < turned ? h - a.heads : h - turned;
        CT* y = (h < turned ? static_cast<CT*>(a.k) + page * a.ksp + g * a.ksh + row * a.kst
                            : static_cast<CT*>(a.v) + page * a.vsp + g * a.vsh + row * a.vst) + e;
        store_vec<CT, VEC>(y, lo);
        store_vec<CT, VEC>(y + half, hi);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// beams follow their parents
// ---------------------------------------------------------------------------

struct ReorderArgs {
  char *k, *v;                  // bytes
  int64_t ksl, ksp, ksh, kst, vsl, vsp, vsh, vst;  // strides in bytes: layer, page, kv head, row
  int64_t layers, pages, kv_heads, ps, row16;      // row16: 16-byte pieces of a cache row
  int* tables;
  int64_t ld, max_blocks;
  const int *parents, *lens;
  int64_t groups;
  int beams;
};

// Bound by the bytes copied (32 groups of 8 beams, 24 layers, 83 MB: 16.4 us, 5.1 TB/s).
// blockIdx.y: group; blockIdx.z: layer, keys or values.  Each thread owns a place (head, row, 16-byte piece) of the
// group's last, partly filled pages, or a column of its table rows, across all beams: it reads what
// every beam will need there before it writes any of it, so beams may trade places without a copy.
template <int KMAX>
__global__ void __launch_bounds__(256) reorder_kernel(const ReorderArgs a) {
  dep_wait();
  dep_release();
  __shared__ int parent[KMAX];
  __shared__ int64_t page[KMAX], from[KMAX];  // own last page; the parent's, -1: nothing to copy
  const int64_t g = blockIdx.y;
  const int64_t len = max(a.lens[g * a.beams], 0);
  const int64_t full = min(len / a.ps, a.max_blocks);
  const int64_t rest = full < a.max_blocks ? len - full * a.ps : 0;
  int* rows = a.tables + g * a.beams * a.ld;
  bool moves = false;
  if (threadIdx.x < a.beams) {
    const int k = threadIdx.x;
    const int p = a.parents[g * a.beams + k];
    parent[k] = p >= 0 && p < a.beams ? p : k;
    moves = parent[k] != k;
    const int own = full < a.max_blocks ? rows[k * a.ld + full] : -1;
    page[k] = own >= 0 && own < a.pages ? own : -1;
  }
  if (!__syncthreads_or(moves)) return;
  if (threadIdx.x < a.beams) {
    const int k = threadIdx.x;
    from[k] = parent[k] != k && page[k] >= 0 ? page[parent[k]] : -1;
  }
  __syncthreads();
  const int z = blockIdx.z;  // layer and keys or values
  const int step = gridDim.x * blockDim.x, i0 = blockIdx.x * blockDim.x + threadIdx.x;
  if (z == 0)
    for (int j = i0; j < full; j += step) {
      int t[KMAX];
#pragma unroll
      for (int k = 0; k < KMAX; ++k)
        if (k < a.beams) t[k] = rows[parent[k] * a.ld + j];
#pragma unroll
      for (int k = 0; k < KMAX; ++k)
        if (k < a.beams && parent[k] != k) rows[k * a.ld + j] = t[k];
    }
  if (z >= 2 * a.layers) return;
  const int64_t l = z >> 1;
  char* base = z & 1 ? a.v + l * a.vsl : a.k + l * a.ksl;
  const int64_t sp = z & 1 ? a.vsp : a.ksp, sh = z & 1 ? a.vsh : a.ksh, st = z & 1 ? a.vst : a.kst;
  const unsigned row16 = (unsigned)a.row16, slab = (unsigned)rest * row16, places = (unsigned)a.kv_heads * slab;
  for (unsigned i = i0; i < places; i += step) {
    const unsigned h = i / slab, w = i - h * slab, r = w / row16, c = w - r * row16;
    char* at = base + h * sh + r * st + c * 16;
    int4 x[KMAX];
#pragma unroll
    for (int k = 0; k < KMAX; ++k)
      if (k < a.beams && from[k] >= 0) x[k] = *reinterpret_cast<const int4*>(at + from[k] * sp);
#pragma unroll
    for (int k = 0; k < KMAX; ++k)
      if (k < a.beams && from[k] >= 0) *reinterpret_cast<int4*>(at + page[k] * sp) = x[k];
  }
}

// ---------------------------------------------------------------------------
// pages that several table rows name
// ---------------------------------------------------------------------------

// shares[p]: how many table rows name page p beyond the first (0 for a free page too, so taking one from
// the stack changes nothing).  Rows leave their pages -- released requests all of them, beams the full pages
// that their parent does not have in the same column -- and a page whose number falls below 0 goes back.
struct GiveArgs {
  int* shares;
  int64_t pages;
  const int* tables;
  int64_t ld, max_blocks, ps;
  const int* lens;
  int64_t rows;
  const int* release;  // NULL: beams follow `parents`
  int* lens_out;
  const int* parents;
  int64_t beams;
  int* stack;
  int64_t cap;
  const int* count;
  int* count_out;
  int* given;  // [rows] scratch: pages that the row gives back
};

struct Leaving {
  const int *row, *next;  // entries that are left, and taken over instead (NULL: none)
  int n;
};

__device__ __forceinline__ Leaving leaving(const GiveArgs& a, int64_t b) {
  Leaving w = {a.tables + b * a.ld, nullptr, 0};
  if (a.release) {
    if (a.release[b]) w.n = (int)min(blocks_of(max(a.lens[b], 0), a.ps), a.max_blocks);
  } else {
    const int64_t first = b / a.beams * a.beams;
    const int p = a.parents[b];
    if (p >= 0 && p < a.beams && first + p != b) {
      w.next = a.tables + (first + p) * a.ld;
      w.n = (int)min(max(a.lens[first], 0) / a.ps, a.max_blocks);
    }
  }
  return w;
}

// the page that column j leaves, -1: none of the pool, or it stays
__device__ __forceinline__ int left_page(const GiveArgs& a, const Leaving& w, int j) {
  const int page = w.row[j];
  if (w.next && w.next[j] == page) return -1;
  return page >= 0 && page < a.pages ? page : -1;
}

// A warp per row, the rows dealt to a cluster of CTAs.  A page that several rows leave at once goes back one time, for
// the first of them (rows, then columns, in order), so the stack does not depend on timing: a page below 0
// takes the number of its first place -- far below what counting reaches -- until that place gives it back.
constexpr int MARK = INT32_MIN;

__global__ void __launch_bounds__(ET) give_back_kernel(const GiveArgs a) {
  __shared__ Sum2 red[ET / 32];
  __shared__ int64_t place[ET];
  dep_wait();
  dep_release();
  const int tid = threadIdx.x, T = blockDim.x, lane = tid & 31, warps = gridDim.x * (T >> 5);
  const int64_t warp = blockIdx.x * (T >> 5) + (tid >> 5);
  int64_t have = min((int64_t)max(*a.count, 0), a.cap);
  auto sync = [&]() {
    if (gridDim.x > 1) cv3p::cluster_sync();
    else __syncthreads();
  };
  for (int64_t b = warp; b < a.rows; b += warps) {
    const Leaving w = leaving(a, b);
    for (int j = lane; j < w.n; j += 32) {
      const int page = left_page(a, w, j);
      if (page >= 0) atomicSub(a.shares + page, 1);
      const int next = w.next ? w.next[j] : -1;
      if (next != w.row[j] && next >= 0 && next < a.pages) atomicAdd(a.shares + next, 1);
    }
  }
  sync();
  for (int64_t b = warp; b < a.rows; b += warps) {
    const Leaving w = leaving(a, b);
    for (int j = lane; j < w.n; j += 32) {
      const int page = left_page(a, w, j);
      if (page >= 0 && __ldcg(a.shares + page) < 0) atomicMin(a.shares + page, MARK + (int)(b * a.max_blocks + j));
    }
  }
  sync();
  for (int64_t b = warp; b < a.rows; b += warps) {
    const Leaving w = leaving(a, b);
    int n = 0;
    for (int j = lane; j < w.n; j += 32) {
      const int page = left_page(a, w, j);
      n += page >= 0 && __ldcg(a.shares + page) == MARK + (int)(b * a.max_blocks + j);
    }
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) a.given[b] = n;
  }
  sync();
  for (int64_t b0 = 0; b0 < a.rows; b0 += T) {
    const int64_t n = b0 + tid < a.rows ? __ldcg(a.given + b0 + tid) : 0;
    Sum2 total;
    place[tid] = have + block_scan(Sum2{n, 0}, red, total).x - n;
    __syncthreads();
    const int most = (int)min((int64_t)T, a.rows - b0);
    for (int i = (int)warp; i < most; i += warps) {
      const int64_t b = b0 + i;
      const Leaving w = leaving(a, b);
      int64_t at = place[i];
      for (int j0 = 0; j0 < w.n; j0 += 32) {
        const int j = j0 + lane, page = j < w.n ? left_page(a, w, j) : -1;
        const bool mine = page >= 0 && __ldcg(a.shares + page) == MARK + (int)(b * a.max_blocks + j);
        const unsigned who = __ballot_sync(0xffffffffu, mine);
        if (mine) {
          const int64_t to = at + __popc(who & ((1u << lane) - 1u));
          if (to < a.cap) a.stack[to] = page;
          a.shares[page] = 0;
        }
        at += __popc(who);
      }
      __syncwarp();  // (lens_out may be lens)
      if (a.lens_out && lane == 0) a.lens_out[b] = a.release[b] ? 0 : max(a.lens[b], 0);
    }
    have += total.x;
    __syncthreads();
  }
  if (blockIdx.x == 0 && tid == 0) *a.count_out = (int)min(have, a.cap);
}

}  // namespace

extern "C" int cv3_paged_give_back(const cv3_paged_give_back_params* p, void* stream) {
  CV3_REQUIRE(p && p->size == (int64_t)sizeof(*p), CV3_ERR_VALUE, "paged_give_back: bad parameter block");
  CV3_REQUIRE(p->num_pages >= 0 && p->rows >= 0 && p->max_blocks >= 0 && p->table_ld >= p->max_blocks &&
                  p->page_size > 0 && p->free_cap >= 0,
              CV3_ERR_VALUE, "paged_give_back: bad shape");
  CV3_REQUIRE((p->release == nullptr) != (p->parents == nullptr), CV3_ERR_VALUE,
              "paged_give_back: either release or parents is given");
  CV3_REQUIRE(p->release ? p->lens_out != nullptr : p->beams > 0 && p->rows % p->beams == 0, CV3_ERR_VALUE,
              "paged_give_back: release goes with lens_out, parents with groups of beams");
  CV3_REQUIRE(p->release || (p->beams <= CV3_MAX_BEAMS && p->rows / p->beams <= 65535), CV3_ERR_UNSUPPORTED,
              "paged_give_back: more than 65535 groups or %d beams", CV3_MAX_BEAMS);
  CV3_REQUIRE(p->num_pages <= INT32_MAX && p->free_cap <= INT32_MAX && p->page_size <= INT32_MAX && p->rows <= 1 << 30 &&
                  p->max_blocks <= 1 << 30 && p->rows * p->max_blocks <= 1 << 30 &&
                  p->max_blocks * p->page_size <= INT32_MAX,
              CV3_ERR_VALUE, "paged_give_back: pages and positions are 32-bit numbers, places of the tables 30-bit ones");
  const GiveArgs a = {p->shares, p->num_pages, p->block_tables, p->table_ld, p->max_blocks, p->page_size, p->lens, p->rows,
                      p->release, p->release ? p->lens_out : nullptr, p->parents, p->beams, p->free_pages, p->free_cap,
                      p->free_count, p->free_count_out, p->scratch};
  const int64_t ctas = p->rows >= 16 ? 8 : 1;
  const unsigned threads = (unsigned)std::min<int64_t>(ET, std::max<int64_t>(64, (p->rows + ctas - 1) / ctas * 32));
  cudaStream_t st = cv3::as_stream(stream);
  return cv3::check_launch("paged_give_back",
                           ctas > 1 ? cv3p::launch_cluster(give_back_kernel, dim3(8), dim3(threads), 0, 8u, st, a)
                                    : cv3::launch_dep(give_back_kernel, dim3(1), dim3(threads), 0, st, a));
}

extern "C" int cv3_paged_extend(const cv3_paged_extend_params* p, void* stream) {
  CV3_REQUIRE(p && p->size == (int64_t)sizeof(*p), CV3_ERR_VALUE, "paged_extend: bad parameter block");
  CV3_REQUIRE(p->batch >= 0 && p->max_blocks >= 0 && p->table_ld >= p->max_blocks && p->page_size > 0 &&
                  p->free_cap >= 0 && p->max_tokens >= 0,
              CV3_ERR_VALUE, "paged_extend: bad shape");
  CV3_REQUIRE(p->batch <= INT32_MAX - 1024 && p->max_tokens <= INT32_MAX - 1024 && p->free_cap <= INT32_MAX && p->page_size <= INT32_MAX &&
                  p->max_blocks <= INT32_MAX && p->max_blocks * p->page_size <= INT32_MAX,
              CV3_ERR_VALUE, "paged_extend: rows, pages and a request's positions are 32-bit numbers");
  const ExtendArgs a = {p->lens, p->new_lens, p->release, p->batch, p->block_tables, p->table_ld, p->max_blocks,
                        p->page_size, p->free_pages, p->free_cap, p->free_count, p->max_tokens, p->slots, p->seq, p->pos,
                        p->offsets, p->lens_out, p->free_count_out,
                        cv3p::aligned16(p->slots) && cv3p::aligned16(p->seq) && cv3p::aligned16(p->pos), p->scratch};
  cudaStream_t st = cv3::as_stream(stream);
  // few rows, or a few for every request (decoding), in the same launch: 64 requests, a row each, 5.5 us against
  // 9.4 us in two; 8 requests of 500 rows 6.2 against 5.0 us
  const int fused = p->max_tokens <= 1024 || (p->max_tokens <= OWN * p->batch && p->max_tokens <= 4 * ET);
  const int64_t work = std::max(p->batch, fused ? (p->max_tokens + RV - 1) / RV : 0);
  const unsigned threads = (unsigned)std::min<int64_t>(ET, std::max<int64_t>(64, (work + 31) / 32 * 32));
  const bool cluster = p->release && p->batch >= 16;
  int rc = cv3::check_launch("paged_extend",
                             cluster ? cv3p::launch_cluster(extend_scan_kernel, dim3(8), dim3(threads), 0, 8u, st, a, fused)
                                     : cv3::launch_dep(extend_scan_kernel, dim3(1), dim3(threads), 0, st, a, fused));
  if (rc || fused) return rc;
  const int64_t grid = (p->max_tokens + 256 * RV - 1) / (256 * RV);
  return cv3::check_launch("paged_extend_rows",
                           cv3::launch_dep(extend_rows_kernel, dim3((unsigned)grid), dim3(256), 0, st, a));
}

extern "C" int cv3_paged_append(const cv3_paged_append_params* p, void* stream) {
  CV3_REQUIRE(p && p->size == (int64_t)sizeof(*p), CV3_ERR_VALUE, "paged_append: bad parameter block");
  CV3_REQUIRE(p->rows >= 0 && p->heads > 0 && p->kv_heads > 0 && p->num_pages >= 0 && p->page_size > 0 &&
                  p->heads + 2 * p->kv_heads <= INT32_MAX / 512,
              CV3_ERR_VALUE, "paged_append: bad shape");
  CV3_REQUIRE(p->head_dim > 0 && p->head_dim % 16 == 0 && p->head_dim <= 256, CV3_ERR_UNSUPPORTED,
              "paged_append: head_dim %lld (a multiple of 16 up to 256)", (long long)p->head_dim);
  CV3_REQUIRE(cv3p::type_ok(p->type) && cv3p::type_ok(p->kv_type), CV3_ERR_VALUE, "paged_append: unknown element type");
  CV3_REQUIRE((p->cos_table == nullptr) == (p->sin_table == nullptr) && (!p->cos_table || (p->pos && p->positions > 0)),
              CV3_ERR_VALUE, "paged_append: cos and sin tables and positions go together");
  CV3_REQUIRE(p->ldq >= (p->heads + 2 * p->kv_heads) * p->head_dim, CV3_ERR_VALUE, "paged_append: ldq too small");
  const int ae = 16 / cv3p::type_size((int)p->type), ce = 16 / cv3p::type_size((int)p->kv_type);
  CV3_REQUIRE(cv3p::aligned16(p->qkv) && cv3p::aligned16(p->q_out) && cv3p::aligned16(p->k_pages) &&
                  cv3p::aligned16(p->v_pages) && cv3p::aligned16(p->cos_table) && cv3p::aligned16(p->sin_table) &&
                  p->ldq % ae == 0 && (p->ksp | p->ksh | p->kst | p->vsp | p->vsh | p->vst) % ce == 0,
              CV3_ERR_VALUE, "paged_append: rows and tables must start on 16-byte boundaries");
  CV3_REQUIRE(p->num_pages <= INT32_MAX && p->page_size <= INT32_MAX, CV3_ERR_VALUE,
              "paged_append: pages and their rows are 32-bit numbers");
  if (p->rows == 0) return CV3_OK;
  // one head a thread until the GPU is full, then two rounds of HU
  const int64_t all = p->heads + 2 * p->kv_heads, per = p->head_dim / 2 / ae, full = (int64_t)cv3::sm_count() * 2048;
  int64_t lanes = all;
  if (p->rows * per * all > full) lanes = std::max((all + 2 * HU - 1) / (2 * HU), std::min(all, full / (p->rows * per)));
  CV3_REQUIRE(p->rows <= (int64_t)INT32_MAX * 256 / (per * lanes), CV3_ERR_VALUE, "paged_append: too many rows");
  const AppendArgs a = {p->qkv, p->rows, p->ldq, p->cos_table, p->sin_table, p->positions, p->slots, p->pos, (int)p->heads,
                        (int)p->kv_heads, (int)p->head_dim, p->q_out, p->k_pages, p->v_pages, p->ksp, p->ksh, p->kst,
                        p->vsp, p->vsh, p->vst, p->num_pages, p->page_size, p->bad, (int)lanes};
  using Fn = void (*)(const AppendArgs);
  Fn fn = nullptr;
  switch ((int)p->type * 3 + (int)p->kv_type) {
    case 0: fn = append_kernel<float, float, 4>; break;
    case 1: fn = append_kernel<float, __half, 4>; break;
    case 2: fn = append_kernel<float, __nv_bfloat16, 4>; break;
    case 3: fn = append_kernel<__half, float, 8>; break;
    case 4: fn = append_kernel<__half, __half, 8>; break;
    case 5: fn = append_kernel<__half, __nv_bfloat16, 8>; break;
    case 6: fn = append_kernel<__nv_bfloat16, float, 8>; break;
    case 7: fn = append_kernel<__nv_bfloat16, __half, 8>; break;
    default: fn = append_kernel<__nv_bfloat16, __nv_bfloat16, 8>; break;
  }
  const int64_t grid = (p->rows * per * lanes + 255) / 256;
  return cv3::check_launch("paged_append", cv3::launch_dep(fn, dim3((unsigned)grid), dim3(256), 0, cv3::as_stream(stream), a));
}

extern "C" int cv3_paged_reorder(const cv3_paged_reorder_params* p, void* stream) {
  CV3_REQUIRE(p && p->size == (int64_t)sizeof(*p), CV3_ERR_VALUE, "paged_reorder: bad parameter block");
  CV3_REQUIRE(p->layers >= 0 && p->num_pages >= 0 && p->kv_heads > 0 && p->page_size > 0 && p->head_dim > 0 &&
                  p->groups >= 0 && p->max_blocks >= 0 && p->table_ld >= p->max_blocks,
              CV3_ERR_VALUE, "paged_reorder: bad shape");
  CV3_REQUIRE(p->beams > 0 && p->beams <= CV3_MAX_BEAMS, CV3_ERR_UNSUPPORTED, "paged_reorder: %lld beams (1 to %d)",
              (long long)p->beams, CV3_MAX_BEAMS);
  CV3_REQUIRE(cv3p::type_ok(p->kv_type), CV3_ERR_VALUE, "paged_reorder: unknown element type");
  CV3_REQUIRE(p->groups <= 65535, CV3_ERR_UNSUPPORTED, "paged_reorder: more than 65535 groups");
  const int64_t es = cv3p::type_size((int)p->kv_type);
  CV3_REQUIRE(cv3p::aligned16(p->k_pages) && cv3p::aligned16(p->v_pages) && p->head_dim * es % 16 == 0 &&
                  (p->ksl | p->ksp | p->ksh | p->kst | p->vsl | p->vsp | p->vsh | p->vst) * es % 16 == 0,
              CV3_ERR_VALUE, "paged_reorder: cache rows must be 16-byte pieces on 16-byte boundaries");
  const ReorderArgs a = {static_cast<char*>(p->k_pages), static_cast<char*>(p->v_pages), p->ksl * es, p->ksp * es,
                         p->ksh * es, p->kst * es, p->vsl * es, p->vsp * es, p->vsh * es, p->vst * es, p->layers,
                         p->num_pages, p->kv_heads, p->page_size, p->head_dim * es / 16, p->block_tables, p->table_ld,
                         p->max_blocks, p->parents, p->lens, p->groups, (int)p->beams};
  // places of a layer's keys or values, and columns, must be 32-bit numbers; z is limited to 65535
  const int64_t most = std::max<int64_t>(p->kv_heads * (p->page_size - 1) * a.row16, 1);
  CV3_REQUIRE(p->kv_heads <= 1 << 16 && p->page_size <= 1 << 20 && a.row16 <= 1 << 12 && most <= 1 << 30 &&
                  p->max_blocks <= 1 << 30 && p->layers <= 32767,
              CV3_ERR_UNSUPPORTED, "paged_reorder: pages too large or too many layers");
  if (p->groups == 0 || p->beams == 1) return CV3_OK;
  const int64_t gz = std::max<int64_t>(1, 2 * p->layers);
  const int64_t gx = std::max<int64_t>(1, std::min<int64_t>((most + 255) / 256, 16 * cv3::sm_count() / (p->groups * gz) + 1));
  using Fn = void (*)(const ReorderArgs);
  const Fn fn = p->beams <= 4 ? (Fn)reorder_kernel<4> : p->beams <= 8 ? (Fn)reorder_kernel<8>
                : p->beams <= 16 ? (Fn)reorder_kernel<16> : (Fn)reorder_kernel<32>;
  return cv3::check_launch("paged_reorder", cv3::launch_dep(fn, dim3((unsigned)gx, (unsigned)p->groups, (unsigned)gz), dim3(256), 0,
                                                            cv3::as_stream(stream), a));
}
