// The paged key/value cache's bookkeeping and writes: block tables and slot maps from request
// lengths (paged_extend), RoPE + store by slot (paged_append), beams following their parents
// (paged_reorder).
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
  int* page_off;  // [batch + 1] scratch: pages taken before request b; [batch]: pages on the stack before the first was taken
};

constexpr int ET = 1024;

__device__ __forceinline__ int64_t blocks_of(int64_t n, int64_t ps) { return (n + ps - 1) / ps; }

// inclusive sum over the block's threads; `total` the whole sum
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* red, int64_t& total) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  __syncthreads();
  if (lane == 31) red[wid] = v;
  __syncthreads();
  if (wid == 0) {
    int64_t w = red[lane];
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t u = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += u;
    }
    red[lane] = w;
  }
  __syncthreads();
  total = red[31];
  return v + (wid ? red[wid - 1] : 0);
}

// Row i of the token outputs.  The page of a token: an old page stands in the table; a page taken
// by this call comes from the stack, and the token that begins it writes it into the table.
__device__ void extend_row(const ExtendArgs& a, int64_t i) {
  const int64_t total = a.offsets[a.batch];
  if (i >= total) {  // rows behind the last token: no slot
    a.slots[i] = -1;
    a.seq[i] = -1;
    a.pos[i] = 0;
    return;
  }
  int64_t lo = 0, hi = a.batch - 1;  // the last request whose first row is <= i and which has rows
  while (lo < hi) {
    const int64_t mid = (lo + hi + 1) >> 1;
    if (a.offsets[mid] <= i) lo = mid;
    else hi = mid - 1;
  }
  const int64_t n = a.offsets[lo + 1] - a.offsets[lo];
  const int64_t base = a.lens_out[lo] - n;
  const int64_t p = base + (i - a.offsets[lo]);
  const int64_t j = p / a.ps, first = blocks_of(base, a.ps);
  int page;
  if (j < first) {
    page = a.tables[lo * a.ld + j];
  } else {
    page = a.stack[a.page_off[a.batch] - 1 - (a.page_off[lo] + (j - first))];
    if (p == j * a.ps) a.tables[lo * a.ld + j] = page;
  }
  a.slots[i] = (int64_t)page * a.ps + (p - j * a.ps);
  a.seq[i] = (int)lo;
  a.pos[i] = (int)p;
}

// One CTA: pages given back, sums over the requests, lengths and counts (and, fused, the rows).
__global__ void __launch_bounds__(ET) extend_scan_kernel(const ExtendArgs a, int fused) {
  __shared__ int64_t red[32];
  __shared__ long long first_out;
  dep_wait();
  dep_release();
  const int tid = threadIdx.x;
  if (tid == 0) first_out = a.batch;
  int64_t have = min((int64_t)max(*a.count, 0), a.cap);
  __syncthreads();
  if (a.release) {
    int64_t carry = 0;
    for (int64_t b0 = 0; b0 < a.batch; b0 += ET) {
      const int64_t b = b0 + tid;
      const bool gives = b < a.batch && a.release[b] != 0;
      const int64_t n = gives ? min(blocks_of(max(a.lens[b], 0), a.ps), a.max_blocks) : 0;
      int64_t total;
      const int64_t at = have + carry + block_scan(n, red, total) - n;
      for (int64_t j = 0; j < n && at + j < a.cap; ++j) a.stack[at + j] = a.tables[b * a.ld + j];
      carry += total;
    }
    have = min(have + carry, a.cap);
    __syncthreads();
  }
  int64_t pages = 0, rows = 0;  // asked for by the requests before this tile
  int64_t taken = 0;            // pages of the requests that are served
  for (int64_t b0 = 0; b0 < a.batch; b0 += ET) {
    const int64_t b = b0 + tid;
    int64_t base = 0, n = 0, need = 0;
    if (b < a.batch) {
      base = a.release && a.release[b] ? 0 : max(a.lens[b], 0);
      n = max(a.fresh[b], 0);
      need = blocks_of(base + n, a.ps) - blocks_of(base, a.ps);
    }
    int64_t tp, tr;
    const int64_t ep = pages + block_scan(need, red, tp), er = rows + block_scan(n, red, tr);
    if (b < a.batch && (ep > have || er > a.rows || base + n > a.max_blocks * a.ps))
      atomicMin(&first_out, (long long)b);
    __syncthreads();
    const int64_t stop = first_out;
    if (b < a.batch) {
      const bool served = b < stop;
      a.lens_out[b] = (int)(served ? base + n : base);
      a.page_off[b] = (int)(ep - need);
      if (served) a.offsets[b + 1] = (int)er;
    }
    // the sums of what is served: all of the tile, or the requests before the first that is not
    if (stop >= b0 + ET || stop >= a.batch) {
      taken = pages + tp;
      pages += tp;
      rows += tr;
      continue;
    }
    __shared__ int64_t cut[2];
    if (b == stop) {
      cut[0] = ep - need;
      cut[1] = er - n;
    }
    __syncthreads();
    taken = cut[0];
    rows = cut[1];
    for (int64_t c = b; c < a.batch; c += ET) {
      if (c >= stop) {
        a.offsets[c + 1] = (int)rows;
        if (c >= b0 + ET) a.lens_out[c] = a.release && a.release[c] ? 0 : max(a.lens[c], 0);
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
  __syncthreads();
  for (int64_t i = tid; i < a.rows; i += ET) extend_row(a, i);
}

__global__ void __launch_bounds__(256) extend_rows_kernel(const ExtendArgs a) {
  dep_wait();
  dep_release();
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < a.rows; i += (int64_t)gridDim.x * blockDim.x)
    extend_row(a, i);
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
};

// One row per CTA step.  A work item is VEC elements of a head's first half and the VEC that face
// them in the second (the half-split rotation mixes the two).
template <typename AT, typename CT, int VEC>
__global__ void __launch_bounds__(256) append_kernel(const AppendArgs a) {
  dep_wait();
  dep_release();
  const int half = a.d / 2, per = half / VEC, all = a.heads + 2 * a.kv_heads;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const int64_t slot = a.slots[r];
    int64_t p = a.pos ? a.pos[r] : 0;
    const bool in_table = !a.cosT || (p >= 0 && p < a.positions);
    const bool stored = slot >= 0 && slot < a.pages * a.ps && in_table;
    if (!stored && slot != -1 && a.bad && threadIdx.x == 0) atomicAdd(a.bad, 1);
    if (!in_table) p = 0;
    const int64_t page = stored ? slot / a.ps : 0, row = stored ? slot - page * a.ps : 0;
    const AT* x = static_cast<const AT*>(a.qkv) + r * a.ld;
    for (int i = threadIdx.x; i < all * per; i += blockDim.x) {
      const int h = i / per, e = (i - h * per) * VEC;
      const bool is_q = h < a.heads;
      if (!is_q && !stored) continue;
      float lo[VEC], hi[VEC];
      load_vec<AT, VEC>(x + (int64_t)h * a.d + e, lo);
      load_vec<AT, VEC>(x + (int64_t)h * a.d + half + e, hi);
      if (h < a.heads + a.kv_heads && a.cosT) {
        const float* c = a.cosT + p * a.d + e;
        const float* s = a.sinT + p * a.d + e;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {  // x * cos + rotate_half(x) * sin, each product rounded
          const float u = lo[j], w = hi[j];
          lo[j] = __fadd_rn(__fmul_rn(u, c[j]), __fmul_rn(-w, s[j]));
          hi[j] = __fadd_rn(__fmul_rn(w, c[half + j]), __fmul_rn(u, s[half + j]));
        }
      }
      if (is_q) {
        AT* y = static_cast<AT*>(a.q) + (r * a.heads + h) * a.d + e;
        store_vec<AT, VEC>(y, lo);
        store_vec<AT, VEC>(y + half, hi);
      } else {
        const bool is_k = h < a.heads + a.kv_heads;
        const int g = h - a.heads - (is_k ? 0 : a.kv_heads);
        CT* y = static_cast<CT*>(is_k ? a.k : a.v) +
                (is_k ? page * a.ksp + g * a.ksh + row * a.kst : page * a.vsp + g * a.vsh + row * a.vst) + e;
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

// blockIdx.y: group.  Each thread owns a place (layer, k or v, head, row, 16-byte piece) of the
// group's last, partly filled pages, or a column of its table rows, across all beams: it reads what
// every beam will need there before it writes any of it, so beams may trade places without a copy.
template <int KMAX>
__global__ void __launch_bounds__(256) reorder_kernel(const ReorderArgs a) {
  dep_wait();
  dep_release();
  __shared__ int parent[KMAX];
  __shared__ int64_t page[KMAX];
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
  const int64_t step = (int64_t)gridDim.x * blockDim.x, i0 = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
  for (int64_t j = i0; j < full; j += step) {
    int t[KMAX];
#pragma unroll
    for (int k = 0; k < KMAX; ++k)
      if (k < a.beams) t[k] = rows[parent[k] * a.ld + j];
#pragma unroll
    for (int k = 0; k < KMAX; ++k)
      if (k < a.beams && parent[k] != k) rows[k * a.ld + j] = t[k];
  }
  const int64_t places = a.layers * 2 * a.kv_heads * rest * a.row16;
  for (int64_t i = i0; i < places; i += step) {
    int64_t u = i;
    const int64_t c = u % a.row16;
    u /= a.row16;
    const int64_t r = u % rest;
    u /= rest;
    const int64_t h = u % a.kv_heads;
    u /= a.kv_heads;
    const bool is_k = (u & 1) == 0;
    const int64_t l = u >> 1;
    char* at = is_k ? a.k + l * a.ksl + h * a.ksh + r * a.kst : a.v + l * a.vsl + h * a.vsh + r * a.vst;
    at += c * 16;
    const int64_t sp = is_k ? a.ksp : a.vsp;
    int4 x[KMAX];
#pragma unroll
    for (int k = 0; k < KMAX; ++k)
      if (k < a.beams && parent[k] != k && page[k] >= 0 && page[parent[k]] >= 0)
        x[k] = *reinterpret_cast<const int4*>(at + page[parent[k]] * sp);
#pragma unroll
    for (int k = 0; k < KMAX; ++k)
      if (k < a.beams && parent[k] != k && page[k] >= 0 && page[parent[k]] >= 0)
        *reinterpret_cast<int4*>(at + page[k] * sp) = x[k];
  }
}

}  // namespace

extern "C" int cv3_paged_extend(const cv3_paged_extend_params* p, void* stream) {
  CV3_REQUIRE(p && p->size == (int64_t)sizeof(*p), CV3_ERR_VALUE, "paged_extend: bad parameter block");
  CV3_REQUIRE(p->batch >= 0 && p->max_blocks >= 0 && p->table_ld >= p->max_blocks && p->page_size > 0 &&
                  p->free_cap >= 0 && p->max_tokens >= 0,
              CV3_ERR_VALUE, "paged_extend: bad shape");
  CV3_REQUIRE(p->max_tokens <= INT32_MAX && p->free_cap <= INT32_MAX && p->page_size <= INT32_MAX &&
                  p->max_blocks <= INT32_MAX && p->max_blocks * p->page_size <= INT32_MAX,
              CV3_ERR_VALUE, "paged_extend: rows, pages and a request's positions are 32-bit numbers");
  const ExtendArgs a = {p->lens, p->new_lens, p->release, p->batch, p->block_tables, p->table_ld, p->max_blocks,
                        p->page_size, p->free_pages, p->free_cap, p->free_count, p->max_tokens, p->slots, p->seq, p->pos,
                        p->offsets, p->lens_out, p->free_count_out, p->scratch};
  cudaStream_t st = cv3::as_stream(stream);
  const int fused = p->max_tokens <= 4 * ET;
  int rc = cv3::check_launch("paged_extend", cv3::launch_dep(extend_scan_kernel, dim3(1), dim3(ET), 0, st, a, fused));
  if (rc || fused) return rc;
  const int64_t grid = std::min<int64_t>((p->max_tokens + 255) / 256, cv3::sm_count() * 8);
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
                  cv3p::aligned16(p->v_pages) && p->ldq % ae == 0 &&
                  (p->ksp | p->ksh | p->kst | p->vsp | p->vsh | p->vst) % ce == 0,
              CV3_ERR_VALUE, "paged_append: rows must start on 16-byte boundaries");
  if (p->rows == 0) return CV3_OK;
  const AppendArgs a = {p->qkv, p->rows, p->ldq, p->cos_table, p->sin_table, p->positions, p->slots, p->pos, (int)p->heads,
                        (int)p->kv_heads, (int)p->head_dim, p->q_out, p->k_pages, p->v_pages, p->ksp, p->ksh, p->kst,
                        p->vsp, p->vsh, p->vst, p->num_pages, p->page_size, p->bad};
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
  const int64_t grid = std::min<int64_t>(p->rows, cv3::sm_count() * 8);
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
  if (p->groups == 0 || p->beams == 1) return CV3_OK;
  const ReorderArgs a = {static_cast<char*>(p->k_pages), static_cast<char*>(p->v_pages), p->ksl * es, p->ksp * es,
                         p->ksh * es, p->kst * es, p->vsl * es, p->vsp * es, p->vsh * es, p->vst * es, p->layers,
                         p->num_pages, p->kv_heads, p->page_size, p->head_dim * es / 16, p->block_tables, p->table_ld,
                         p->max_blocks, p->parents, p->lens, p->groups, (int)p->beams};
  const int64_t most = std::max<int64_t>(p->layers * 2 * p->kv_heads * (p->page_size - 1) * a.row16, p->max_blocks);
  const int64_t gx = std::max<int64_t>(1, std::min<int64_t>((most + 255) / 256, (cv3::sm_count() * 8 + p->groups - 1) / p->groups));
  using Fn = void (*)(const ReorderArgs);
  const Fn fn = p->beams <= 4 ? (Fn)reorder_kernel<4> : p->beams <= 8 ? (Fn)reorder_kernel<8>
                : p->beams <= 16 ? (Fn)reorder_kernel<16> : (Fn)reorder_kernel<32>;
  return cv3::check_launch("paged_reorder", cv3::launch_dep(fn, dim3((unsigned)gx, (unsigned)p->groups), dim3(256), 0,
                                                            cv3::as_stream(stream), a));
}
