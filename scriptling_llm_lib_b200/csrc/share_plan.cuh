// The plan of an attention over shared pages (cache/share.py) as its kernels read it.
#pragma once
#include "common.cuh"

#define SHARE_LOG2E 1.4426950408889634f
#define SHARE_ERR_PAGE 5          // what *err says: a page id outside the storage, or a position outside the block table

// A plan on the device, as the host hands it over: one for every call that goes by it
struct SharePlanDev {
  const int *first, *thin_first, *items, *toks, *list_first, *list;
  long long part_rows;
  int T, H, G, workers, thin_warps;
};

struct ShareArgs {
  const void* q;             // [T, q_ld] queries that have their positions; head h at columns h * hd
  int q_ld;
  const int* tok_pos;        // [T]
  const int* block_table;    // [n_seqs, max_pages]
  int max_pages;
  const void *kpages, *vpages;   // [n_pages][G][PAGE][hd], [n_pages][G][PAGE][vd]
  int n_pages;
  // of the plan: where a block's items begin and where each of its warps' thin items do, items of eight words, rows of the step in the
  // tree's order
  const int *first, *thin_first, *items, *toks;
  float* part;               // the rows' sums over the values (share_at), then [part_rows][2]: m and l
  long long part_rows;       // a multiple of 32
  int H, G, hd, vd;
  float scale, softcap;
  int* err;
};

// Where dims d .. d + 3 (d a multiple of 4) of a row of the scratch stand: 32 rows together, four dims of a row side by side. Threads that
// have a row each then write 512 bytes in a row to memory with 16 bytes a thread (in rows of vd floats the same stores took 5 us of a block's
// 256 x 128 sums, one line a thread).
__device__ __forceinline__ size_t share_at(size_t row, int d, int vd) { return (row >> 5) * 32 * (size_t)vd + (size_t)d * 32 + (row & 31) * 4; }

// An item as a block works on it: pages [p0, p1) of row `seq` of the table; keys up to `last`, the position of its last token. A leaf's
// tokens are of one sequence and follow one another; a node's see all of its keys, whatever their positions (last: SHARE_NODE).
#define SHARE_NODE 0x3fffffff
struct ShareItem {
  int tok0, n_tok, g, p0, p1, last, part0, seq;
};
__device__ __forceinline__ ShareItem share_item(const ShareArgs& p, int i) {
  const int4 a = *(const int4*)(p.items + 8 * (size_t)i), b = *(const int4*)(p.items + 8 * (size_t)i + 4);
  ShareItem it;
  it.tok0 = a.x;
  it.n_tok = a.y;
  it.last = a.z < 0 ? SHARE_NODE : max(-1, min(p.tok_pos[a.z], SHARE_NODE - 1));
  it.g = a.w;
  it.p0 = b.x;
  // (a plan may be older than the step, and its sequences longer now; of a position outside the table, the pages that are there)
  const int end = (it.last + SLLM_PAGE) / SLLM_PAGE, most = it.last == SHARE_NODE ? end : min(end, p.max_pages);
  it.p1 = b.y < 0 || b.y > most ? most : b.y;
  it.part0 = b.z;
  it.seq = b.w;
  return it;
}
// an item's last token may stand outside the table: one of those that read the item says so
__device__ __forceinline__ void share_check(const ShareArgs& p, const ShareItem& it) {
  if (it.last < 0 || (it.last != SHARE_NODE && it.last / SLLM_PAGE >= p.max_pages)) atomicExch(p.err, SHARE_ERR_PAGE);
}
// the position up to which row `rho` of an item's tile sees keys; -1 for a row past the tile's end
__device__ __forceinline__ int share_sees(const ShareItem& it, int rho, int rep) {
  const int i = rho / rep;
  return i >= it.n_tok ? -1 : it.last == SHARE_NODE ? SHARE_NODE : it.last - (it.n_tok - 1 - i);
}
// the page at place `i` of a row of the table; -1 (and *err) where there is none
__device__ __forceinline__ int share_page(const ShareArgs& p, const int* row, int i) {
  const int page = i < p.max_pages ? row[i] : -1;
  if (page >= 0 && page < p.n_pages) return page;
  atomicExch(p.err, SHARE_ERR_PAGE);
  return -1;
}

// Four elements of a row's weighted sum of values, key by key and over those alone that it sees: for a row whose sum came out not
// finite. In a tile's product a page's values all enter it, with weights of zero, and 0 times what is not finite is NaN. Pages t0,
// t0 + step, ... of the item's.
template <typename A>
__device__ __noinline__ float4 share_sum_by_key(const ShareArgs& p, const ShareItem it, const A* q, int qpos, float m, int d0, int t0, int step) {
  const int* row = p.block_table + (size_t)it.seq * p.max_pages;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int key = t0 * SLLM_PAGE; key <= qpos && key < it.p1 * SLLM_PAGE; key++) {
    if (key % SLLM_PAGE == 0 && (key / SLLM_PAGE - t0) % step) {        // a page of the other half's
      key += SLLM_PAGE - 1;
      continue;
    }
    const int page = share_page(p, row, key / SLLM_PAGE);
    if (page < 0) continue;
    const size_t at = ((size_t)page * p.G + it.g) * SLLM_PAGE + key % SLLM_PAGE;
    const A *k = (const A*)p.kpages + at * p.hd, *v = (const A*)p.vpages + at * p.vd + d0;
    float s = 0.f;
    for (int d = 0; d < p.hd; d += 4) {
      const float4 a = ld4(q + d), b = ld4(k + d);
      s = fmaf(a.x, b.x, s);
      s = fmaf(a.y, b.y, s);
      s = fmaf(a.z, b.z, s);
      s = fmaf(a.w, b.w, s);
    }
    s *= p.scale;
    if (p.softcap > 0.f) s = p.softcap * tanhf(s / p.softcap);
    const float w = exp2f(fmaf(s, SHARE_LOG2E, m == -INFINITY ? 0.f : -m));
    const float4 x = ld4(v);
    acc.x = fmaf(w, x.x, acc.x);
    acc.y = fmaf(w, x.y, acc.y);
    acc.z = fmaf(w, x.z, acc.z);
    acc.w = fmaf(w, x.w, acc.w);
  }
  return acc;
}

// ------------------------------------------------------------------ host side
static inline bool share_aligned(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }
static inline bool share_call_ok(const SharePlanDev& plan, int rows, int q_ld, int hd, long long n_pages, int max_pages, const float* part) {
  return plan.T >= 0 && plan.G >= 1 && plan.H >= 1 && plan.H % plan.G == 0 && plan.H / plan.G <= rows && plan.workers >= 1 && plan.part_rows >= 1 &&
         plan.part_rows % 32 == 0 && (long long)plan.T * plan.H <= 0x7fffffffLL && q_ld >= plan.H * hd && n_pages >= 1 && n_pages <= 0x7fffffffLL &&
         (long long)plan.G * SLLM_PAGE <= 0x7fffffffLL && max_pages >= 1 && share_aligned(part, 16) && share_aligned(plan.items, 16);
}
static inline ShareArgs share_args(const SharePlanDev& plan, const void* q, int q_ld, const int* tok_pos, const int* block_table, int max_pages,
                                   const void* kpages, const void* vpages, long long n_pages, float* part, int hd, int vd, float scale,
                                   float softcap, int* err) {
  return ShareArgs{q, q_ld, tok_pos, block_table, max_pages, kpages, vpages, (int)n_pages, plan.first, plan.thin_first, plan.items, plan.toks, part,
                   plan.part_rows, plan.H, plan.G, hd, vd, scale, softcap, err};
}
