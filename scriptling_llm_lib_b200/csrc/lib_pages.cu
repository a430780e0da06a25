// Copies of cache pages and of sequences' fixed-size states: what forking a sequence and compacting a cache move. The reference holds
// one sequence and copies nothing.
//
// An area is a tensor to copy from and one to copy to (the same one, or another of the same layout): units of items of `runs` runs each,
// a run `row_bytes` bytes for every row that is copied, runs `run_bytes` apart. For pages an item is a page, a run the positions of one
// key/value head and a row a position; for states an item is a slot, with one run of one row. Pair (src[i], dst[i]) copies rows[i] rows
// (null: `max_rows`) of every run of item src[i] to item dst[i], in every unit of every area, with one launch for up to
// PG_AREAS areas. Only bytes move: the element type does not matter beyond the width of the accesses, and what a pair does not cover stays as it is.
// Bound by memory: every byte read once and written once (from one page to many: read from L2 after the first). 600 pages of 32 layers,
// 8 heads of 128 moved: 10.1 GB in 1,571 us (6.4 TB/s); 63 copies of 37 positions of 24 layers, 32 heads of 64: 89 us (5.2 TB/s written); 31
// copies of a slot of 8.4 MB: 46 us (6.0 TB/s).
#include "common.cuh"

#define PG_AREAS 16
#define PG_THREADS 256
#define PG_VECS 4             // accesses of a thread in flight (eight: fewer blocks on an SM, partly copied pages 2.7 times slower)
#define PG_ERR 5              // what *err says: an id or a number of rows out of range; that pair is not copied

struct PgArea {
  const char* from;
  char* to;
  long long from_unit, to_unit;      // bytes from one unit to the next
  long long item_bytes, run_bytes;   // of an item (the same in both tensors), of a run
  int row_bytes, units, runs, from_items, to_items, chunks;   // chunks: pieces that an item is copied in
};
struct PgArgs {
  PgArea area[PG_AREAS];
  long long first[PG_AREAS + 1];     // pieces of the areas before: pieces are dealt to the blocks in one line
  int n_areas, n_pairs, max_rows;
  int steps;                         // of a piece: PG_THREADS * PG_VECS accesses each
  const int *src, *dst, *rows;
  int* err;
};

// What is written is not read soon: streaming stores give way to what is (63 copies of a page, 458 MB written: 122 us without, 100 with four
// blocks for every one that is resident, 89 with both; torch.fill_ of as many bytes takes 119).
template <typename V>
__device__ __forceinline__ void pg_store(V* p, V v) { *p = v; }
template <>
__device__ __forceinline__ void pg_store<uint4>(uint4* p, uint4 v) { __stcs(p, v); }
template <typename V>
__device__ __forceinline__ V pg_load(const V* p) { return *p; }
template <>
__device__ __forceinline__ uint4 pg_load<uint4>(const uint4* p) { return ld_dep16_stream(p); }

// What a piece copies.
struct PgPiece {
  int area, piece, unit, from, to, rows;      // from < 0: no such item, nothing to copy
};
__device__ __forceinline__ PgPiece pg_piece(const PgArgs& p, long long c) {
  PgPiece w;
  w.area = 0;
  while (c >= p.first[w.area + 1]) w.area++;
  const PgArea& a = p.area[w.area];
  const unsigned long long local = (unsigned long long)(c - p.first[w.area]);
  const unsigned long long pair = local / (unsigned)a.chunks;
  w.piece = (int)(local - pair * (unsigned)a.chunks);
  w.unit = (int)(pair / (unsigned)p.n_pairs);
  const int i = (int)(pair - (unsigned long long)w.unit * (unsigned)p.n_pairs);
  w.from = p.src[i];
  w.to = p.dst[i];
  w.rows = p.rows ? p.rows[i] : p.max_rows;
  if (w.from < 0 || w.from >= a.from_items || w.to < 0 || w.to >= a.to_items || w.rows < 0 || w.rows > p.max_rows) w.from = -1;
  return w;
}

template <typename V>
__global__ void __launch_bounds__(PG_THREADS, 6) page_copy_kernel(const __grid_constant__ PgArgs p) {
  pdl_launch_dependents();
  pdl_wait();
  const long long end = p.first[p.n_areas];
  for (long long c = blockIdx.x; c < end; c += gridDim.x) {
    const PgPiece w = pg_piece(p, c);
    if (w.from < 0) {
      if (threadIdx.x == 0) atomicExch(p.err, PG_ERR);
      continue;
    }
    const PgArea& a = p.area[w.area];
    const V* from = (const V*)(a.from + w.unit * a.from_unit + w.from * a.item_bytes);
    V* to = (V*)(a.to + w.unit * a.to_unit + w.to * a.item_bytes);
    // a run's vectors; an item copied whole is one run
    const bool whole = w.rows == p.max_rows;
    const unsigned per = whole ? (unsigned)(a.item_bytes / (int)sizeof(V)) : (unsigned)(w.rows * (a.row_bytes / (int)sizeof(V)));
    const unsigned apart = (unsigned)(a.run_bytes / (int)sizeof(V));
    const unsigned first = (unsigned)w.piece * p.steps * (PG_THREADS * PG_VECS);
    const unsigned total = min(whole ? per : per * (unsigned)a.runs, first + p.steps * (PG_THREADS * PG_VECS));
    for (unsigned v0 = first + threadIdx.x; v0 < total; v0 += PG_THREADS * PG_VECS) {
      V v[PG_VECS];
      unsigned at[PG_VECS];
#pragma unroll
      for (int j = 0; j < PG_VECS; j++) {
        const unsigned e = v0 + j * PG_THREADS;
        if (e < total) {
          const unsigned run = whole ? 0 : e / per;
          at[j] = run * apart + (e - run * per);
          v[j] = pg_load(from + at[j]);
        }
      }
#pragma unroll
      for (int j = 0; j < PG_VECS; j++)
        if (v0 + j * PG_THREADS < total) pg_store(to + at[j], v[j]);
    }
  }
}

template <typename V>
static int pg_launch(PgArgs& a, cudaStream_t stream) {
  // four blocks for every one that is resident (six an SM): an SM that is done early takes more; pieces of 64 KB where that leaves each
  // block one, else of 16 KB
  const long long blocks = 24LL * sllm_sm_count();
  for (a.steps = 4; a.steps >= 1; a.steps -= 3) {
    const long long vecs = (long long)a.steps * PG_THREADS * PG_VECS;
    a.first[0] = 0;
    for (int k = 0; k < a.n_areas; k++) {
      PgArea& r = a.area[k];
      const long long chunks = (r.item_bytes / (int)sizeof(V) + vecs - 1) / vecs;
      if (chunks > 0x7fffffffLL) return SLLM_ERR_ARG;
      r.chunks = (int)chunks;
      a.first[k + 1] = a.first[k] + chunks * a.n_pairs * r.units;
    }
    if (a.first[a.n_areas] >= blocks) break;
  }
  if (a.steps < 1) a.steps = 1;
  const long long n = a.first[a.n_areas];
  return (int)sllm_launch(page_copy_kernel<V>, dim3((unsigned)(n < blocks ? n : blocks)), dim3(PG_THREADS), 0, stream, a);
}

// areas: n_areas times {from, to, bytes between units of from, of to, bytes of an item (below 2^31), of a run, of a row, units, runs, items
// of from, of to}, as 64-bit words. Runs of an item stand side by side (item_bytes = runs * run_bytes), max_rows rows fill a run.
SLLM_EXPORT int sllm_page_copy(const long long* areas, int n_areas, const int* src, const int* dst, const int* rows, int n_pairs, int max_rows,
                               int* err, cudaStream_t stream) {
  if (n_areas == 0 || n_pairs == 0) return 0;
  if (n_areas < 0 || n_areas > PG_AREAS || n_pairs < 0 || max_rows < 1 || !src || !dst || !err) return SLLM_ERR_ARG;
  PgArgs a;
  a.n_areas = n_areas;
  a.n_pairs = n_pairs;
  a.max_rows = max_rows;
  a.src = src;
  a.dst = dst;
  a.rows = rows;
  a.err = err;
  unsigned long long bits = 0;
  for (int k = 0; k < n_areas; k++) {
    const long long* w = areas + 11 * k;
    PgArea& r = a.area[k];
    r.from = (const char*)w[0];
    r.to = (char*)w[1];
    r.from_unit = w[2];
    r.to_unit = w[3];
    r.item_bytes = w[4];
    r.run_bytes = w[5];
    if (!r.from || !r.to || w[4] < 1 || w[4] > 0x7fffffffLL || w[5] < 1 || w[6] < 1 || w[6] > 0x7fffffffLL || w[7] < 1 || w[7] > 0x7fffffffLL || w[8] < 1 || w[8] > 0x7fffffffLL ||
        w[9] < 0 || w[9] > 0x7fffffffLL || w[10] < 0 || w[10] > 0x7fffffffLL || w[5] != w[6] * max_rows || w[4] != w[5] * w[8])
      return SLLM_ERR_ARG;
    r.row_bytes = (int)w[6];
    r.units = (int)w[7];
    r.runs = (int)w[8];
    r.from_items = (int)w[9];
    r.to_items = (int)w[10];
    bits |= (unsigned long long)w[0] | (unsigned long long)w[1] | (unsigned long long)w[2] | (unsigned long long)w[3] | (unsigned long long)w[6];
  }
  // the widest access that every address and length is a multiple of
  if ((bits & 15) == 0) return pg_launch<uint4>(a, stream);
  if ((bits & 7) == 0) return pg_launch<uint2>(a, stream);
  if ((bits & 3) == 0) return pg_launch<uint32_t>(a, stream);
  if ((bits & 1) == 0) return pg_launch<uint16_t>(a, stream);
  return pg_launch<uint8_t>(a, stream);
}
