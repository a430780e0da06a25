// Attention of a step whose sequences share pages on tcgen05 tensor cores (bfloat16; keys and values of up to 128 dims in multiples of
// 8): every shared run of pages is read once for all rows that see it. The mathematics is at the head of share_kernels.cuh, the plan in
// cache/share.py; results are partial and joined by share_merge_kernel.
//
// One block per SM stays and walks its list of items; barriers, tensor memory, the ring of pages and two query buffers live across items.
// A tile has up to 256 rows (tokens x query heads of one key/value head) and two halves of the block work on it, each with an issuing
// warp, four softmax warps and 256 columns of tensor memory. A tile of more than 128 rows gives each half 128 rows and the same
// pages, so that a page is fetched once for 256 rows; a tile of at most 128 rows is worked on by both halves, which take its pages
// in turn and leave two partial results: the chain of a page (scores, maximum, weights, product with the values), which bounds a tile of
// few rows, then runs twice at a time. Both halves go through the one ring; a half that does not use a page gives it back as it passes.
//
// Tiles of at most 16 rows (one token of a sequence's own pages, as a rule) are thin: 128 rows of tensor memory would be filled for a few.
// They come behind the others, when the ring and its roles are done: each warp has its own list, fetches keys and values by TMA into
// two or three buffers of its own and computes with mma.sync, so that six to eight chains run side by side and memory is what
// bounds them. A plan gives every block its share of either kind.
//
// Rows of a tile belong to several sequences and stand anywhere in the step, so warps gather them (16 bytes a lane, asynchronously,
// into the 128-byte swizzle; the first tile's the softmax warps, the others' a warp of its own) where keys and values come by TMA, a page
// and head at a time. S = Q K^T (128 x 64) and O += P V as in attn_prefill_tcgen05.cu: thread = row = tensor-memory lane, P back into
// tensor memory as bfloat16 pairs (the weights' only rounding; their sum is taken before it), O rescaled only when a row's maximum has
// outgrown its reference by 2^8. With PARTS 2 the weights go into the product in two parts, P and L, that hold a weight to 2^-16 of
// itself, for layers whose other kernels keep them in float32 (outputs 1e-5 to 4e-4 from 32-bit sums rounded once, 1.8e-3 to 2.6e-3 in one
// part; 8 single tokens behind 4,096, heads of 64, 13.7 us, 13.3 in one part; 64 behind 8,192, heads of 128, 41.6, 36.3). Warps whose rows
// are all past the tile's end pass the barriers and compute nothing. Waits are bounded (2 s), after which the kernel raises *err, lets its
// copies land, frees its tensor memory and returns.
//
// Bound by the chain of a page where tiles are full (1.05 us for 256 rows x 64 keys at heads of 128: 1.2 PFLOP/s while it runs, the
// tensor pipe half busy, the exponentials 46% of their unit), by an item's start and end (5 us) and the thin tiles' chains (3 us a page and
// warp) where there are few rows. With the joining kernel: 64 runs of up to 40 tokens behind 16,384 shared ones, 32 heads of 128 on 8, 395
// us (0.91 PFLOP/s; 2,220 each for itself); 64 single tokens behind 8,192 and up to 300 of their own 37 us (73 MB to read and write; 344);
// 8 behind 4,096 and up to 150, 32 heads of 64, 13.5 us (41).
#include "attn_tcgen05.cuh"
#include "share_merge.cuh"
#include <type_traits>

#define FS_THREADS 384       // warp 0: TMA, warps 1-2: the products of either half, warp 3: queries, warps 4-7 and 8-11: softmax of either half
#define FS_ROWS 128          // rows of a half
#define FS_BK SLLM_PAGE
#define FS_CACHED 64         // items that a block keeps decoded in shared memory
#define FS_THIN 16           // rows of a thin tile

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
               ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(bar) : "memory");
}
// 16 bytes from global to shared memory, or 16 zero bytes
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool copy) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(copy ? 16 : 0) : "memory");
}

// this thread's row of tensor memory: 16, or 8, 32-bit columns
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
               ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                 "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// two weights as bfloat16 pairs: rounded (off by 2^-8 of a weight at most), and, with PARTS 2, what that left of them, rounded again (off by
// 2^-16 of a weight: a 256th of what rounding the output to bfloat16 costs)
template <int PARTS>
__device__ __forceinline__ void fs_parts(float u, float v, uint32_t& hi, uint32_t& lo) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(u, v);
  hi = *(const uint32_t*)&h;
  if (PARTS == 2) {
    const __nv_bfloat162 l = __floats2bfloat162_rn(u - __uint_as_float(hi << 16), v - __uint_as_float(hi & 0xffff0000u));
    lo = *(const uint32_t*)&l;
  }
}

// an 8 x 8 matrix of 16-bit elements, two of a row in each lane, turned over
__device__ __forceinline__ uint32_t transposed8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// the 32 lanes' rows of queries, from row r32 of a buffer's n on, into the buffer at sQ: 64-wide blocks of FS_ROWS rows, 128-byte swizzle;
// `row`: this lane's row's address
template <int KD>
__device__ __forceinline__ void fs_gather32(unsigned long long row, uint32_t sQ, int r32, int n, int k_vecs, int k_used, int lane) {
  constexpr int VECS = KD / 8;                    // 16-byte vectors of a row: 32 / VECS rows go together, a lane to a vector
  const int c = lane % VECS;
#pragma unroll
  for (int e = 0; e < VECS; e++) {
    const int r = r32 + e * (32 / VECS) + lane / VECS;
    const char* from = (const char*)__shfl_sync(0xffffffffu, row, r & 31);
    if (r < n && c < k_used)
      cp_async16(sQ + (c >> 3) * (FS_ROWS * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4), from + (c < k_vecs ? 16 * c : 0), c < k_vecs);
  }
}
__device__ __forceinline__ unsigned long long fs_row(const ShareArgs& p, const ShareItem& it, int rho, int rep) {
  const int r = min(rho, it.n_tok * rep - 1);
  return (unsigned long long)((const bf16*)p.q + (size_t)p.toks[it.tok0 + r / rep] * p.q_ld + (size_t)(it.g * rep + r % rep) * p.hd);
}

// warps with thin tiles, and the buffers (a page of keys or of values) that each has
template <int KD, int VD>
__host__ __device__ constexpr int fs_thin_warps() { return KD <= 64 && VD <= 64 ? 8 : KD > 64 && VD > 64 ? 7 : 6; }
template <int KD, int VD>
__host__ __device__ constexpr int fs_thin_bufs() { return KD <= 64 && VD <= 64 ? 3 : 2; }

// One warp's thin items [i0, i1): a page's keys, then its values, into the buffer that comes round, fetched as far ahead as there are
// buffers (across items: a cursor walks the list in front of the work). Keys, and dims of the values, are the 16 rows of mma.m16n8k16 and
// the tile's rows its 8 columns, twice where it has more than 8: half the products of the other way round for the usual tile, whose few
// rows would leave most of 16 empty. Lane (r = lane / 4, c = lane % 4) has of the scores keys 16 n + r and + 8 of rows 2 c and 2 c + 1,
// of the output their dims 16 d + r and + 8.
template <int KD, int VD, int PARTS>
__device__ __forceinline__ void fs_thin(const CUtensorMap* map_k, const CUtensorMap* map_v, const ShareArgs& p, int i0, int i1, uint8_t* buf,
                                        uint32_t bar, volatile int* abort) {
  constexpr uint32_t K_BYTES = FS_BK * KD * 2, V_BYTES = FS_BK * VD * 2, BUF = K_BYTES > V_BYTES ? K_BYTES : V_BYTES, KA = FS_BK * 128;
  constexpr int NK = KD / 64, NV = VD / 64, BUFS = fs_thin_bufs<KD, VD>();
  const int lane = threadIdx.x & 31, rep = p.H / p.G, r0 = lane >> 2, c2 = 2 * (lane & 3);
  const uint32_t sB = smem_u32(buf);
  const float sc = p.scale * FT_LOG2E;
  if (i0 >= i1) return;

  // ---- 32 items at a time are held one a lane, with their first token and the ids of their first four pages: what an item needs before
  // its first product is then on the way together (one by one, each item was three loads deep: 4 us)
  int hbase = i0;
  ShareItem held;
  int tok_first = 0, page4[4];
  auto hold = [&](int base) {
    hbase = base;
    if (base + lane < i1) {
      held = share_item(p, base + lane);
      share_check(p, held);
      tok_first = p.toks[held.tok0];
      const int* row = p.block_table + (size_t)held.seq * p.max_pages;
#pragma unroll
      for (int k = 0; k < 4; k++) page4[k] = held.p0 + k < held.p1 ? share_page(p, row, held.p0 + k) : -1;
    }
  };
  auto held_item = [&](int i) -> ShareItem {
    const int from = i - hbase;
    ShareItem it;
    it.tok0 = __shfl_sync(0xffffffffu, held.tok0, from);
    it.n_tok = __shfl_sync(0xffffffffu, held.n_tok, from);
    it.g = __shfl_sync(0xffffffffu, held.g, from);
    it.p0 = __shfl_sync(0xffffffffu, held.p0, from);
    it.p1 = __shfl_sync(0xffffffffu, held.p1, from);
    it.last = __shfl_sync(0xffffffffu, held.last, from);
    it.part0 = __shfl_sync(0xffffffffu, held.part0, from);
    it.seq = __shfl_sync(0xffffffffu, held.seq, from);
    return it;
  };
  // ---- the cursor: what is fetched next, among the items held
  int fi = i0, ft = 0, fp0 = 0, fp1 = 0, fg = 0, fseq = 0, fetched = 0, taken = 0;
  auto settle = [&]() {               // to an item that has pages left
    while (ft >= fp1 && ++fi < min(i1, hbase + 32)) {
      const ShareItem f = held_item(fi);
      ft = fp0 = f.p0;
      fp1 = f.p1;
      fg = f.g;
      fseq = f.seq;
    }
  };
  auto fetch = [&]() {                // one buffer: a page's keys if `fetched` is even, else its values
    if (fi >= min(i1, hbase + 32)) return;
    const int b = fetched % BUFS, k = ft - fp0;
    int page;
    if (k < 4) {
      const int mine = k == 0 ? page4[0] : k == 1 ? page4[1] : k == 2 ? page4[2] : page4[3];
      page = __shfl_sync(0xffffffffu, mine, fi - hbase);
    } else {
      page = share_page(p, p.block_table + (size_t)fseq * p.max_pages, ft);
    }
    if (lane == 0) {
      const int at = page < 0 ? p.n_pages : page;
      const uint32_t to = sB + b * BUF, on = bar + 8 * b;
      if (fetched & 1) {
        mbar_expect_tx(on, V_BYTES);
#pragma unroll
        for (int a = 0; a < NV; a++) tma_load_3d(to + a * KA, map_v, 64 * a, fg * FS_BK, at, on);
      } else {
        mbar_expect_tx(on, K_BYTES);
#pragma unroll
        for (int a = 0; a < NK; a++) tma_load_3d(to + a * KA, map_k, 64 * a, fg * FS_BK, at, on);
      }
    }
    __syncwarp();
    if ((fetched & 1) && ++ft >= fp1) settle();
    fetched++;
  };
  auto begin = [&](int base) {        // the buffers are empty: hold the next items and fill them
    hold(base);
    fi = base - 1;
    ft = fp1 = 0;
    settle();
    for (int b = 0; b < BUFS; b++) fetch();
  };
  begin(i0);

  bool ok = true;
  for (int i = i0; ok && i < i1; i++) {
    if (i == hbase + 32) begin(i);
    const ShareItem it = held_item(i);
    const int n_rows = it.n_tok * rep, see0 = share_sees(it, r0, rep), see1 = share_sees(it, r0 + 8, rep);
    const int first = __shfl_sync(0xffffffffu, tok_first, i - hbase);       // (a leaf's tokens follow one another)
    const int t0 = see0 < 0 ? 0 : it.last != SHARE_NODE ? first + r0 / rep : p.toks[it.tok0 + r0 / rep];
    const int t1 = see1 < 0 ? 0 : it.last != SHARE_NODE ? first + (r0 + 8) / rep : p.toks[it.tok0 + (r0 + 8) / rep];
    const bf16* q0 = (const bf16*)p.q + (see0 < 0 ? 0 : (size_t)t0 * p.q_ld + (size_t)(it.g * rep + r0 % rep) * p.hd);
    const bf16* q1 = (const bf16*)p.q + (see1 < 0 ? 0 : (size_t)t1 * p.q_ld + (size_t)(it.g * rep + (r0 + 8) % rep) * p.hd);
    auto work = [&](auto groups) {                    // 1: up to 8 rows, 2: up to 16
    constexpr int GROUPS = decltype(groups)::value;
    uint32_t q[GROUPS][KD / 16][2];                      // queries of rows r0 and r0 + 8: the second operand of the scores' products
#pragma unroll
    for (int k = 0; k < KD / 16; k++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const int d = 16 * k + c2 + 8 * e;
        q[0][k][e] = d < p.hd && see0 >= 0 ? *(const uint32_t*)(q0 + d) : 0u;
        if (GROUPS == 2) q[GROUPS - 1][k][e] = d < p.hd && see1 >= 0 ? *(const uint32_t*)(q1 + d) : 0u;
      }
    int see[GROUPS][2];                                  // of rows c2, c2 + 1 and of those 8 on
    float o[GROUPS][VD / 16][4], m[GROUPS][2], l[GROUPS][2];
#pragma unroll
    for (int x = 0; x < GROUPS; x++) {
#pragma unroll
      for (int e = 0; e < 2; e++) {
        see[x][e] = share_sees(it, 8 * x + c2 + e, rep);
        m[x][e] = -INFINITY;
        l[x][e] = 0.f;
      }
#pragma unroll
      for (int d = 0; d < VD / 16; d++)
#pragma unroll
        for (int e = 0; e < 4; e++) o[x][d][e] = 0.f;
    }
    const bool masked = it.last != SHARE_NODE;
    for (int t = it.p0; t < it.p1; t++) {
      float s[GROUPS][4][4];
#pragma unroll
      for (int x = 0; x < GROUPS; x++)
#pragma unroll
        for (int n = 0; n < 4; n++)
#pragma unroll
          for (int e = 0; e < 4; e++) s[x][n][e] = 0.f;
      {
        const int b = taken % BUFS;
        ok = mbar_wait(bar + 8 * b, (taken / BUFS) & 1, abort);
        if (!ok) return;
        const uint32_t from = sB + b * BUF, key = (lane & 7) + (((lane >> 3) & 1) << 3), ch = lane >> 4;
        // (a step's four matrices are on their way while the products of the step before run: in turn with them each load's 33 clocks show)
        uint32_t r[2][4][4];
        auto load = [&](int k) {
#pragma unroll
          for (int n = 0; n < 4; n++) {
            const uint32_t row = 16 * n + key, c = (2 * k + ch) & 7;
            ldmatrix4(from + (k >> 2) * KA + row * 128 + ((c ^ (row & 7)) << 4), r[k & 1][n]);
          }
        };
        load(0);
#pragma unroll
        for (int k = 0; k < KD / 16; k++) {
          if (k + 1 < KD / 16) load(k + 1);          // (past hd: zeros)
#pragma unroll
          for (int x = 0; x < GROUPS; x++)
#pragma unroll
            for (int n = 0; n < 4; n++) mma16816(s[x][n], r[k & 1][n], q[x][k][0], q[x][k][1]);
        }
        taken++;
        __syncwarp();
        fetch();
      }
      uint32_t w[PARTS][GROUPS][4][2];           // weights of 16 keys: the second operand of the product with their values
#pragma unroll
      for (int x = 0; x < GROUPS; x++) {
        if (p.softcap > 0.f) {
          const float cap_out = p.softcap / p.scale, cap_in = p.scale / p.softcap;
#pragma unroll
          for (int n = 0; n < 4; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) s[x][n][e] = __uint_as_float(ft_cap(__float_as_uint(s[x][n][e]), cap_out, cap_in));
        }
        if (masked && t * FS_BK + FS_BK - 1 > it.last - (it.n_tok - 1)) {      // (rows past the tile's end see nothing here, zeros elsewhere)
#pragma unroll
          for (int n = 0; n < 4; n++)
#pragma unroll
            for (int e = 0; e < 4; e++)
              if (t * FS_BK + 16 * n + r0 + 8 * (e >> 1) > see[x][e & 1]) s[x][n][e] = -INFINITY;
        }
        float mx[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
          mx[e] = fmaxf(ft_max3(s[x][0][e], s[x][0][e + 2], s[x][1][e]), ft_max3(s[x][1][e + 2], s[x][2][e], s[x][2][e + 2]));
          mx[e] = ft_max3(mx[e], s[x][3][e], s[x][3][e + 2]);
        }
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], d));
          mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], d));
        }
        if (__any_sync(0xffffffffu, mx[0] > m[x][0] || mx[1] > m[x][1])) {
          float f[2];
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const float grown = fmaxf(m[x][e], mx[e]);
            f[e] = m[x][e] == -INFINITY ? 0.f : ft_ex2((m[x][e] - grown) * sc);
            m[x][e] = grown;
            l[x][e] *= f[e];
          }
#pragma unroll
          for (int d = 0; d < VD / 16; d++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[x][d][e] *= f[e & 1];
        }
        const float a0 = m[x][0] == -INFINITY ? 0.f : -m[x][0] * sc, a1 = m[x][1] == -INFINITY ? 0.f : -m[x][1] * sc;
#pragma unroll
        for (int n = 0; n < 4; n++) {
          const float e0 = ft_ex2(fmaf(s[x][n][0], sc, a0)), e1 = ft_ex2(fmaf(s[x][n][1], sc, a1)), e2 = ft_ex2(fmaf(s[x][n][2], sc, a0)), e3 = ft_ex2(fmaf(s[x][n][3], sc, a1));
          l[x][0] += e0 + e2;
          l[x][1] += e1 + e3;
          uint32_t u[2], v[2];
          fs_parts<PARTS>(e0, e1, u[0], u[1]);
          fs_parts<PARTS>(e2, e3, v[0], v[1]);
#pragma unroll
          for (int part = 0; part < PARTS; part++) {
            w[part][x][n][0] = transposed8x8(u[part]);
            w[part][x][n][1] = transposed8x8(v[part]);
          }
        }
      }
      {
        const int b = taken % BUFS;
        ok = mbar_wait(bar + 8 * b, (taken / BUFS) & 1, abort);
        if (!ok) return;
        const uint32_t from = sB + b * BUF;
        const int n_valid = it.last + 1 - t * FS_BK;
        if (n_valid < FS_BK) {           // behind the last token: weights are zero, but 0 * NaN is NaN
          for (int e = lane; e < (FS_BK - n_valid) * 8 * NV; e += 32) {
            const int blk = NV == 1 ? 0 : e & 1, e1 = e / NV;
            *(uint4*)(buf + b * BUF + blk * KA + (n_valid + e1 / 8) * 128 + (e1 % 8) * 16) = make_uint4(0, 0, 0, 0);
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
        }
        const uint32_t key = (lane & 7) + ((lane >> 4) << 3), ch = (lane >> 3) & 1;
        uint32_t r[2][4][4];
        auto load = [&](int n, int d4) {             // 16 keys of 64 dims
#pragma unroll
          for (int d = 0; d < 4; d++) {
            const uint32_t row = 16 * n + key, c = 2 * d + ch;
            ldmatrix4_trans(from + d4 * KA + row * 128 + ((c ^ (row & 7)) << 4), r[n & 1][d]);
          }
        };
#pragma unroll
        for (int d4 = 0; d4 < NV; d4++) {
          load(0, d4);
#pragma unroll
          for (int n = 0; n < 4; n++) {
            if (n < 3) load(n + 1, d4);
#pragma unroll
            for (int part = 0; part < PARTS; part++)
#pragma unroll
              for (int x = 0; x < GROUPS; x++)
#pragma unroll
                for (int d = 0; d < 4; d++) mma16816(o[x][4 * d4 + d], r[n & 1][d], w[part][x][n][0], w[part][x][n][1]);
          }
        }
        taken++;
        __syncwarp();
        fetch();
      }
    }
    if (!ok) return;
    float* ml = p.part + (size_t)p.part_rows * p.vd;
#pragma unroll
    for (int x = 0; x < GROUPS; x++) {
#pragma unroll
      for (int e = 0; e < 2; e++) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[x][e] += __shfl_xor_sync(0xffffffffu, l[x][e], d);
        const int r = 8 * x + c2 + e;
        if (r >= n_rows) continue;
        const size_t at = (size_t)it.part0 + r;
        float any = 0.f;                            // not 0: something is not finite
#pragma unroll
        for (int d = 0; d < VD / 16; d++) any = fmaf(o[x][d][e], 0.f, fmaf(o[x][d][e + 2], 0.f, any));
        if (any != 0.f && l[x][e] < INFINITY) {
          const bf16* qr = (const bf16*)p.q + (size_t)p.toks[it.tok0 + r / rep] * p.q_ld + (size_t)(it.g * rep + r % rep) * p.hd;
#pragma unroll 1
          for (int d = r0; d < p.vd; d += 8) {
            const float4 v = share_sum_by_key(p, it, qr, see[x][e], m[x][e] * sc, d & ~3, it.p0, 1);
            p.part[share_at(at, d & ~3, p.vd) + (d & 3)] = (d & 3) == 0 ? v.x : (d & 3) == 1 ? v.y : (d & 3) == 2 ? v.z : v.w;
          }
        } else {
#pragma unroll
          for (int d = 0; d < VD / 16; d++)
#pragma unroll
            for (int k = 0; k < 2; k++) {
              const int dim = 16 * d + 8 * k + r0;
              if (dim < p.vd) p.part[share_at(at, dim & ~3, p.vd) + (dim & 3)] = o[x][d][e + 2 * k];
            }
        }
        if (r0 == 0) *(float2*)(ml + 2 * at) = make_float2(m[x][e] * sc, l[x][e]);
      }
    }
    };
    if (n_rows <= 8) work(std::integral_constant<int, 1>());
    else work(std::integral_constant<int, 2>());
    if (!ok) break;
    __syncwarp();
  }
  if (!ok || *abort) {                // let the copies that are under way land before the block leaves
    volatile int never = 0;
    for (int j = taken; j < fetched; j++) mbar_wait(bar + 8 * (j % BUFS), (j / BUFS) & 1, &never);
  }
}

// Keys of up to KD and values of up to VD dims (64 or 128 either): narrower ones are filled up with zeros on the chip.
template <int KD, int VD, int STAGES, int PARTS>
__global__ void __launch_bounds__(FS_THREADS, 1)
attn_share_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ ShareArgs p,
                  uint32_t smem_bytes) {
  constexpr uint32_t Q_BYTES = FS_ROWS * KD * 2, K_BYTES = FS_BK * KD * 2, V_BYTES = FS_BK * VD * 2;
  constexpr uint32_t QA = FS_ROWS * 128, KA = FS_BK * 128;     // bytes of one 64-wide block of Q and of a K or V page
  constexpr int NK = KD / 64, NV = VD / 64;
  // tensor-memory columns of a half (256): values of 64 have S0 0-63, S1 64-127, O 128-191, P0 192-223, P1 224-255, and in two parts L0
  // 0-31, L1 64-95 in the place of the scores that they come from; values of 128, whose O takes 128-255, have one S 0-63 and P0 64-95,
  // P1 96-127, and in two parts one P 64-95 and one L 96-127
  constexpr int NBUF = VD > 64 ? 1 : 2, PBUF = VD > 64 && PARTS == 2 ? 1 : 2;
  constexpr uint32_t P_COL0 = VD > 64 ? 64 : 192, P_STEP = 32, L_COL0 = VD > 64 ? 96 : 0, L_STEP = 64, SUB_COLS = 256;
  constexpr int THIN_BUF = K_BYTES > V_BYTES ? K_BYTES : V_BYTES, THIN_BUFS = fs_thin_bufs<KD, VD>(), THIN_WARPS = fs_thin_warps<KD, VD>();
  static_assert(THIN_WARPS * THIN_BUFS * THIN_BUF <= 2 * Q_BYTES + STAGES * (K_BYTES + V_BYTES), "the thin tiles' buffers take the ring's place");
  static_assert(STAGES >= 4, "a half that takes every other page has its next page's scores issued ahead");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  // [two Q][K stages][V stages][barriers]
  const uint32_t sQ = smem_u32(smem), sK = sQ + 2 * Q_BYTES, sV = sK + STAGES * K_BYTES;
  uint64_t* bars = (uint64_t*)(smem + 2 * Q_BYTES + STAGES * (K_BYTES + V_BYTES));
  // q_full[2], q_empty[2], kv_full[ST], kv_empty[ST], then for either half s_full[2], s_empty[2], p_full[2], o_full[2]
  const uint32_t b_qfull = smem_u32(bars), b_qempty = b_qfull + 16, b_kvfull = b_qempty + 16, b_kvempty = b_kvfull + 8 * STAGES,
                 b_sub = b_kvempty + 8 * STAGES;
  constexpr uint32_t SUB_BARS = 64, B_SEMPTY = 16, B_PFULL = 32, B_OFULL = 48;
  uint32_t* tmem_slot = (uint32_t*)(bars + 4 + 2 * STAGES + 16);
  volatile int* abort = (volatile int*)(tmem_slot + 1);
  ShareItem* cached = (ShareItem*)(bars + 4 + 2 * STAGES + 16 + 2 + THIN_WARPS * THIN_BUFS);
  const uint32_t b_thin = smem_u32(bars + 4 + 2 * STAGES + 16 + 2);     // a barrier for every thin buffer
  if ((uint8_t*)(cached + FS_CACHED) > smem_raw + smem_bytes) {      // the 1 KB alignment took more than the launch left room for
    if (threadIdx.x == 0) atomicExch(p.err, 3);
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int a = 0; a < 2; a++) {
      mbar_init(b_qfull + 8 * a, 1);
      mbar_init(b_qempty + 8 * a, 2);                // either issuing warp
    }
    for (int s = 0; s < STAGES; s++) {
      mbar_init(b_kvfull + 8 * s, 1);
      mbar_init(b_kvempty + 8 * s, 2);
    }
    for (int x = 0; x < 2; x++)
      for (int a = 0; a < 2; a++) {
        mbar_init(b_sub + SUB_BARS * x + 8 * a, 1);
        mbar_init(b_sub + SUB_BARS * x + B_SEMPTY + 8 * a, 4);
        mbar_init(b_sub + SUB_BARS * x + B_PFULL + 8 * a, 4);
        mbar_init(b_sub + SUB_BARS * x + B_OFULL + 8 * a, 1);
      }
    for (int a = 0; a < THIN_WARPS * THIN_BUFS; a++) mbar_init(b_thin + 8 * a, 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = *tmem_slot;
  pdl_launch_dependents();               // (behind the allocation: a dependent's block must not take the columns first)
  pdl_wait();

  // Every role walks the same items and counts by itself the pages fetched (JU), the pages its half has taken (J) and the query
  // buffers used (Q: one by a tile of at most 128 rows, two by a larger one); a barrier's phase follows from those counts.
  const int rep = p.H / p.G, i0 = p.first[blockIdx.x], i1 = p.first[blockIdx.x + 1];
  const int k_vecs = p.hd / 8, k_used = (p.hd + 15) / 16 * 2;      // of a query row: what it has, and what the products' steps of 16 dims read
  if (i1 > i0) {
    if (threadIdx.x < min(FS_CACHED, i1 - i0)) cached[threadIdx.x] = share_item(p, i0 + threadIdx.x);
    __syncthreads();
  }
  auto item = [&](int i) -> ShareItem { return i - i0 < FS_CACHED ? cached[i - i0] : share_item(p, i); };
  if (warp == 0) {
    const bool one = elect_one();
    int JU = 0;
    bool ok = true;
    for (int i = i0; ok && i < i1; i++) {
      const ShareItem it = item(i);
      share_check(p, it);
      const int* row = p.block_table + (size_t)it.seq * p.max_pages;
      for (int t0 = it.p0; ok && t0 < it.p1; t0 += 32) {
        // (a page that is none is fetched past the storage's end: zeros)
        const int mine = t0 + lane < it.p1 ? share_page(p, row, t0 + lane) : 0, n = min(32, it.p1 - t0);
        for (int j = 0; j < n; j++) {
          const int page = __shfl_sync(0xffffffffu, mine, j), s = JU % STAGES;
          ok = mbar_wait(b_kvempty + 8 * s, ((JU / STAGES) & 1) ^ 1, abort);      // (the whole warp: lanes that part here stay apart)
          if (!ok) break;
          if (one) {
            const int at = page < 0 ? p.n_pages : page;
            mbar_expect_tx(b_kvfull + 8 * s, K_BYTES + V_BYTES);
#pragma unroll
            for (int a = 0; a < NK; a++) tma_load_3d(sK + s * K_BYTES + a * KA, &map_k, 64 * a, it.g * FS_BK, at, b_kvfull + 8 * s);
#pragma unroll
            for (int a = 0; a < NV; a++) tma_load_3d(sV + s * V_BYTES + a * KA, &map_v, 64 * a, it.g * FS_BK, at, b_kvfull + 8 * s);
          }
          __syncwarp();
          JU++;
        }
      }
    }
    if (lane == 0 && *abort) {            // let the copies that are under way land before the block leaves
      volatile int never = 0;
      for (int j = max(0, JU - STAGES); j < JU; j++) mbar_wait(b_kvfull + 8 * (j % STAGES), (j / STAGES) & 1, &never);
    }
  } else if (warp == 3) {
    int Q = 0;
    bool ok = true;
    for (int i = i0; ok && i < i1; i++) {
      const ShareItem it = item(i);
      const int n_rows = it.n_tok * rep;
      for (int b0 = 0; ok && b0 < n_rows; b0 += FS_ROWS, Q++) {
        if (i == i0) continue;                       // (the softmax warps fetch the first item's, having nothing else to do)
        const int b = Q & 1;
        // the products that read what the buffer held are done
        ok = mbar_wait(b_qempty + 8 * b, ((Q >> 1) & 1) ^ 1, abort);
        if (!ok) break;
        __syncwarp();
        const int n = min(FS_ROWS, n_rows - b0);
        unsigned long long row[FS_ROWS / 32];
#pragma unroll
        for (int k = 0; k < FS_ROWS / 32; k++) row[k] = fs_row(p, it, b0 + 32 * k + lane, rep);
#pragma unroll
        for (int k = 0; k < FS_ROWS / 32; k++) {
          if (32 * k >= n) break;
          fs_gather32<KD>(row[k], sQ + b * Q_BYTES, 32 * k, n, k_vecs, k_used, lane);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(b_qfull + 8 * b);
      }
    }
  } else if (warp <= 2) {
    const bool one = elect_one();
    const int x = warp - 1;
    constexpr uint32_t idesc_s = umma_idesc_bf16(FS_ROWS, FS_BK);          // S = Q K^T: both K-major
    constexpr uint32_t idesc_o = umma_idesc_bf16_bmn(FS_ROWS, VD);         // O = P V: V is MN-major (dims contiguous)
    const uint32_t b_sfull = b_sub + SUB_BARS * x, b_sempty = b_sfull + B_SEMPTY, b_pfull = b_sfull + B_PFULL, b_ofull = b_sfull + B_OFULL;
    const uint32_t t_sub = tmem_base + x * SUB_COLS;
    int JU0 = 0, J0 = 0, Q = 0;
    bool ok = true;
    for (int i = i0; ok && i < i1; i++) {
      const ShareItem it = item(i);
      const bool pair = it.n_tok * rep > FS_ROWS;
      const int n = it.p1 - it.p0, step = pair ? 1 : 2, u0 = pair ? 0 : x, n_mine = n > u0 ? (n - u0 + step - 1) / step : 0;
      const int mine = pair ? Q + x : Q, b = mine & 1;
      ok = mbar_wait(b_qfull + 8 * b, (mine >> 1) & 1, abort);
      if (!ok) break;
      if (n_mine <= 0 && one) mbar_arrive(b_qempty + 8 * b);
      auto issue_s = [&](int j) -> bool {
        const int JUg = JU0 + u0 + j * step, s = JUg % STAGES, Jg = J0 + j, sb = Jg % NBUF;
        if (!mbar_wait(b_kvfull + 8 * s, (JUg / STAGES) & 1, abort)) return false;
        // S(Jg) takes the place of S(Jg - NBUF), which the softmax threads have taken into their registers: with two buffers their
        // P(Jg - 2) was waited for (and L(Jg - 2) is there until the product that reads it is complete); the single buffer has a
        // barrier for it
        if (NBUF == 1 && !mbar_wait(b_sempty + 8 * sb, ((Jg / NBUF) & 1) ^ 1, abort)) return false;
        if (NBUF == 2 && PARTS == 2 && Jg >= 2 && !mbar_wait(b_ofull + 8 * sb, ((Jg - 2) >> 1) & 1, abort)) return false;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
        for (int k = 0; k < KD / 16; k++)         // 16 dims a step: four steps in each 64-wide block
          if (16 * k < p.hd && one)
            umma_bf16(t_sub + sb * 64, umma_desc_sw128(sQ + b * Q_BYTES + (k >> 2) * QA + (k & 3) * 32),
                      umma_desc_sw128(sK + s * K_BYTES + (k >> 2) * KA + (k & 3) * 32), idesc_s, k ? 1u : 0u);
        if (one) {
          umma_commit(b_sfull + 8 * sb);
          if (j == n_mine - 1) umma_commit(b_qempty + 8 * b);     // the item's last product of this half that reads Q
        }
        return true;
      };
      if (n_mine > 0) ok = issue_s(0);
      for (int u = 0, j = 0; u < n && ok; u++) {
        const int JUg = JU0 + u, s = JUg % STAGES;
        if (!pair && (u & 1) != x) {           // the other half's page
          ok = mbar_wait(b_kvfull + 8 * s, (JUg / STAGES) & 1, abort);
          if (ok && one) mbar_arrive(b_kvempty + 8 * s);
          continue;
        }
        if (j + 1 < n_mine) {
          ok = issue_s(j + 1);
          if (!ok) break;
        }
        const int Jg = J0 + j, a = Jg & 1;
        ok = mbar_wait(b_pfull + 8 * a, (Jg >> 1) & 1, abort);   // P of this page is written, and O has been rescaled if it had to be
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
        for (int k = 0; k < FS_BK / 16; k++)
          if (one) {
            const uint64_t v = umma_desc_sw128_mn(sV + s * V_BYTES + k * 2048, NV > 1 ? KA : 0);
            umma_bf16_ta(t_sub + 128, t_sub + P_COL0 + (PBUF == 2 ? a : 0) * P_STEP + k * 8, v, idesc_o, (j | k) ? 1u : 0u);
            if (PARTS == 2) umma_bf16_ta(t_sub + 128, t_sub + L_COL0 + (PBUF == 2 ? a : 0) * L_STEP + k * 8, v, idesc_o, 1u);
          }
        if (one) {
          umma_commit(b_ofull + 8 * a);
          umma_commit(b_kvempty + 8 * s);
        }
        j++;
      }
      if (ok && pair) {                     // the other half's buffer: not read, given back
        const int other = Q + 1 - x;
        ok = mbar_wait(b_qfull + 8 * (other & 1), (other >> 1) & 1, abort);
        if (ok && one) mbar_arrive(b_qempty + 8 * (other & 1));
      }
      Q += pair ? 2 : 1;
      JU0 += max(0, n);
      J0 += n_mine;
    }
  } else {
    const int x = (warp >> 2) - 1;                 // which half
    const int q = warp & 3;                        // tensor-memory quarter of this warp
    const int r = q * 32 + lane;                   // row of this thread in the half
    const float sc = p.scale * FT_LOG2E;
    const uint32_t t_lane = tmem_base + x * SUB_COLS + ((uint32_t)(q * 32) << 16);
    const uint32_t b_sfull = b_sub + SUB_BARS * x, b_sempty = b_sfull + B_SEMPTY, b_pfull = b_sfull + B_PFULL, b_ofull = b_sfull + B_OFULL;
    float* const ml = p.part + (size_t)p.part_rows * p.vd;
    int JU0 = 0, J0 = 0;
    bool ok = true;
    if (i0 < i1) {                                 // the first item's queries: this half's buffer, 32 rows a warp
      const ShareItem it = item(i0);
      const int n_rows = it.n_tok * rep, n = min(FS_ROWS, n_rows - x * FS_ROWS);
      if (n > 0) {
        if (32 * q < n) fs_gather32<KD>(fs_row(p, it, x * FS_ROWS + r, rep), sQ + x * Q_BYTES, 32 * q, n, k_vecs, k_used, lane);
        asm volatile("cp.async.wait_all;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        asm volatile("bar.sync %0, 128;" ::"r"(1 + x) : "memory");
        if (q == 0 && lane == 0) mbar_arrive(b_qfull + 8 * x);
      }
    }
    for (int i = i0; ok && i < i1; i++) {
      const ShareItem it = item(i);
      const int n_rows = it.n_tok * rep;
      const bool pair = n_rows > FS_ROWS;
      const int n = it.p1 - it.p0, step = pair ? 1 : 2, u0 = pair ? 0 : x, n_mine = n > u0 ? (n - u0 + step - 1) / step : 0;
      const int rho = pair ? x * FS_ROWS + r : r;                       // row of the tile
      const bool warp_has_rows = rho - lane < n_rows, has_row = rho < n_rows;
      const int qpos = share_sees(it, rho, rep);
      float m_ref = -INFINITY, l = 0.f;              // reference maximum (raw score units) and sum relative to it
#pragma unroll 1
      for (int j = 0; j < n_mine && ok; j++) {
        const int Jg = J0 + j, a = Jg & 1, bf = Jg % NBUF, u = u0 + j * step, t = it.p0 + u;
        uint32_t pk[32], pl[32];                      // 64 weights as bfloat16 pairs: keys 2i, 2i+1, and their second parts
        ok = mbar_wait(b_sfull + 8 * bf, (Jg / NBUF) & 1, abort);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (warp_has_rows) {
          uint32_t s[64];
          ft_ld64(t_lane + bf * 64, s);
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
          if (NBUF == 1) {                // the one S buffer may take the next page's scores
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(b_sempty + 8 * bf);
          }
          if (p.softcap > 0.f) {
            const float cap_out = p.softcap / p.scale, cap_in = p.scale / p.softcap;
#pragma unroll
            for (int k = 0; k < 64; k++) s[k] = ft_cap(s[k], cap_out, cap_in);
          }
          if (t * FS_BK + FS_BK - 1 > qpos) {
#pragma unroll
            for (int k = 0; k < 64; k++)
              if (t * FS_BK + k > qpos) s[k] = 0xff800000u;   // -inf
          }
          const float mx = ft_rowmax(s);
          // ---- move the reference maximum only when the row's maximum has outgrown it by 2^8
          const bool grow = mx > m_ref && (m_ref == -INFINITY || (mx - m_ref) * sc > 8.0f);
          if (__any_sync(0xffffffffu, grow)) {
            const float factor = grow ? ((m_ref == -INFINITY) ? 0.f : ft_ex2((m_ref - mx) * sc)) : 1.f;
            if (j >= 1) {
              // O holds the products of the pages before: they must be complete before it is rewritten
              ok = mbar_wait(b_ofull + 8 * (a ^ 1), ((Jg - 1) >> 1) & 1, abort);
              if (!ok) break;
              asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
              uint32_t v[32];
#pragma unroll 1
              for (int c0 = 0; c0 < VD; c0 += 32) {
                tmem_ld32(t_lane + 128 + c0, v);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                for (int k = 0; k < 32; k++) v[k] = __float_as_uint(__uint_as_float(v[k]) * factor);
                tmem_st32(t_lane + 128 + c0, v);
              }
              asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
              asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            }
            l *= factor;
            if (grow) m_ref = mx;
          }
          // ---- the weights, into tensor memory as they come (all at once behind the last: 3% slower). With two buffers the product that
          // read this one's last P, two pages ago, is complete: it was issued before S(Jg), and the commit that announced S(Jg) covers
          // every product issued before it.
          const uint32_t t_p = t_lane + P_COL0 + (PBUF == 2 ? a : 0) * P_STEP, t_l = t_lane + L_COL0 + (PBUF == 2 ? a : 0) * L_STEP;
          if (PBUF == 1 && j >= 1) {                    // the one buffer's last P and L are read when the product of the page before is complete
            ok = mbar_wait(b_ofull + 8 * (a ^ 1), ((Jg - 1) >> 1) & 1, abort);
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          }
          const float msc = (m_ref == -INFINITY) ? 0.f : m_ref * sc;
          uint64_t rs2 = 0ull;                          // two partial sums side by side
          const uint64_t sc2 = ft_pack2(sc, sc), nm2 = ft_pack2(-msc, -msc);
#pragma unroll
          for (int k = 0; k < 32; k += 2) {
            float x0, x1, x2, x3;
            ft_unpack2(ft_fma2(ft_pack2(__uint_as_float(s[2 * k]), __uint_as_float(s[2 * k + 1])), sc2, nm2), x0, x1);
            ft_unpack2(ft_fma2(ft_pack2(__uint_as_float(s[2 * k + 2]), __uint_as_float(s[2 * k + 3])), sc2, nm2), x2, x3);
            const float e0 = ft_ex2(x0), e1 = ft_ex2(x1), e2 = ft_ex2(x2), e3 = ft_ex2(x3);
            rs2 = ft_add2(rs2, ft_add2(ft_pack2(e0, e1), ft_pack2(e2, e3)));
            fs_parts<PARTS>(e0, e1, pk[k], pl[k]);
            fs_parts<PARTS>(e2, e3, pk[k + 1], pl[k + 1]);
            if (k == 14) {
              tmem_st16(t_p, pk);
              if (PARTS == 2) tmem_st16(t_l, pl);
            }
            if (k == 22) {
              tmem_st8(t_p + 16, pk + 16);
              if (PARTS == 2) tmem_st8(t_l + 16, pl + 16);
            }
          }
          tmem_st8(t_p + 24, pk + 24);
          if (PARTS == 2) tmem_st8(t_l + 24, pl + 24);
          float ra, rb;
          ft_unpack2(rs2, ra, rb);
          l += ra + rb;
        } else if (NBUF == 1) {
          if (lane == 0) mbar_arrive(b_sempty + 8 * bf);
        }
        if (t * FS_BK + FS_BK - 1 > it.last) {
          // keys behind the tile's last token hold whatever the page held before, or what this tile does not see: their weights are
          // zero, but 0 * NaN is NaN, so their value rows are cleared, by either half before its own product
          const int JUg = JU0 + u, st = JUg % STAGES, n_valid = max(0, it.last + 1 - t * FS_BK);
          ok = mbar_wait(b_kvfull + 8 * st, (JUg / STAGES) & 1, abort);
          if (!ok) break;
          for (int e = q * 32 + lane; e < (FS_BK - n_valid) * 8 * NV; e += 128) {
            const int blk = e / ((FS_BK - n_valid) * 8), e1 = e % ((FS_BK - n_valid) * 8), vr = n_valid + e1 / 8, c = e1 % 8;
            *(uint4*)(smem + 2 * Q_BYTES + STAGES * K_BYTES + st * V_BYTES + blk * KA + vr * 128 + ((c ^ (vr & 7)) << 4)) = make_uint4(0, 0, 0, 0);
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        if (warp_has_rows) asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(b_pfull + 8 * a);
      }
      if (ok && n_mine > 0) ok = mbar_wait(b_ofull + 8 * ((J0 + n_mine - 1) & 1), ((J0 + n_mine - 1) >> 1) & 1, abort);
      if (ok && warp_has_rows) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const size_t at = (size_t)it.part0 + rho + (pair || x == 0 ? 0 : n_rows);
        const float m = m_ref * sc;
        if (n_mine > 0) {
#pragma unroll 1
          for (int c0 = 0; c0 < VD; c0 += 32) {
            uint32_t v[32];
            tmem_ld32(t_lane + 128 + c0, v);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            float any = 0.f;                            // not 0: something is not finite (a sum l that is not has seen a score that is not)
#pragma unroll
            for (int k = 0; k < 32; k++) any = fmaf(__uint_as_float(v[k]), 0.f, any);
            if (has_row) {
              if (any != 0.f && l < INFINITY) {
                const bf16* qr = (const bf16*)p.q + (size_t)p.toks[it.tok0 + rho / rep] * p.q_ld + (size_t)(it.g * rep + rho % rep) * p.hd;
#pragma unroll 1
                for (int c = 0; c < 32 && c0 + c < p.vd; c += 4)
                  *(float4*)(p.part + share_at(at, c0 + c, p.vd)) = share_sum_by_key(p, it, qr, qpos, m, c0 + c, it.p0 + u0, step);
              } else {
#pragma unroll
                for (int c = 0; c < 32; c += 4)
                  if (c0 + c < p.vd)
                    *(float4*)(p.part + share_at(at, c0 + c, p.vd)) = make_float4(__uint_as_float(v[c]), __uint_as_float(v[c + 1]),
                                                                                  __uint_as_float(v[c + 2]), __uint_as_float(v[c + 3]));
              }
            }
            __syncwarp();
          }
        }
        if (has_row) *(float2*)(ml + 2 * at) = make_float2(m, l);
      }
      // the rows of O are read (the loads above were waited for) before this thread signals the next item's first P
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      JU0 += max(0, n);
      J0 += n_mine;
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp < THIN_WARPS && !*abort) {
    const int w = blockIdx.x * THIN_WARPS + warp;
    fs_thin<KD, VD, PARTS>(&map_k, &map_v, p, p.thin_first[w], p.thin_first[w + 1], smem + warp * THIN_BUFS * THIN_BUF, b_thin + 8 * warp * THIN_BUFS, abort);
  }
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512) : "memory");
  if (lane == 0 && *abort) atomicExch(p.err, 2);
}

// pages [n_pages][G * 64][width] bfloat16; a box is 64 columns of one head's 64 positions, 128-byte swizzle, zero fill
static int fs_make_map(CUtensorMap* map, const void* base, long long n_pages, int G, int width) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return SLLM_ERR_ARG - 1;
  cuuint64_t dims[3] = {(cuuint64_t)width, (cuuint64_t)G * FS_BK, (cuuint64_t)n_pages};
  cuuint64_t strides[2] = {(cuuint64_t)width * 2, (cuuint64_t)G * FS_BK * width * 2};
  cuuint32_t box[3] = {64, FS_BK, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : SLLM_ERR_ARG - 2;
}

template <int KD, int VD, int STAGES, int PARTS>
static int fs_launch_parts(const CUtensorMap& mk, const CUtensorMap& mv, const ShareArgs& a, int workers, cudaStream_t stream) {
  // what the kernel lays out after aligning to 1 KB; one block on an SM
  constexpr size_t need = 2 * FS_ROWS * KD * 2 + STAGES * FS_BK * (KD + VD) * 2 + (4 + 2 * STAGES + 16 + 2 + fs_thin_warps<KD, VD>() * fs_thin_bufs<KD, VD>()) * 8 +
                          FS_CACHED * sizeof(ShareItem);
  constexpr size_t room = 232448;
  constexpr size_t smem = need + 1024 <= room ? need + 1024 : room;     // the slack for the alignment, as far as it fits
  static_assert(need + 512 <= smem, "the block of this head width does not fit an SM");
  static SllmPerDevice allowed;
  const cudaError_t e = sllm_allow_smem(allowed, attn_share_kernel<KD, VD, STAGES, PARTS>, smem);
  if (e != cudaSuccess) return (int)e;
  return (int)sllm_launch(attn_share_kernel<KD, VD, STAGES, PARTS>, dim3(workers), dim3(FS_THREADS), smem, stream, mk, mv, a, (uint32_t)smem);
}
template <int KD, int VD, int STAGES>
static int fs_launch(const CUtensorMap& mk, const CUtensorMap& mv, const ShareArgs& a, int workers, int exact, cudaStream_t stream) {
  return exact ? fs_launch_parts<KD, VD, STAGES, 2>(mk, mv, a, workers, stream) : fs_launch_parts<KD, VD, STAGES, 1>(mk, mv, a, workers, stream);
}

// The plan is one for tiles of 256 rows in halves, with thin ones of at most FS_THIN rows; part: plan->part_rows * (vd + 2) floats; exact:
// the weights go into the product with the values in two parts.
SLLM_EXPORT int sllm_share_attn_tc_bf16(const SharePlanDev* plan, const void* q, int q_ld, const int* tok_pos, const int* block_table,
                                        int max_pages, const void* kpages, const void* vpages, long long n_pages, float* part, void* out,
                                        const float* sink, int hd, int vd, float scale, float softcap, int exact, int* err,
                                        cudaStream_t stream) {
  if (hd < 8 || hd > 128 || hd % 8 || vd < 8 || vd > 128 || vd % 8 || (q_ld & 7) || !share_call_ok(*plan, 2 * FS_ROWS, q_ld, hd, n_pages, max_pages, part) ||
      plan->thin_warps != (hd <= 64 && vd <= 64 ? fs_thin_warps<64, 64>() : hd > 64 && vd > 64 ? fs_thin_warps<128, 128>() : fs_thin_warps<128, 64>()) || !share_aligned(q, 16) ||
      !share_aligned(kpages, 16) || !share_aligned(vpages, 16) || !share_aligned(out, 16))
    return SLLM_ERR_ARG;
  if (plan->T == 0) return 0;
  const ShareArgs a = share_args(*plan, q, q_ld, tok_pos, block_table, max_pages, kpages, vpages, n_pages, part, hd, vd, scale, softcap, err);
  CUtensorMap mk, mv;
  int rc = fs_make_map(&mk, kpages, n_pages, plan->G, hd);
  if (rc == 0) rc = fs_make_map(&mv, vpages, n_pages, plan->G, vd);
  if (rc) return rc;
  const int workers = plan->workers;
  if (vd <= 64) rc = hd <= 64 ? fs_launch<64, 64, 10>(mk, mv, a, workers, exact, stream) : fs_launch<128, 64, 6>(mk, mv, a, workers, exact, stream);
  else rc = hd <= 64 ? fs_launch<64, 128, 7>(mk, mv, a, workers, exact, stream) : fs_launch<128, 128, 5>(mk, mv, a, workers, exact, stream);
  return rc ? rc : share_merge_run<bf16>(*plan, part, out, sink, vd, stream);
}
