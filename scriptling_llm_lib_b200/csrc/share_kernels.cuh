// Attention for a step whose sequences share pages, read once for all that share them: the form for any width and precision on FP32
// FMA, and the kernel that joins partial results. (The tcgen05 form is in attn_share_tcgen05.cu; the reference holds one sequence,
// model_f32.go:310-317, and has none of this.)
//
// The work comes as a plan (cache/share.py): items of a few tokens ("a tile": the tokens' query heads on one key/value head are its rows)
// over a run of pages that all of the tile's tokens see the front of. A row's softmax over its keys is split exactly over the items that
// it is in: an item leaves, for each row, m = the largest score it saw, l = sum of 2^(s - m) and o = sum of 2^(s - m) v, all float32
// (scores in units of log2 e), and share_merge_kernel joins them,
//   out = sum_i 2^(m_i - M) o_i / (sum_i 2^(m_i - M) l_i + 2^(sink log2 e - M)),   M the largest of the m_i and the sink,
// in the order of the plan's list, so that a call's result does not change from run to run.
#pragma once
#include "share_merge.cuh"

// ------------------------------------------------------------------ FP32 FMA tiles
// A block of 256 threads: up to 64 rows (16 where a tile has no more: QPT 1) against a page of 64 keys at a time. Thread (ty = tid / 16,
// tx = tid % 16) has rows QPT ty .. of the tile, keys tx, tx + 16, .. of the page's scores and the dims 4 (tx + 16 g) .. + 3 of the
// output. Queries, keys and values stand in shared memory as rows (keys and values as they are stored, rows padded by 16 bytes against
// bank conflicts), the next page on its way by asynchronous copies while one is worked on, where two fit. Bound by FMA issue and the
// shared-memory reads that feed it (a 4 x 4 register tile: 128 bytes for 64 FMAs); a tile of few rows by those reads alone. 32-bit, 5 runs
// of up to 33 tokens behind 600, 16 heads of 64 on 4: 29 us with the joining kernel (87 each for itself); 12 single tokens behind 1,000, 32 heads on 8, 20
// us (23.5).
#define SF_ROWS 64
#define SF_PS (SLLM_PAGE + 4)

template <typename A>
__host__ __device__ __forceinline__ int share_row_len(int width) { return width + 16 / (int)sizeof(A); }
// bytes of shared memory with `stages` pages
template <typename A>
static inline size_t share_fma_smem(int hd, int vd, int stages) {
  return ((size_t)SF_ROWS * (hd + 4) + (size_t)SF_ROWS * SF_PS) * 4 + (size_t)stages * SLLM_PAGE * (share_row_len<A>(hd) + share_row_len<A>(vd)) * sizeof(A);
}
// four elements from global to shared memory, or zeros
template <typename A>
__device__ __forceinline__ void share_copy4(A* to, const A* from, bool copy) {
  const uint32_t dst = (uint32_t)__cvta_generic_to_shared(to);
  if constexpr (sizeof(A) == 4) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(from), "r"(copy ? 16 : 0) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(from), "r"(copy ? 8 : 0) : "memory");
}

template <typename A, int NG, int QPT>
__device__ __forceinline__ void share_fma_item(const ShareArgs& p, const ShareItem& it, int stages, float* sm) {
  const int hd = p.hd, vd = p.vd, rep = p.H / p.G, n_rows = it.n_tok * rep, kq = hd >> 2, vq = vd >> 2;
  const int ql = hd + 4, kl = share_row_len<A>(hd), vl = share_row_len<A>(vd);
  float* Qs = sm;                              // [64][ql]
  float* Ps = Qs + SF_ROWS * ql;               // [64][68]
  A* Ks = (A*)(Ps + SF_ROWS * SF_PS);          // [stages][64][kl]
  A* Vs = Ks + stages * SLLM_PAGE * kl;        // [stages][64][vl]
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const A *kp = (const A*)p.kpages, *vp = (const A*)p.vpages;
  const int* row = p.block_table + (size_t)it.seq * p.max_pages;

  // a thread's place in a row of four-element pieces, and its first row, of keys and of values
  const int kd = 4 * (tid % kq), k0 = tid < 256 / kq * kq ? tid / kq : SLLM_PAGE, vd0 = 4 * (tid % vq), v0 = tid < 256 / vq * vq ? tid / vq : SLLM_PAGE;
  auto fetch = [&](int t) {                    // keys behind the last token, and a page that is none: zeros
    const int page = share_page(p, row, t), n_keys = page < 0 ? 0 : min(SLLM_PAGE, it.last + 1 - t * SLLM_PAGE), s = (t - it.p0) % stages;
    const size_t at = ((size_t)max(page, 0) * p.G + it.g) * SLLM_PAGE;
    for (int kk = k0; kk < SLLM_PAGE; kk += 256 / kq) share_copy4(Ks + (s * SLLM_PAGE + kk) * kl + kd, kp + (at + kk) * hd + kd, kk < n_keys);
    for (int kk = v0; kk < SLLM_PAGE; kk += 256 / vq) share_copy4(Vs + (s * SLLM_PAGE + kk) * vl + vd0, vp + (at + kk) * vd + vd0, kk < n_keys);
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if (it.p0 < it.p1) fetch(it.p0);
  for (int e = tid; e < 16 * QPT * kq; e += 256) {
    const int r = e / kq, d = 4 * (e % kq);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r < n_rows) v = ld4((const A*)p.q + (size_t)p.toks[it.tok0 + r / rep] * p.q_ld + (size_t)(it.g * rep + r % rep) * hd + d);
    *(float4*)(Qs + r * ql + d) = v;
  }
  float m[QPT], l[QPT], o[QPT][NG][4];
  int qpos[QPT];
#pragma unroll
  for (int i = 0; i < QPT; i++) {
    qpos[i] = share_sees(it, ty * QPT + i, rep);
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int gg = 0; gg < NG; gg++)
#pragma unroll
      for (int c = 0; c < 4; c++) o[i][gg][c] = 0.f;
  }
  for (int t = it.p0; t < it.p1; t++) {
    if (stages == 2 && t + 1 < it.p1) {
      fetch(t + 1);
      asm volatile("cp.async.wait_group 1;" ::: "memory");
    } else {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    __syncthreads();
    const A *K = Ks + ((t - it.p0) % stages) * SLLM_PAGE * kl, *V = Vs + ((t - it.p0) % stages) * SLLM_PAGE * vl;
    float s[QPT][4];
#pragma unroll
    for (int i = 0; i < QPT; i++)
#pragma unroll
      for (int j = 0; j < 4; j++) s[i][j] = 0.f;
#pragma unroll 4
    for (int d = 0; d < hd; d += 4) {
      float4 a[QPT], k[4];
#pragma unroll
      for (int i = 0; i < QPT; i++) a[i] = *(const float4*)(Qs + (ty * QPT + i) * ql + d);
#pragma unroll
      for (int j = 0; j < 4; j++) k[j] = ld4(K + (tx + 16 * j) * kl + d);
#pragma unroll
      for (int i = 0; i < QPT; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
          s[i][j] = fmaf(a[i].x, k[j].x, s[i][j]);
          s[i][j] = fmaf(a[i].y, k[j].y, s[i][j]);
          s[i][j] = fmaf(a[i].z, k[j].z, s[i][j]);
          s[i][j] = fmaf(a[i].w, k[j].w, s[i][j]);
        }
    }
#pragma unroll
    for (int i = 0; i < QPT; i++) {
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        float v = s[i][j] * p.scale;
        if (p.softcap > 0.f) v = p.softcap * tanhf(v / p.softcap);
        s[i][j] = t * SLLM_PAGE + tx + 16 * j <= qpos[i] ? v * SHARE_LOG2E : -INFINITY;
        mx = fmaxf(mx, s[i][j]);
      }
#pragma unroll
      for (int off = 1; off < 16; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
      const float m_new = fmaxf(m[i], mx), corr = m_new == -INFINITY ? 1.f : exp2f(m[i] - m_new);
      float rs = 0.f;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float pr = s[i][j] == -INFINITY ? 0.f : exp2f(s[i][j] - m_new);
        rs += pr;
        Ps[(ty * QPT + i) * SF_PS + tx + 16 * j] = pr;
      }
      l[i] = fmaf(l[i], corr, rs);                                      // this lane's share of the row's sum
      m[i] = m_new;
#pragma unroll
      for (int gg = 0; gg < NG; gg++)
#pragma unroll
        for (int c = 0; c < 4; c++) o[i][gg][c] *= corr;
    }
    __syncwarp();                               // (a row's weights are read by the lanes that wrote them)
#pragma unroll 2
    for (int k4 = 0; k4 < SLLM_PAGE; k4 += 4) {
      float pv[QPT][4];
#pragma unroll
      for (int i = 0; i < QPT; i++) {
        const float4 v = *(const float4*)(Ps + (ty * QPT + i) * SF_PS + k4);
        pv[i][0] = v.x; pv[i][1] = v.y; pv[i][2] = v.z; pv[i][3] = v.w;
      }
#pragma unroll
      for (int gg = 0; gg < NG; gg++) {
        const int d0 = (tx + 16 * gg) * 4;
        if (d0 >= vd) continue;
#pragma unroll
        for (int kk = 0; kk < 4; kk++) {
          const float4 v = ld4(V + (k4 + kk) * vl + d0);
#pragma unroll
          for (int i = 0; i < QPT; i++) {
            o[i][gg][0] = fmaf(pv[i][kk], v.x, o[i][gg][0]);
            o[i][gg][1] = fmaf(pv[i][kk], v.y, o[i][gg][1]);
            o[i][gg][2] = fmaf(pv[i][kk], v.z, o[i][gg][2]);
            o[i][gg][3] = fmaf(pv[i][kk], v.w, o[i][gg][3]);
          }
        }
      }
    }
    __syncthreads();                            // this page's place is free
    if (stages == 1 && t + 1 < it.p1) fetch(t + 1);
  }
  float* ml = p.part + (size_t)p.part_rows * vd;
#pragma unroll
  for (int i = 0; i < QPT; i++) {
    const int r = ty * QPT + i;
    float ls = l[i];
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) ls += __shfl_xor_sync(0xffffffffu, ls, off);
    if (r >= n_rows) continue;
    const size_t at = (size_t)it.part0 + r;
#pragma unroll
    for (int gg = 0; gg < NG; gg++) {
      const int d0 = (tx + 16 * gg) * 4;
      if (d0 >= vd) continue;
      float4 v = make_float4(o[i][gg][0], o[i][gg][1], o[i][gg][2], o[i][gg][3]);
      if (!(fabsf(v.x) + fabsf(v.y) + fabsf(v.z) + fabsf(v.w) < INFINITY) && ls < INFINITY)
        v = share_sum_by_key(p, it, (const A*)p.q + (size_t)p.toks[it.tok0 + r / rep] * p.q_ld + (size_t)(it.g * rep + r % rep) * hd, qpos[i], m[i], d0, it.p0, 1);
      *(float4*)(p.part + share_at(at, d0, vd)) = v;
    }
    if (tx == 0) *(float2*)(ml + 2 * at) = make_float2(m[i], ls);
  }
  __syncthreads();                              // the next item's queries take this one's place
}

// The same for tiles of at most 4 rows, a decode step's token on a sequence's own pages as a rule: there the tiles above would read every
// key and value from shared memory 4 times over for 4 times the rows. A key belongs to four neighbouring lanes (a quarter of its dims
// each), a row's weights to one warp, and four dims of the values to a thread, for every kgs-th key; the threads' sums over their keys meet
// once, behind the last page. Keys and values are read from shared memory once (64 sequences of 100 tokens of their own and 1,000 shared,
// 32 heads of 64: 117 us a call, 178 on the tiles above).
template <typename A>
__device__ __forceinline__ void share_few_item(const ShareArgs& p, const ShareItem& it, int stages, float* sm) {
  const int hd = p.hd, vd = p.vd, rep = p.H / p.G, n_rows = it.n_tok * rep, kq = hd >> 2, vq = vd >> 2;
  const int ql = hd + 4, kl = share_row_len<A>(hd), vl = share_row_len<A>(vd), kgs = 256 / vq;
  float* Qs = sm;                              // [4][ql]
  float* Ps = Qs + SF_ROWS * ql;               // [4][64] weights, then the threads' sums
  float* corr = Ps + SF_ROWS * SF_PS - 4;      // [4]
  A* Ks = (A*)(Ps + SF_ROWS * SF_PS);
  A* Vs = Ks + stages * SLLM_PAGE * kl;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, key = tid >> 2, sub = tid & 3, dg = 4 * (tid % vq), kg = tid / vq;
  const int* row = p.block_table + (size_t)it.seq * p.max_pages;
  const A *kp = (const A*)p.kpages, *vp = (const A*)p.vpages;

  const int kd = 4 * (tid % kq), k0 = tid < 256 / kq * kq ? tid / kq : SLLM_PAGE, v0 = kg < kgs ? kg : SLLM_PAGE;
  auto fetch = [&](int t) {                    // keys behind the last token, and a page that is none: zeros
    const int page = share_page(p, row, t), n_keys = page < 0 ? 0 : min(SLLM_PAGE, it.last + 1 - t * SLLM_PAGE), s = (t - it.p0) % stages;
    const size_t at = ((size_t)max(page, 0) * p.G + it.g) * SLLM_PAGE;
    for (int kk = k0; kk < SLLM_PAGE; kk += 256 / kq) share_copy4(Ks + (s * SLLM_PAGE + kk) * kl + kd, kp + (at + kk) * hd + kd, kk < n_keys);
    for (int kk = v0; kk < SLLM_PAGE; kk += kgs) share_copy4(Vs + (s * SLLM_PAGE + kk) * vl + dg, vp + (at + kk) * vd + dg, kk < n_keys);
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if (it.p0 < it.p1) fetch(it.p0);
  for (int e = tid; e < 4 * kq; e += 256) {
    const int r = e / kq, d = 4 * (e % kq);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r < n_rows) v = ld4((const A*)p.q + (size_t)p.toks[it.tok0 + r / rep] * p.q_ld + (size_t)(it.g * rep + r % rep) * hd + d);
    *(float4*)(Qs + r * ql + d) = v;
  }
  const int sees = share_sees(it, sub, rep);   // of row `sub`
  float m = -INFINITY, l = 0.f, o[4][4];       // m, l: of row `warp`, in warps 0 to 3
#pragma unroll
  for (int r = 0; r < 4; r++)
#pragma unroll
    for (int c = 0; c < 4; c++) o[r][c] = 0.f;
  for (int t = it.p0; t < it.p1; t++) {
    if (stages == 2 && t + 1 < it.p1) {
      fetch(t + 1);
      asm volatile("cp.async.wait_group 1;" ::: "memory");
    } else {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    __syncthreads();
    const A *K = Ks + (((t - it.p0) % stages) * SLLM_PAGE + key) * kl, *V = Vs + ((t - it.p0) % stages) * SLLM_PAGE * vl + dg;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int d = 4 * sub; d < hd; d += 16) {
      const float4 k = ld4(K + d);
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const float4 q = *(const float4*)(Qs + r * ql + d);
        s[r] = fmaf(q.x, k.x, s[r]);
        s[r] = fmaf(q.y, k.y, s[r]);
        s[r] = fmaf(q.z, k.z, s[r]);
        s[r] = fmaf(q.w, k.w, s[r]);
      }
    }
#pragma unroll
    for (int r = 0; r < 4; r++) {
      s[r] += __shfl_xor_sync(0xffffffffu, s[r], 1);
      s[r] += __shfl_xor_sync(0xffffffffu, s[r], 2);
    }
    float v = (sub == 0 ? s[0] : sub == 1 ? s[1] : sub == 2 ? s[2] : s[3]) * p.scale;
    if (p.softcap > 0.f) v = p.softcap * tanhf(v / p.softcap);
    Ps[sub * SLLM_PAGE + key] = t * SLLM_PAGE + key <= sees ? v * SHARE_LOG2E : -INFINITY;
    __syncthreads();
    if (warp < 4) {
      const float a = Ps[warp * SLLM_PAGE + lane], b = Ps[warp * SLLM_PAGE + lane + 32];
      const float m_new = fmaxf(m, warp_max(fmaxf(a, b))), f = m_new == -INFINITY ? 1.f : exp2f(m - m_new);
      const float x = a == -INFINITY ? 0.f : exp2f(a - m_new), y = b == -INFINITY ? 0.f : exp2f(b - m_new);
      l = fmaf(l, f, warp_sum(x + y));
      m = m_new;
      Ps[warp * SLLM_PAGE + lane] = x;
      Ps[warp * SLLM_PAGE + lane + 32] = y;
      if (lane == 0) corr[warp] = f;
    }
    __syncthreads();
    if (kg < kgs) {
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const float f = corr[r];
#pragma unroll
        for (int c = 0; c < 4; c++) o[r][c] *= f;
      }
#pragma unroll 4
      for (int kk = kg; kk < SLLM_PAGE; kk += kgs) {
        const float4 x = ld4(V + kk * vl);
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const float w = Ps[r * SLLM_PAGE + kk];
          o[r][0] = fmaf(w, x.x, o[r][0]);
          o[r][1] = fmaf(w, x.y, o[r][1]);
          o[r][2] = fmaf(w, x.z, o[r][2]);
          o[r][3] = fmaf(w, x.w, o[r][3]);
        }
      }
    }
    __syncthreads();                            // this page's place is free, and so are the weights
    if (stages == 1 && t + 1 < it.p1) fetch(t + 1);
  }
  float* ml = p.part + (size_t)p.part_rows * vd;
  if (warp < n_rows && lane == 0) {
    *(float2*)(ml + 2 * ((size_t)it.part0 + warp)) = make_float2(m, l);
    Qs[SF_ROWS * ql - 8 + 2 * warp] = m;        // (behind the queries)
    Qs[SF_ROWS * ql - 7 + 2 * warp] = l;
  }
  if (kg < kgs)
#pragma unroll
    for (int r = 0; r < 4; r++)
      if (r < n_rows) *(float4*)(Ps + ((size_t)kg * n_rows + r) * vd + dg) = make_float4(o[r][0], o[r][1], o[r][2], o[r][3]);
  __syncthreads();
  for (int e = tid; e < n_rows * vq; e += 256) {
    const int r = e / vq, d = 4 * (e % vq);
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < kgs; k++) {
      const float4 b = *(const float4*)(Ps + ((size_t)k * n_rows + r) * vd + d);
      a.x += b.x;
      a.y += b.y;
      a.z += b.z;
      a.w += b.w;
    }
    const float mr = Qs[SF_ROWS * ql - 8 + 2 * r], lr = Qs[SF_ROWS * ql - 7 + 2 * r];
    if (!(fabsf(a.x) + fabsf(a.y) + fabsf(a.z) + fabsf(a.w) < INFINITY) && lr < INFINITY)
      a = share_sum_by_key(p, it, (const A*)p.q + (size_t)p.toks[it.tok0 + r / rep] * p.q_ld + (size_t)(it.g * rep + r % rep) * hd,
                           share_sees(it, r, rep), mr, d, it.p0, 1);
    *(float4*)(p.part + share_at((size_t)it.part0 + r, d, vd)) = a;
  }
  __syncthreads();                              // the next item takes this one's place
}

template <typename A, int NG, int BLOCKS>
__global__ void __launch_bounds__(256, BLOCKS) share_fma_kernel(ShareArgs p, int stages) {
  extern __shared__ __align__(16) float share_sm[];
  pdl_launch_dependents();
  pdl_wait();
  const int i1 = p.first[blockIdx.x + 1];
  for (int i = p.first[blockIdx.x]; i < i1; i++) {
    const ShareItem it = share_item(p, i);
    if (threadIdx.x == 0) share_check(p, it);
    const int n_rows = it.n_tok * (p.H / p.G);
    if (n_rows <= 4) share_few_item<A>(p, it, stages, share_sm);
    else if (n_rows <= 16) share_fma_item<A, NG, 1>(p, it, stages, share_sm);
    else share_fma_item<A, NG, 4>(p, it, stages, share_sm);
  }
}
