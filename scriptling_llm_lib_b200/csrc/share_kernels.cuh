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
#include "share_plan.cuh"

// ------------------------------------------------------------------ FP32 FMA tiles
// A block of 256 threads: up to 64 rows (16 where a tile has no more: QPT 1) against a page of 64 keys at a time. Thread (ty = tid / 16,
// tx = tid % 16) has rows QPT ty .. of the tile, keys 4 tx .. + 3 of the page's scores and the dims 4 (tx + 16 g) .. + 3 of the output.
// Q and K stand in shared memory with their dims outermost, V and the weights by keys; 16-byte accesses. Bound by FMA issue and the
// shared-memory reads that feed it (a 4 x 4 register tile: 32 bytes for 16 FMAs).
#define SF_ROWS 64
#define SF_PS (SLLM_PAGE + 4)

template <typename A, int NG, int QPT>
__device__ __forceinline__ void share_fma_item(const ShareArgs& p, const ShareItem& it, float* sm) {
  constexpr int BQ = 16 * QPT;
  const int hd = p.hd, vd = p.vd, rep = p.H / p.G, n_rows = it.n_tok * rep;
  float* Qs = sm;                              // [hd][BQ]
  float* Ks = Qs + hd * SF_ROWS;               // [hd][64]
  float* Vs = Ks + hd * SLLM_PAGE;             // [64][vd]
  float* Ps = Vs + SLLM_PAGE * vd;             // [BQ][68]
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const A *kp = (const A*)p.kpages, *vp = (const A*)p.vpages;
  const int kq = hd >> 2, vq = vd >> 2;

  for (int e = tid; e < BQ * kq; e += 256) {
    const int r = e % BQ, d = e / BQ;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r < n_rows) v = ld4((const A*)p.q + (size_t)p.toks[it.tok0 + r / rep] * p.q_ld + (size_t)(it.g * rep + r % rep) * hd + 4 * d);
    Qs[(4 * d + 0) * BQ + r] = v.x;
    Qs[(4 * d + 1) * BQ + r] = v.y;
    Qs[(4 * d + 2) * BQ + r] = v.z;
    Qs[(4 * d + 3) * BQ + r] = v.w;
  }
  float m[QPT], l[QPT], o[QPT][NG][4];
  int qpos[QPT];
#pragma unroll
  for (int i = 0; i < QPT; i++) {
    const int r = ty * QPT + i;
    qpos[i] = r < n_rows ? p.tok_pos[p.toks[it.tok0 + r / rep]] : -1;
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int gg = 0; gg < NG; gg++)
#pragma unroll
      for (int c = 0; c < 4; c++) o[i][gg][c] = 0.f;
  }
  const int* row = p.block_table + (size_t)it.seq * p.max_pages;
  for (int t = it.p0; t < it.p1; t++) {
    const int page = share_page(p, row, t), n_keys = page < 0 ? 0 : min(SLLM_PAGE, it.last + 1 - t * SLLM_PAGE);
    const size_t at = ((size_t)max(page, 0) * p.G + it.g) * SLLM_PAGE;
    __syncthreads();
    for (int e = tid; e < SLLM_PAGE * kq; e += 256) {
      const int kk = e % SLLM_PAGE, d = e / SLLM_PAGE;
      const float4 v = kk < n_keys ? ld4(kp + (at + kk) * hd + 4 * d) : make_float4(0.f, 0.f, 0.f, 0.f);
      Ks[(4 * d + 0) * SLLM_PAGE + kk] = v.x;
      Ks[(4 * d + 1) * SLLM_PAGE + kk] = v.y;
      Ks[(4 * d + 2) * SLLM_PAGE + kk] = v.z;
      Ks[(4 * d + 3) * SLLM_PAGE + kk] = v.w;
    }
    for (int e = tid; e < SLLM_PAGE * vq; e += 256) {
      const int kk = e / vq, d = e % vq;
      *(float4*)(Vs + kk * vd + 4 * d) = kk < n_keys ? ld4(vp + (at + kk) * vd + 4 * d) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    __syncthreads();
    float s[QPT][4];
#pragma unroll
    for (int i = 0; i < QPT; i++)
#pragma unroll
      for (int j = 0; j < 4; j++) s[i][j] = 0.f;
#pragma unroll 4
    for (int d = 0; d < hd; d++) {
      float a[QPT];
      if constexpr (QPT == 4) {
        const float4 v = *(const float4*)(Qs + d * BQ + ty * 4);
        a[0] = v.x; a[1] = v.y; a[2] = v.z; a[3] = v.w;
      } else {
        a[0] = Qs[d * BQ + ty];
      }
      const float4 kb = *(const float4*)(Ks + d * SLLM_PAGE + tx * 4);
      const float kv[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
      for (int i = 0; i < QPT; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) s[i][j] = fmaf(a[i], kv[j], s[i][j]);
    }
#pragma unroll
    for (int i = 0; i < QPT; i++) {
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int key = 4 * tx + j;
        float v = s[i][j] * p.scale;
        if (p.softcap > 0.f) v = p.softcap * tanhf(v / p.softcap);
        s[i][j] = key < n_keys && t * SLLM_PAGE + key <= qpos[i] ? v * SHARE_LOG2E : -INFINITY;
        mx = fmaxf(mx, s[i][j]);
      }
#pragma unroll
      for (int off = 1; off < 16; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
      const float m_new = fmaxf(m[i], mx), corr = m_new == -INFINITY ? 1.f : exp2f(m[i] - m_new);
      float pr[4], rs = 0.f;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        pr[j] = s[i][j] == -INFINITY ? 0.f : exp2f(s[i][j] - m_new);
        rs += pr[j];
      }
      l[i] = fmaf(l[i], corr, rs);                                      // this lane's share of the row's sum
      m[i] = m_new;
#pragma unroll
      for (int gg = 0; gg < NG; gg++)
#pragma unroll
        for (int c = 0; c < 4; c++) o[i][gg][c] *= corr;
      *(float4*)(Ps + (ty * QPT + i) * SF_PS + tx * 4) = make_float4(pr[0], pr[1], pr[2], pr[3]);
    }
    __syncthreads();
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
          const float4 v = *(const float4*)(Vs + (k4 + kk) * vd + d0);
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
      *(float4*)(p.part + at * vd + d0) = v;
    }
    if (tx == 0) *(float2*)(ml + 2 * at) = make_float2(m[i], ls);
  }
  __syncthreads();                              // the next item's queries take this one's place
}

template <typename A, int NG>
__global__ void __launch_bounds__(256) share_fma_kernel(ShareArgs p) {
  extern __shared__ __align__(16) float share_sm[];
  pdl_launch_dependents();
  pdl_wait();
  const int i1 = p.first[blockIdx.x + 1];
  for (int i = p.first[blockIdx.x]; i < i1; i++) {
    const ShareItem it = share_item(p, i);
    if (it.n_tok * (p.H / p.G) <= 16) share_fma_item<A, NG, 1>(p, it, share_sm);
    else share_fma_item<A, NG, 4>(p, it, share_sm);
  }
}

// ------------------------------------------------------------------ joining partial results
// A warp for a token and query head: the list's entries are read once for M, then every lane adds four values' sums over them.
struct ShareMergeArgs {
  const float* part;
  long long part_rows;
  const int *list_first, *list;
  void* out;                 // [T, H * vd]
  const float* sink;         // [H] or null
  int T, H, G, vd;
};
template <typename A>
__global__ void __launch_bounds__(128) share_merge_kernel(ShareMergeArgs p) {
  pdl_launch_dependents();
  pdl_wait();
  const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (w >= (long long)p.T * p.H) return;
  const int lane = threadIdx.x & 31, t = (int)(w / p.H), h = (int)(w % p.H), rep = p.H / p.G, g = h / rep, r = h % rep;
  const int i0 = p.list_first[(size_t)t * p.G + g], n = p.list_first[(size_t)t * p.G + g + 1] - i0;
  const float2* ml = (const float2*)(p.part + (size_t)p.part_rows * p.vd);
  const float sink = p.sink ? p.sink[h] * SHARE_LOG2E : -INFINITY;
  float M = -INFINITY;
  for (int i = lane; i < n; i += 32) M = fmaxf(M, ml[p.list[i0 + i] + r].x);
  M = fmaxf(warp_max(M), sink);
  const float M0 = M == -INFINITY ? 0.f : M;                    // (nothing seen: every weight below is 2^-inf = 0)
  float den = 0.f;
  for (int i = lane; i < n; i += 32) {
    const float2 v = ml[p.list[i0 + i] + r];
    den = fmaf(exp2f(v.x - M0), v.y, den);
  }
  den = warp_sum(den);
  if (p.sink) den += exp2f(sink - M0);
  const float inv = den > 0.f || den != den ? 1.0f / den : 0.f;
  for (int d0 = 4 * lane; d0 < p.vd; d0 += 128) {
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = 0; i < n; i++) {
      const size_t at = (size_t)p.list[i0 + i] + r;
      const float m = ml[at].x;
      if (m == -INFINITY) continue;                             // an item none of whose keys this row sees
      const float c = exp2f(m - M0);
      const float4 v = *(const float4*)(p.part + at * p.vd + d0);
      a.x = fmaf(c, v.x, a.x);
      a.y = fmaf(c, v.y, a.y);
      a.z = fmaf(c, v.z, a.z);
      a.w = fmaf(c, v.w, a.w);
    }
    st4((A*)p.out + (size_t)w * p.vd + d0, make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv));
  }
}
