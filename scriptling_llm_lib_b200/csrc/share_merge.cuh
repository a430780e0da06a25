// Joining the partial results of an attention over shared pages (share_kernels.cuh has the mathematics), float32 sums to either element
// type.
#pragma once
#include "share_plan.cuh"

// A warp for a token and RB query heads that stand side by side in the scratch (a power of two that divides the heads of a key/value
// head, so that their 16-byte pieces fill whole sectors). Lane j RB + r has head r of them: first entry base + j of the list (row of the
// scratch, m, l), then the dims 4 (j + k 32 / RB) .. + 3 of the sum, of which NQ fit. Loads of two entries are under way at once (with four
// fewer warps fit an SM: prompt steps of 700 rows 2 to 6% slower), of four with SPLIT. Bound by the chain of its loads (which entries,
// their m and l beside the sums): 4 to 8 us where outputs are few, about 20 for 146,688 rows of 128 (75 MB).
struct ShareMergeArgs {
  const float* part;
  long long part_rows;
  const int *list_first, *list;
  void* out;                 // [T, H * vd]
  const float* sink;         // [H] or null
  int T, H, G, vd;
};
// With SPLIT the eight warps of a block share an output's entries and meet in shared memory: where outputs are few, the chain of an output's
// loads (a microsecond for every four entries) is what the kernel lasts.
#define SHARE_MERGE_WARPS 8
template <typename A, int RB, int NQ, bool SPLIT>
__global__ void __launch_bounds__(32 * SHARE_MERGE_WARPS, SPLIT ? 2 : 3) share_merge_kernel(ShareMergeArgs p) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int J = 32 / RB, W = SHARE_MERGE_WARPS, MET = SPLIT ? W : 1;      // J: entries that a warp holds at a time
  constexpr int E = SPLIT ? 4 : 2;                                           // of which so many are under way at once
  __shared__ float4 met[MET][NQ][32];
  __shared__ float2 met_ml[MET][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, per = p.H / RB;
  const long long w = SPLIT ? (long long)blockIdx.x : (long long)blockIdx.x * W + warp;
  if (w >= (long long)p.T * per) return;
  const int j = lane / RB, t = (int)(w / per), h = (int)(w % per) * RB + lane % RB, rep = p.H / p.G, g = h / rep, r = h % rep;
  const int i0 = p.list_first[(size_t)t * p.G + g], n = p.list_first[(size_t)t * p.G + g + 1] - i0;
  // lane (j, .) holds entry base + j * apart: the warps of an output take its entries in turn
  constexpr int apart = SPLIT ? W : 1, step = apart * J;
  const int first = SPLIT ? warp : 0;
  const float2* ml = (const float2*)(p.part + (size_t)p.part_rows * p.vd);
  // ---- the largest score of this warp's entries; the first of them stay at hand
  int at = first + j * apart < n ? p.list[i0 + first + j * apart] + r : 0;
  float2 v = first + j * apart < n ? ml[at] : make_float2(-INFINITY, 0.f);
  // the first entries' sums, on their way beside the (m, l) that weigh them: what a row does not see is loaded and left out
  float4 x[E][NQ];
  auto load = [&](int e0, int m) {
#pragma unroll
    for (int e = 0; e < E; e++) {
      const size_t row = __shfl_sync(0xffffffffu, at, ((e0 + e) * RB + lane % RB) & 31);
#pragma unroll
      for (int k = 0; k < NQ; k++) {
        const int d = 4 * (j + k * J);
        if (e0 + e < m && d < p.vd) x[e][k] = *(const float4*)(p.part + share_at(row, d, p.vd));
        else x[e][k] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
  };
  auto held = [&](int base) { return min(J, (n - base + apart - 1) / apart); };
  load(0, held(first));
  float M = v.x;
#pragma unroll 4
  for (int i = first + step + j * apart; i < n; i += step) M = fmaxf(M, ml[p.list[i0 + i] + r].x);
#pragma unroll
  for (int d = RB; d < 32; d <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
  const float M0 = M == -INFINITY ? 0.f : M;                    // (nothing seen: every weight below is 2^-inf = 0)
  float den = 0.f;
  float4 a[NQ];
#pragma unroll
  for (int k = 0; k < NQ; k++) a[k] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int base = first; base < n; base += step) {
    if (base != first) {
      at = base + j * apart < n ? p.list[i0 + base + j * apart] + r : 0;
      v = base + j * apart < n ? ml[at] : make_float2(-INFINITY, 0.f);
    }
    // an entry none of whose keys this row sees, or none at all, weighs 0 and its values are left out; a sum that is NaN spoils the row
    const float wgt = v.y != v.y ? v.y : exp2f(v.x - M0);
    if (wgt != 0.f) den = fmaf(wgt, v.y, den);
    const int m = held(base);
    for (int e0 = 0; e0 < m; e0 += E) {
      if (base != first || e0 > 0) load(e0, m);
#pragma unroll
      for (int e = 0; e < E; e++) {
        const float c = __shfl_sync(0xffffffffu, wgt, ((e0 + e) * RB + lane % RB) & 31);
        if (e0 + e < m && c != 0.f) {
#pragma unroll
          for (int k = 0; k < NQ; k++) {
            a[k].x = fmaf(c, x[e][k].x, a[k].x);
            a[k].y = fmaf(c, x[e][k].y, a[k].y);
            a[k].z = fmaf(c, x[e][k].z, a[k].z);
            a[k].w = fmaf(c, x[e][k].w, a[k].w);
          }
        }
      }
    }
  }
#pragma unroll
  for (int d = RB; d < 32; d <<= 1) den += __shfl_xor_sync(0xffffffffu, den, d);
  // ---- the warps' sums, and the sink's share
  const float sink = p.sink ? p.sink[h] * SHARE_LOG2E : -INFINITY;
  float top = fmaxf(M, sink);
  if constexpr (SPLIT) {
    met_ml[warp][lane] = make_float2(M, den);
#pragma unroll
    for (int k = 0; k < NQ; k++) met[warp][k][lane] = a[k];
    __syncthreads();
    if (warp >= NQ) return;                         // warp k adds the dims that the lanes hold under k
#pragma unroll
    for (int o = 0; o < W; o++) top = fmaxf(top, met_ml[o][lane].x);
  }
  const float top0 = top == -INFINITY ? 0.f : top;
  float all = p.sink ? exp2f(sink - top0) : 0.f;
  A* out = (A*)p.out + ((size_t)t * p.H + h) * p.vd;
  if constexpr (SPLIT) {
    float4 b = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int o = 0; o < W; o++) {
      const float2 e = met_ml[o][lane];
      const float c = e.x == -INFINITY && e.y == 0.f ? 0.f : exp2f((e.x == -INFINITY ? 0.f : e.x) - top0);
      const float4 x = met[o][warp][lane];
      all = fmaf(c, e.y, all);
      b.x = fmaf(c, x.x, b.x);
      b.y = fmaf(c, x.y, b.y);
      b.z = fmaf(c, x.z, b.z);
      b.w = fmaf(c, x.w, b.w);
    }
    const float inv = all > 0.f || all != all ? 1.0f / all : 0.f;
    const int d = 4 * (j + warp * J);
    if (d < p.vd) st4(out + d, make_float4(b.x * inv, b.y * inv, b.z * inv, b.w * inv));
  } else {
    const float c = M == -INFINITY ? 0.f : exp2f(M0 - top0);      // (nothing seen: 2^-sink may be infinite, and times 0 is NaN)
    all = fmaf(c, den, all);
    const float inv = all > 0.f || all != all ? c / all : 0.f;
#pragma unroll
    for (int k = 0; k < NQ; k++) {
      const int d = 4 * (j + k * J);
      if (d < p.vd) st4(out + d, make_float4(a[k].x * inv, a[k].y * inv, a[k].z * inv, a[k].w * inv));
    }
  }
}

template <typename A, int RB, int NQ>
static int share_merge_launch(const ShareMergeArgs& a, cudaStream_t stream) {
  // a block an output while those are no more than 16 an SM, else a warp
  const long long n = (long long)a.T * (a.H / RB);
  const dim3 block(32 * SHARE_MERGE_WARPS);
  // Launched the ordinary way, when the kernel in front is done on every SM. That kernel leaves the SMs with nearly all of their memory as
  // shared memory, and where each kernel starts before the one in front has ended no SM is ever idle and it stays so: the decode step's
  // products, which read their few rows through L1, then take twice as long (8 sequences behind 4,096 tokens, 32 layers of width 4,096: 6.4
  // ms a step, 3.8 this way; 4.0 each for itself).
  if (n <= 16LL * sllm_sm_count()) share_merge_kernel<A, RB, NQ, true><<<(unsigned)n, block, 0, stream>>>(a);
  else share_merge_kernel<A, RB, NQ, false><<<(unsigned)((n + SHARE_MERGE_WARPS - 1) / SHARE_MERGE_WARPS), block, 0, stream>>>(a);
  SLLM_RETURN_LAST();
}
template <typename A>
static int share_merge_run(const SharePlanDev& plan, const float* part, void* out, const float* sink, int vd, cudaStream_t stream) {
  const ShareMergeArgs a{part, plan.part_rows, plan.list_first, plan.list, out, sink, plan.T, plan.H, plan.G, vd};
  const int rep = plan.H / plan.G, rb = rep % 8 == 0 && vd <= 64 ? 8 : rep % 4 == 0 && vd <= 128 ? 4 : rep % 2 == 0 ? 2 : 1;
  switch (rb) {
    case 8: return share_merge_launch<A, 8, 4>(a, stream);
    case 4: return share_merge_launch<A, 4, 4>(a, stream);
    case 2: return vd <= 128 ? share_merge_launch<A, 2, 2>(a, stream) : share_merge_launch<A, 2, 4>(a, stream);
    default: return vd <= 128 ? share_merge_launch<A, 1, 1>(a, stream) : share_merge_launch<A, 1, 2>(a, stream);
  }
}
