// The merges of key ranges that were walked by several workgroups: O[row] = sum_s w_s O_s[row] / sum_s w_s with
// w_s = exp(LSE_s - max LSE), LSE[row] = max LSE + log(sum_s w_s).  Every order of summation is fixed.
#pragma once
#include "paged_tile.h"

namespace tsr950 {

// A chunk's split walks: a workgroup for 32 rows of one of the tile kernel's blocks (blockIdx.y: which of them), a thread
// for four columns of up to 32 D / 1024 rows, whose loads are all on their way together.
template <class T, int FMT, int DP>
__global__ __launch_bounds__(256) void paged_tile_merge_kernel(const PagedTileParams tp, int block) {
  constexpr int PER_ROW = DP / 4, ITEMS = 32 * PER_ROW / 256;
  __shared__ int odd[32];
  const PagedParams& p = tp.p;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, D = p.c.D;
  int h, b, r0;
  PagedSeq s;
  if (!find_block(tp, blockIdx.x, block, h, b, r0, s)) return;
  int lo, count, share;
  tile_range(tp, s, r0, block, lo, count, share);
  const int ns = count ? (count + share - 1) / share : 0;
  const int rows = s.n * p.ratio.value, first = r0 + 32 * blockIdx.y;
  if (first >= rows) return;
  if (tid < 32) odd[tid] = 0;
  __syncthreads();
  const long total_rows = (long)p.total_q * p.Hq;
  const int d = tid % PER_ROW * 4;
  long at[ITEMS];
  int tok[ITEMS], hq[ITEMS];
  float mx[ITEMS], wsum[ITEMS];
  float4 acc[ITEMS];
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const int row = min(first + j * (256 / PER_ROW) + tid / PER_ROW, rows - 1);
    tok[j] = p.ratio.quotient(row);
    hq[j] = h * p.ratio.value + row - tok[j] * p.ratio.value;
    at[j] = (long)(s.q0 + tok[j]) * p.Hq + hq[j];
    mx[j] = -INFINITY;
    wsum[j] = 0.f;
    acc[j] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  constexpr int PARTS = ITEMS <= 4 ? 4 : 2;                // fetched together
  for (int k0 = 0; k0 < ns; k0 += PARTS) {
    float l[ITEMS][PARTS];
    float4 v[ITEMS][PARTS];
#pragma unroll
    for (int u = 0; u < PARTS; ++u)
#pragma unroll
      for (int j = 0; j < ITEMS; ++j) {
        const long from = min(k0 + u, ns - 1) * total_rows + at[j];
        l[j][u] = k0 + u < ns ? tp.part_lse[from] : -INFINITY;
        if (k0 + u < ns) v[j][u] = *reinterpret_cast<const float4*>(tp.part_o + from * D + (d < D ? d : 0));
        else v[j][u] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
      float top = mx[j];
#pragma unroll
      for (int u = 0; u < PARTS; ++u) top = fmaxf(top, l[j][u]);
      const float ref = top > -INFINITY ? top : 0.f, corr = __expf(mx[j] - ref);
      mx[j] = top;
      wsum[j] *= corr;
      acc[j] = make_float4(acc[j].x * corr, acc[j].y * corr, acc[j].z * corr, acc[j].w * corr);
#pragma unroll
      for (int u = 0; u < PARTS; ++u) {
        const float w = __expf(l[j][u] - ref);
        acc[j].x += w * v[j][u].x; acc[j].y += w * v[j][u].y; acc[j].z += w * v[j][u].z; acc[j].w += w * v[j][u].w;
        wsum[j] += w;
      }
    }
  }
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const int il = j * (256 / PER_ROW) + tid / PER_ROW;
    if (first + il >= rows || d >= D) continue;
    const float inv = wsum[j] == 0.f ? 0.f : 1.0f / wsum[j];
    const float4 o = make_float4(acc[j].x * inv, acc[j].y * inv, acc[j].z * inv, acc[j].w * inv);
    if (!finite4(o) || !(wsum[j] > 0.f)) odd[il] = 1;
    store_o4<T>(p, s.q0 + tok[j], hq[j], d, o);
    if (p.LSE && d == 0) p.LSE[at[j]] = wsum[j] == 0.f ? -INFINITY : mx[j] + __logf(wsum[j]);
  }
  __syncthreads();
  for (int il = wave; il < min(32, rows - first); il += 4) {                // see the kernels' ends
    if (!odd[il]) continue;
    const int t = p.ratio.quotient(first + il);
    paged_row<T, FMT>(p, b, s.q0 + t, t, s.n, s.kv, h * p.ratio.value + first + il - t * p.ratio.value);
  }
}

// The few-rows kernel's shares, where a sequence is cut into more than a few: a workgroup for a row, its
// threads share the partials among 256 / (D / 4) groups, whose sums are added in their order.
template <class T, int FMT>
__global__ __launch_bounds__(256) void paged_few_merge_kernel(const PagedFewParams fp) {
  __shared__ float4 sh_acc[256];
  __shared__ float sh_sum[256], sh_red[4];
  const PagedParams& p = fp.p;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, D = p.c.D;
  const int hq = blockIdx.y;
  const unsigned token = blockIdx.z * gridDim.x + blockIdx.x;
  if (token >= (unsigned)p.total_q) return;
  const int t = (int)token;
  // the row's sequence, where it lies on the axis, and the share
  int total = 0, b = -1, start = 0, places = 0;
  PagedSeq s{0, 0, 0};
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    const PagedSeq mine = b0 + lane < p.B ? paged_seq(p, b0 + lane) : PagedSeq{0, 0, 0};
    const int own = few_places(fp, mine), sum = running_sum(own);
    const unsigned long long past = __ballot(b0 + lane < p.B && mine.q0 + mine.n > t);
    if (past && b < 0) {
      const int first = __builtin_ctzll(past);
      b = b0 + first;
      places = __shfl(own, first, 64);
      start = total + __shfl(sum, first, 64) - places;
      s = PagedSeq{__shfl(mine.q0, first, 64), __shfl(mine.n, first, 64), __shfl(mine.kv, first, 64)};
    }
    total += __shfl(sum, 63, 64);
  }
  const int i = t - s.q0;
  if (b < 0 || places == 0 || i < 0) return;
  const int share = max((total + fp.groups - 1) / fp.groups, 1);
  int w0, w1;
  few_shares(fp, start, places, share, w0, w1);
  if (w0 == w1) return;                                    // it was written whole
  const int h = p.ratio.quotient(hq), in_group = i * p.ratio.value + hq - h * p.ratio.value, ns = w1 - w0 + 1;
  auto at = [&](int k) { return few_partial(fp, w0 + k, h, start, share) + in_group; };
  float mx = -INFINITY;
  for (int k = tid; k < ns; k += 256) mx = fmaxf(mx, fp.part_lse[at(k)]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
  if (lane == 0) sh_red[wave] = mx;
  __syncthreads();
  mx = fmaxf(fmaxf(sh_red[0], sh_red[1]), fmaxf(sh_red[2], sh_red[3]));
  const float ref = mx > -INFINITY ? mx : 0.f;
  const int per_row = D / 4, G = 256 / per_row, gr = tid / per_row, c = tid - gr * per_row;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float wsum = 0.f;
  if (gr < G) {
    for (int k0 = gr; k0 < ns; k0 += 4 * G) {
      float l[4];
      float4 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int k = k0 + u * G;
        const long from = at(min(k, ns - 1));
        l[u] = k < ns ? fp.part_lse[from] : -INFINITY;
        v[u] = *reinterpret_cast<const float4*>(fp.part_o + from * D + 4 * c);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float w = __expf(l[u] - ref);
        if (k0 + u * G >= ns) continue;
        acc.x += w * v[u].x; acc.y += w * v[u].y; acc.z += w * v[u].z; acc.w += w * v[u].w;
        wsum += w;
      }
    }
  }
  sh_acc[tid] = acc;
  sh_sum[tid] = wsum;
  __syncthreads();
  if (wave != 0) return;                                   // (per_row <= 64: the first wave has the row's columns)
  for (int g = 1; g < G && lane < per_row; ++g) {
    const float4 v = sh_acc[g * per_row + lane];
    acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
    wsum += sh_sum[g * per_row + lane];
  }
  const float inv = wsum == 0.f ? 0.f : 1.0f / wsum;
  acc.x *= inv; acc.y *= inv; acc.z *= inv; acc.w *= inv;
  if (__any(lane < per_row && (!finite4(acc) || !(wsum > 0.f)))) {
    paged_row<T, FMT>(p, b, t, i, s.n, s.kv, hq);
    return;
  }
  if (lane < per_row) store_o4<T>(p, t, hq, 4 * lane, acc);
  if (p.LSE && lane == 0) p.LSE[(long)t * p.Hq + hq] = wsum == 0.f ? -INFINITY : mx + __logf(wsum);
}

}  // namespace tsr950
