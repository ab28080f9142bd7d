// Host side of the paged attention kernels, instantiated once for each storage type and cache format.
#pragma once
#include <algorithm>
#include <cstdint>
#include <mutex>
#include "host_util.h"
#include "paged_merge.h"

namespace tsr950 {

// Query rows a KV head that the few-rows kernel serves: one, two or four MFMA tiles, what the registers hold of their
// accumulators.
inline int paged_few_limit(int D) { return D <= 64 ? 128 : D <= 128 ? 64 : 32; }

// A key range that no sequence's visible keys exceed, for `tokens` neighbouring tokens.
inline int paged_span(const PagedParams& p, int tokens) {
  if (p.window <= 0) return p.max_kv;
  const int64_t span = (int64_t)(p.causal ? p.window : p.window / 2 * 2 + 1) + tokens - 1;
  return (int)std::min<int64_t>(span, p.max_kv);
}
// Tiles of `keys` keys that it touches at most.
inline int paged_tiles(const PagedParams& p, int tokens, int keys) {
  const int span = paged_span(p, tokens);
  return std::min(ceil_div(p.max_kv, keys), span > 0 ? (span - 1) / keys + 2 : 0);
}

inline int lds_limit(const void* kern, int bytes) {
  return finish(hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
}

// How one call's work is divided.
struct PagedPlan {
  bool few = false, tile = false;
  int few_rows = 0;
  int waves = 8, block = 0, blocks = 0, tile_split = 1;
};

// The kernel for a number of rows, its dynamic LDS and how many of its workgroups a compute unit holds.
struct FewKernel {
  void (*run)(const PagedFewParams);
  int threads, lds, per_cu;
};
template <class T, int FMT, int DP, int NQ, bool FAR>
FewKernel few_kernel_as() {
  using G = FewGeom<FMT, DP>;
  static std::once_flag once;
  static int per_cu = 0;
  std::call_once(once, [] {
    const void* kern = reinterpret_cast<const void*>(paged_few_kernel<T, FMT, DP, NQ, FAR>);
    if (lds_limit(kern, G::SMEM) != kOk || hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, kern, G::THREADS, G::SMEM) != hipSuccess)
      per_cu = 0;
  });
  return FewKernel{paged_few_kernel<T, FMT, DP, NQ, FAR>, G::THREADS, G::SMEM, per_cu};
}
template <class T, int FMT, int DP, int NQ>
FewKernel few_kernel(const PagedParams& p) {
  return p.softcap > kPlainCap ? few_kernel_as<T, FMT, DP, NQ, true>() : few_kernel_as<T, FMT, DP, NQ, false>();
}
template <class T, int FMT>
FewKernel few_kernel_for(const PagedParams& p, int rows) {
  const int D = p.c.D;
  if (D <= 64) return rows <= 32 ? few_kernel<T, FMT, 64, 1>(p) : rows <= 64 ? few_kernel<T, FMT, 64, 2>(p) : few_kernel<T, FMT, 64, 4>(p);
  if (D <= 128) return rows <= 32 ? few_kernel<T, FMT, 128, 1>(p) : few_kernel<T, FMT, 128, 2>(p);
  return few_kernel<T, FMT, 256, 1>(p);
}

template <class T, int FMT, int DP, int W, int EXT>
int launch_tile_as(const PagedTileParams& tp, int blocks, hipStream_t s) {
  constexpr int SMEM = TileGeom<DP, W>::SMEM(FMT != kStorage);
  auto kern = paged_tile_kernel<T, FMT, DP, W, EXT>;
  static std::once_flag once;
  static int attr = kOk;
  std::call_once(once, [&] { attr = lds_limit(reinterpret_cast<const void*>(kern), SMEM); });
  if (attr != kOk) return attr;
  hipLaunchKernelGGL(kern, dim3((unsigned)tp.p.c.heads * (unsigned)blocks, (unsigned)tp.nsplit), dim3(TileGeom<DP, W>::THREADS), SMEM, s, tp);
  return launch_status();
}
template <class T, int FMT, int DP, int W>
int launch_tile(const PagedTileParams& tp, int blocks, hipStream_t s) {
  if (folds(tp.p)) return launch_tile_as<T, FMT, DP, W, 0>(tp, blocks, s);
  return tp.p.softcap > kPlainCap ? launch_tile_as<T, FMT, DP, W, 2>(tp, blocks, s) : launch_tile_as<T, FMT, DP, W, 1>(tp, blocks, s);
}
template <class T, int FMT>
int launch_tile_for(const PagedTileParams& tp, const PagedPlan& plan, hipStream_t s) {
  if (tp.p.c.D <= 64) return plan.waves == 4 ? launch_tile<T, FMT, 64, 4>(tp, plan.blocks, s) : launch_tile<T, FMT, 64, 8>(tp, plan.blocks, s);
  if (tp.p.c.D <= 128) return plan.waves == 4 ? launch_tile<T, FMT, 128, 4>(tp, plan.blocks, s) : launch_tile<T, FMT, 128, 8>(tp, plan.blocks, s);
  return launch_tile<T, FMT, 256, 4>(tp, plan.blocks, s);
}

constexpr int kTileSplits = 32;

// Workgroup size (8 waves: 256 rows, 4: 128; at DP = 256 always 4) and key splits of the tile kernel: the least estimated
// time in us over both and up to 32 splits.  What it weighs, with times at D 128, Hq 32, Hkv 8, causal, bf16 pages:
// - a workgroup costs 7 (4 waves: 6) and 1.6 to 2.05 a 64-key tile, the more of the chip works the more; 4 waves 1.45 to 1.65, and
//   2.3 with a second workgroup on the compute unit (not at DP = 256): 512 tokens on 512 keys 21.7 in 8 waves, 18.4 in 4; 2048 on
//   2048, two sequences, 85 and 92;
// - splits leave partials (of at most `room` rows) and a merge, 4 us and the bytes: 1024 tokens on 8192 keys 220 unsplit, 153 in two, 183 in three
//   (a second turn of workgroups); 100 on 16384 342 to 414, 52 as planned; but 512 on 512 18.4, 22.3 in two.
// - codes 1.2 times as long in both forms (4 waves, 512 tokens on 512 keys: 18.7 over 16 bits, e4m3 22.4, int8 23.2; f16 programs 24.8 and 26.1).
// Returns the estimate.
inline double plan_tiles(const PagedParams& p, bool codes, double chunks, int64_t room, PagedPlan& plan) {
  const int D = p.c.D, ratio = p.ratio.value, H = p.c.heads;
  const int64_t max_rows = (int64_t)p.max_q * ratio, all_rows = (int64_t)p.total_q * ratio;
  const double width = (D <= 64 ? 0.63 : D <= 128 ? 1.0 : 2.2) * (codes ? 1.2 : 1.0);
  const double merge_bytes = (plan.few ? chunks * max_rows : (double)all_rows) * H * D * 4.0;
  const int longest = paged_tiles(p, std::min(256 / ratio + 1, p.max_q), FA_BKV);
  // (a causal walk ends at its block: on the average half of the new tokens before the end)
  const double mean = std::max(1.0, p.causal && p.window <= 0 ? longest - p.max_q / 2.0 / FA_BKV : longest);
  double best = 1e30;
  for (int waves : {4, 8}) {
    if (D > 128 && waves == 8) continue;
    const int block = 32 * waves;
    const int64_t most = std::min<int64_t>(p.B * ((max_rows + block - 1) / block), all_rows / block + p.B);
    // (chunks of one length, and single tokens where no other kernel has them)
    const double blocks = std::min<double>((double)most, chunks * std::ceil((double)max_rows / block) + (plan.few ? 0.0 : p.B - chunks));
    for (int n = 1; n <= kTileSplits && (n == 1 || (n <= longest / 2 && n * (int64_t)p.total_q * p.Hq <= room)); ++n) {
      const double wgs = blocks * H * n;
      const double load = std::min(1.0, wgs / 256);
      double t;
      if (waves == 8 || D > 128 || wgs <= 256) {
        const double step = (waves == 8 ? 1.6 + 0.45 * load : 1.45 + 0.2 * load) * width, ends = waves == 8 ? 7 : 6;
        t = wgs <= 256 ? ends + step * std::ceil((double)longest / n) : std::ceil(wgs / 256) * (ends + step * std::ceil(mean / n));
      } else {
        const double step = 2.3 * width;
        t = wgs <= 512 ? 6 + step * std::ceil((double)longest / n) : std::ceil(wgs / 512) * (6 + step * std::ceil(mean / n));
      }
      if (n > 1) t += 4 + merge_bytes * (2 * n + 1) / 4.5e6;
      if (t < best) {
        best = t;
        plan.waves = waves;
        plan.block = block;
        plan.blocks = (int)most;
        plan.tile_split = n;
      }
    }
  }
  return best;
}

inline PagedPlan paged_plan(const PagedParams& p, bool codes, int64_t room) {
  PagedPlan plan;
  const int D = p.c.D, ratio = p.ratio.value, limit = paged_few_limit(D);
  const int64_t max_rows = (int64_t)p.max_q * ratio;
  plan.tile = max_rows > limit;
  if (!plan.tile) {
    plan.few_rows = (int)max_rows;
    plan.few = true;
    return plan;
  }
  // Sequences that are chunks, as far as the host can tell: of the longest length, the others of one token.
  const double chunks = std::min<double>(p.B, std::max(1.0, std::ceil((double)(p.total_q - p.B) / std::max(p.max_q - 1, 1))));
  PagedPlan both = plan;
  const double all = plan_tiles(p, codes, chunks, room, plan);
  // Single tokens beside chunks: the few-rows kernel takes the sequences with up to a tile's rows (or a token's, where the
  // group is larger), where its launch (10 us) and its reads cost less than such sequences among the tiles: 31 of 3000 to
  // 6000 keys beside a chunk of 500 tokens, e4m3, yes; 4 of 464 keys beside one of 202, no.
  const int single = ratio <= 32 ? 32 : ratio <= 64 ? 64 : 128;
  if (single <= limit && p.total_q < (int64_t)p.B * p.max_q && p.total_q < (1 << 23)) {
    both.few = true;
    both.few_rows = single;
    const double reads = 2.0 * (p.B - chunks) * p.c.heads * paged_span(p, 1) * D * (codes ? 1 : 2);
    if (plan_tiles(p, codes, chunks, room, both) + 10 + reads / 5e6 < all) return both;
  }
  return plan;
}

// Rows of partials that no call needs more of whose arguments are no larger: every eager call makes room for them, so that
// a capture behind it finds what the recorded call needs, whichever plan that one has.  Few rows: as many groups as the LDS lets
// a compute unit hold, of the most rows (plan_few).  Split walks: 2^17 rows (68 MB at D 128; 512 tokens of 32 heads in eight parts);
// where a recorded call's plan has more of them than there is room for, it is made again with fewer splits.
template <int FMT>
size_t few_reserve(const PagedParams& p) {
  const int D = p.c.D, smem = D <= 64 ? FewGeom<FMT, 64>::SMEM : D <= 128 ? FewGeom<FMT, 128>::SMEM : FewGeom<FMT, 256>::SMEM;
  const int waves = D <= 64 ? FewGeom<FMT, 64>::WAVES : D <= 128 ? FewGeom<FMT, 128>::WAVES : FewGeom<FMT, 256>::WAVES;
  const int64_t tiles = (int64_t)p.B * ceil_div(p.max_kv, 32), groups = std::max<int64_t>(p.B, tiles / (2 * waves));
  const int64_t rows = std::min<int64_t>(paged_few_limit(D), (int64_t)p.max_q * p.ratio.value);
  return (size_t)(std::min<int64_t>(256 * (160 * 1024 / smem), groups * p.c.heads) * 2 * rows);
}
inline size_t tile_reserve(const PagedParams& p) {
  if ((int64_t)p.max_q * p.ratio.value <= paged_few_limit(p.c.D)) return 0;
  return (size_t)std::min<int64_t>((int64_t)kTileSplits * p.total_q * p.Hq, 1 << 17);
}

// The few-rows part of a plan: its kernel and how the axis is cut.
template <class T, int FMT>
bool plan_few(const PagedPlan& plan, PagedFewParams& fp, FewKernel& few) {
  const PagedParams& p = fp.p;
  few = few_kernel_for<T, FMT>(p, plan.few_rows);
  if (few.per_cu <= 0) return false;
  // As many equal shares as the chip holds workgroups for every head, at least one for a sequence and two tiles
  // for a wave.  Starting a sequence costs about two steps of a workgroup.
  const int waves = few.threads / 64;
  const int64_t tiles = (int64_t)p.B * paged_tiles(p, plan.tile ? ceil_div(plan.few_rows, p.ratio.value) : p.max_q, 32);
  fp.rows = plan.few_rows;
  fp.ahead = p.B > 1 ? 2 * waves : 0;
  fp.groups = (int)std::max<int64_t>(1, std::min<int64_t>(256 * few.per_cu / p.c.heads, std::max<int64_t>(p.B, tiles / (2 * waves))));
  // Nothing is cut where a sequence takes two steps, or eight where the workgroups fill half of the chip anyway.
  const int64_t each = tiles / p.B;
  if (each <= 2 * waves || (each <= 8 * waves && (int64_t)p.B * p.c.heads >= 128 * few.per_cu)) fp.groups = 0;
  // (the rule of the contiguous decode kernel, common.h)
  fp.once = 64.0 * tiles * p.c.heads * p.c.D * (FMT == kStorage ? 2 : 1) >= kStreamOnceBytes;
  return true;
}

template <class T, int FMT>
int launch_paged(const PagedParams& p, hipStream_t s) {
  const size_t D = (size_t)p.c.D, row_bytes = (D + 1) * sizeof(float);
  PagedFewParams fp{};
  PagedTileParams tp{};
  fp.p = p;
  tp.p = p;
  FewKernel few{};
  PagedPlan plan;
  size_t fr = 0, tr = 0;                                   // rows of partials
  auto make_plan = [&](int64_t room) {
    plan = paged_plan(p, FMT != kStorage, room);
    fp.groups = 0;
    if (plan.few && !plan_few<T, FMT>(plan, fp, few)) return false;
    fr = fp.groups > 1 ? (size_t)fp.groups * p.c.heads * 2 * fp.rows : 0;
    tr = plan.tile && plan.tile_split > 1 ? (size_t)plan.tile_split * p.total_q * p.Hq : 0;
    return true;
  };
  if (!make_plan(INT64_MAX)) return kDeviceFailed;
  const size_t most = few_reserve<FMT>(p) + tile_reserve(p);
  const size_t there = stream_reserve(s, (fr + tr) * row_bytes, std::max(fr + tr, most) * row_bytes, (size_t)p.B * p.c.heads) / row_bytes;
  if (tr && fr + tr > there && !make_plan((int64_t)there - (int64_t)few_reserve<FMT>(p))) return kDeviceFailed;
  tp.nsplit = plan.tile_split;
  tp.min_rows = plan.few_rows;
  const bool few_cut = fp.groups > 1, tile_cut = plan.tile && plan.tile_split > 1;
  // A sequence's partials are merged by the last of its workgroups, or by a kernel of their own: more than 16 of them, or
  // more than two passes of a workgroup's threads of a few sequences.
  const bool few_kernel_merges = few_cut && (fp.groups > 16 * p.B || (p.B <= 16 && fp.rows * p.c.D / 4 > 2 * few.threads));
  if (few_cut || tile_cut) {
    float* ws = static_cast<float*>(stream_workspace(s, (fr + tr) * row_bytes));
    if (!ws) return kDeviceFailed;
    fp.part_o = ws;
    tp.part_o = ws + fr * D;
    fp.part_lse = ws + (fr + tr) * D;
    tp.part_lse = fp.part_lse + fr;
    if (few_cut && !few_kernel_merges) {
      fp.arrived = stream_counters(s, (size_t)p.B * p.c.heads);
      if (!fp.arrived) return kDeviceFailed;
    }
  }
  if (plan.tile)
    if (int rc = launch_tile_for<T, FMT>(tp, plan, s); rc != kOk) return rc;
  if (plan.few) {
    hipLaunchKernelGGL(few.run, dim3((unsigned)((fp.groups ? fp.groups : p.B) * p.c.heads)), dim3(few.threads), few.lds, s, fp);
    if (int rc = launch_status(); rc != kOk) return rc;
  }
  if (few_kernel_merges) {
    // (a dimension's threads are a 32-bit number; what is beyond it wraps, without an error)
    const unsigned tokens = (unsigned)p.total_q, along = std::min(tokens, 1u << 23);
    hipLaunchKernelGGL((paged_few_merge_kernel<T, FMT>), dim3(along, (unsigned)p.Hq, (tokens + along - 1) / along), dim3(256), 0, s, fp);
    if (int rc = launch_status(); rc != kOk) return rc;
  }
  if (!tile_cut) return kOk;
  const dim3 grid((unsigned)(plan.blocks * p.c.heads), (unsigned)(plan.block / 32));
  auto merge = D <= 64 ? paged_tile_merge_kernel<T, FMT, 64> : D <= 128 ? paged_tile_merge_kernel<T, FMT, 128> : paged_tile_merge_kernel<T, FMT, 256>;
  hipLaunchKernelGGL(merge, grid, dim3(256), 0, s, tp, plan.block);
  return launch_status();
}

}  // namespace tsr950
