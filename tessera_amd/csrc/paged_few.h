// Attention over a paged cache for sequences with few new tokens (decode, speculative steps).
//
// The rows of a whole group of query heads, (Hq / heads) x n of them, at most 32 NQ, are the columns of NQ MFMA tiles that
// share every K and V fragment, so a sequence's K and V are read once for each KV head: that read bounds the kernel.  The
// products are the transposed ones of the contiguous kernels (flash_attn.h): S^T = K Q^T, O^T += V^T P^T, a lane's scores
// all belong to query row lane % 32, P goes from the score registers straight into the second product.
//
// Work: the 32-key tiles of all sequences lie one after another on an axis (with some empty places ahead of each sequence for
// what starting one costs), which is cut into `groups` equal shares; workgroup (g, h) walks share g for KV head h.  Shares
// are equal however the lengths differ, and the heads of a share run side by side on one XCD, which fetches a line of scales
// of several heads once.  A sequence inside one share is finished there; one that is cut leaves normalised partials, which
// are merged in the order of the shares: few of them by the workgroup that leaves the last one, many by a kernel with a
// workgroup for a row.  Inside a workgroup wave w takes the tiles w, w + WAVES, ... of a sequence's part.  Tiles go from
// memory straight into a wave-private LDS region, two stages, no workgroup
// barrier in the loop.  What paging adds: a lane finds its row's page from the key's number (a multiplication for the
// division by the page size, any size), the page's number from the sequence's table, whose entries for a tile are themselves
// loaded into LDS one tile ahead of the rows, so that nothing waits for them; and rows past the last key repeat the last
// key's row, so that neither an unset table entry nor an unwritten slot is ever touched.  8-bit codes stay codes in LDS and
// become 16-bit values in registers, between the LDS read and the product; K's scales multiply the scores, V's join the
// exponents (weight_scale), in f32.
//
// Measured (Hq 32, Hkv 8, D 128): 64 sequences of 2048 to 4096 keys, 802 MB, 136 us = 5.9 TB/s; 128 of 4096 to 8192, e4m3, 1651
// MB, 301 us = 5.5 TB/s; four tokens on 131072 int8 keys, f16, 277 MB, 65 us (with the merge, 5) = 4.3 TB/s; one token on 1000 keys
// 10.9 us, of which 4 MB take one: what is left is a chain of some ten waits for memory (lengths, page, row, partials, merge).
#pragma once
#include "paged_attn.h"

namespace tsr950 {

// 16 (4) bytes per lane from a global address of its own into LDS at lds_base + 16 (4) lane.  NT: the non-temporal hint.
template <bool NT = false>
__device__ __forceinline__ void gather16_to_lds(const void* from, uint32_t lds_base) {
  if constexpr (NT)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off nt" :: "s"(lds_base), "v"(from) : "memory");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" :: "s"(lds_base), "v"(from) : "memory");
}
__device__ __forceinline__ void gather4_to_lds(const void* from, uint32_t lds_base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" :: "s"(lds_base), "v"(from) : "memory");
}
template <int N> __device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" :: "n"(N) : "memory"); }

// Where the 16-byte chunks of a K or V row lie in LDS: physical chunk = logical ^ swizzle(row), rows unpadded.  K is read by
// 32 consecutive rows, one chunk each: rows that start in the same bank (256 / row bytes apart) take different chunks.  V is
// read transposed: 16-bit, four rows of 64 bytes; 8-bit, rows {0..3, 8..11} (+4) of 32 bytes.
template <int ROWB> __device__ __forceinline__ int k_swizzle(int row) {
  return ROWB >= 256 ? row & 15 : ROWB == 128 ? (row >> 1) & 7 : (row >> 2) & 3;
}
template <int ROWB, bool CODES> __device__ __forceinline__ int v_swizzle(int row) {
  if constexpr (!CODES) return ROWB >= 256 ? (row & 3) << 2 : ((row >> 1) & 1) << 2;
  else if constexpr (ROWB >= 256) return ((row & 3) | ((row >> 3) & 1) << 2) << 1;
  else if constexpr (ROWB == 128) return (((row >> 1) & 1) | ((row >> 3) & 1) << 1) << 1;
  else return ((row >> 3) & 1) << 1;
}

// Weights of a second product in f16 (TV) are formed 2^14 over their share of the largest, which the sum and the result's quotient
// carry alike: f16 keeps 11 bits down to 2^-28 of the largest weight and something down to 2^-39, where weights of at most 1 lose
// bits from 2^-14 and become nothing at 2^-25.  (4999 keys 17.4 under one other hold 1.4e-4 of the probability, and all of the result in
// columns where that one's value is zero; it came out as nothing there.)
template <class TV> constexpr float weight_lift() { return std::is_same<TV, F16>::value ? 14.0f : 0.f; }

// With codes the second product is in f16, in which they are exact, over the weights w = p vs (vs: V's scale of the key).  They are
// formed as 2^(x + log2 vs - m + 14), x the score's exponent and m the running maximum of x + log2 vs, so that w has f16's range and
// 11 bits whatever the scales; the softmax's sum is that of w / vs, under the same m.  log2 vs and 1 / vs are formed once a key.
// Error of the f32 result, 4000 keys, bf16 and f16 programs: 1.6e-4 (a product in bf16: 1.7e-3, and 4 to 8 % less time where
// LDS waits show: 8 sequences of 1000 int8 keys 15.8 us, 15.2 so; at large batches level).  A scale under 1e-25 counts as
// 1e-25: its row is nothing either way, the key's probability has to come back from w / vs, and 2^30 such keys' sum stays finite.
__device__ __forceinline__ float weight_scale(float vs) { return fmaxf(vs, 1e-25f) + vs * 0.f; }      // (not finite: stays so)

template <int FMT, int DP> struct FewGeom {
  static constexpr int ESZ = FMT == kStorage ? 2 : 1;
  static constexpr int ROWB = DP * ESZ, CHUNKS = ROWB / 16;
  static constexpr int BK = 32, TILE = BK * ROWB;
  static constexpr int WAVES = ROWB >= 256 ? 2 : 4, THREADS = WAVES * 64;  // (two workgroups to a compute unit)
  static constexpr int LD = BK * CHUNKS / 64;                          // load instructions of one K (or V) tile
  static constexpr int PITCH = DP * 4 + 16;                            // a row of a wave's f32 partial O
  static constexpr int BODY = 4 * TILE > 32 * PITCH ? 4 * TILE : 32 * PITCH;
  static constexpr int TABLE_AT = BODY;                                // two stages of 32 page numbers
  static constexpr int ROWS_AT = TABLE_AT + 256;                       // 32 K row offsets, 32 of V
  static constexpr int SCALE_AT = ROWS_AT + 512;                       // two stages of 32 K and 32 V scales
  static constexpr int INVERSE_AT = SCALE_AT + 512;                    // 1 / V's scales of the tile at hand
  static constexpr int WAVE_LDS = SCALE_AT + (FMT == kStorage ? 0 : 640);
  static constexpr int ML_AT = WAVES * WAVE_LDS;                       // the waves' (max, sum), the merged ones, flags
  static constexpr int SMEM = ML_AT + (2 * WAVES + 3) * 128 + 16;
};

struct PagedFewParams {
  PagedParams p;
  float* part_o;          // [groups * heads][2][rows][D] normalised partial O
  float* part_lse;        // [groups * heads][2][rows]
  int* arrived;           // [B * heads] zero before and after: how many partials of a sequence are there; null: another kernel merges
  int groups;             // shares; 0: a sequence for each workgroup of a head, nothing is cut
  int rows;               // (of the sequences served; those with more rows a KV head are another kernel's)
  int ahead;              // empty places ahead of a sequence
  int once;               // K and V are too large to be found in the caches again
};

// The 32-key tiles [lo, end) that a sequence's rows see between them.
__device__ __forceinline__ void few_tiles(const PagedParams& p, const PagedSeq& s, int& lo, int& end) {
  int lo0, hi0, lo1, hi1;
  key_bounds(0, s.n, s.kv, p.causal, p.window, lo0, hi0);
  key_bounds(s.n - 1, s.n, s.kv, p.causal, p.window, lo1, hi1);
  lo = lo0 / 32;
  end = hi1 >= lo0 ? hi1 / 32 + 1 : lo;
}

// Places of a sequence on the axis; one with no visible key takes one tile, so that its rows are written.
__device__ __forceinline__ int few_places(const PagedFewParams& fp, const PagedSeq& s) {
  const int rows = s.n * fp.p.ratio.value;
  if (rows == 0 || rows > fp.rows) return 0;
  int lo, end;
  few_tiles(fp.p, s, lo, end);
  return fp.ahead + max(end - lo, 1);
}
// The inclusive running sum over a wave's lanes.
__device__ __forceinline__ int running_sum(int v) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int below = __shfl_up(v, o, 64);
    if ((int)(threadIdx.x & 63) >= o) v += below;
  }
  return v;
}
// The shares first .. last that hold a sequence's tiles; `start` is its place on the axis.
__device__ __forceinline__ void few_shares(const PagedFewParams& fp, int start, int places, int share, int& first, int& last) {
  first = (start + fp.ahead) / share;
  last = (start + places - 1) / share;
}
// A share's partial of a sequence: slot 0 for the sequence the share begins in, 1 for one that begins inside the share.
__device__ __forceinline__ long few_partial(const PagedFewParams& fp, int g, int h, int start, int share) {
  return (((long)g * fp.p.c.heads + h) * 2 + (g * share >= start ? 0 : 1)) * fp.rows;
}

// Partials pass between workgroups on different XCDs inside a launch: written through to, and read from, where all of them
// see the same memory.
__device__ __forceinline__ void store_shared(float* to, float v) {
  __hip_atomic_store(to, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void store_shared4(float* to, const float4& v) {
  auto* w = reinterpret_cast<unsigned long long*>(to);
  __hip_atomic_store(w, __builtin_bit_cast(unsigned long long, make_float2(v.x, v.y)), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __hip_atomic_store(w + 1, __builtin_bit_cast(unsigned long long, make_float2(v.z, v.w)), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float load_shared(const float* from) {
  return __hip_atomic_load(from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float4 load_shared4(const float* from) {
  const auto* w = reinterpret_cast<const unsigned long long*>(from);
  const float2 a = __builtin_bit_cast(float2, __hip_atomic_load(w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
  const float2 b = __builtin_bit_cast(float2, __hip_atomic_load(w + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
  return make_float4(a.x, a.y, b.x, b.y);
}
// Called by all threads of a workgroup once their store_shared calls are issued: whether it is the last of `expected` to
// arrive at the counter, which is then zero again.  A thread's stores have reached memory before the workgroup is counted.
__device__ __forceinline__ bool arrive_last(int* counter, int expected, int* in_lds) {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    const bool last = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == expected - 1;
    if (last) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *in_lds = last;
  }
  __syncthreads();
  return *in_lds != 0;
}

__device__ __forceinline__ bool finite4(const float4& v) {
  return __builtin_isfinite(v.x) && __builtin_isfinite(v.y) && __builtin_isfinite(v.z) && __builtin_isfinite(v.w);
}

template <class T>
__device__ __forceinline__ void store_o4(const PagedParams& p, int token, int hq, int d, const float4& v) {
  const long at = token * p.o_token + hq * p.o_head + d;
  if (p.out_storage) *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p.O) + at) = make_uint2(pack2<T>(v.x, v.y), pack2<T>(v.z, v.w));
  else *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.O) + at) = v;
}

// FAR: a soft cap over kPlainCap.
template <class T, int FMT, int DP, int NQ, bool FAR>
__global__ __launch_bounds__((FewGeom<FMT, DP>::THREADS), (DP <= 128 && NQ == 1 ? 2 : 1)) void paged_few_kernel(const PagedFewParams fp) {
  using G = FewGeom<FMT, DP>;
  using TV = typename std::conditional<FMT == kStorage, T, F16>::type;    // type of the second product
  const PagedParams& p = fp.p;
  constexpr int KSTEPS = DP / 16, DT = DP / 32, ROWB = G::ROWB, TILE = G::TILE, LD = G::LD, CHUNKS = G::CHUNKS;
  constexpr bool CODES = FMT != kStorage;
  constexpr int TILE_LOADS = 2 * LD + (CODES ? 1 : 0);
  constexpr float LIFT = weight_lift<TV>();
  // A far cap's exponents can be large and yet exact (every score of a row at the cap): log2 vs joins them behind the maximum, not rounded
  // to their magnitude.  Elsewhere an exponent is as large as its score, whose f32 sum is off by more than that rounding, and the
  // second read of log2 vs would cost 2 to 5 % (four tokens on 131072 int8 keys 65.9 -> 68.3 us).
  constexpr bool LATE = CODES && FAR;

  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, lh = lane >> 5;
  char* wsm = smem + wave * G::WAVE_LDS;                // K0 K1 V0 V1, tables, scales
  const uint32_t wlds = (uint32_t)(uintptr_t)(TSR_LDS char*)wsm;

  const int D = p.c.D, H = p.c.heads;
  // Workgroups are dealt to the XCDs round-robin: eight groups at a time, their first heads, their second heads, ...
  int g, h;
  {
    const int i = blockIdx.x, groups = fp.groups ? fp.groups : p.B, full = groups / 8 * 8, rest = groups - full;
    if (i < full * H) {
      const int r = i % (8 * H);
      g = i / (8 * H) * 8 + r % 8;
      h = r / 8;
    } else {
      const int r = i - full * H;
      g = full + r % rest;
      h = r / rest;
    }
  }
  // ---- this group's share of the axis, and the sequence it starts in.  The sequences' places are added up 64 at a time.
  auto seq_of = [&](int b) { return b < p.B ? paged_seq(p, b) : PagedSeq{0, 0, 0}; };
  const PagedSeq mine = fp.groups ? seq_of(lane) : PagedSeq{0, 0, 0};    // the first 64 sequences, one in a lane
  int b = 0, start = 0, share = 1, pos, pos_end;          // start: where sequence b starts on the axis
  if (fp.groups) {
    const int own0 = few_places(fp, mine), sum0 = running_sum(own0);
    int total = __shfl(sum0, 63, 64);
    for (int b0 = 64; b0 < p.B; b0 += 64) total += __shfl(running_sum(few_places(fp, seq_of(b0 + lane))), 63, 64);
    total = __builtin_amdgcn_readfirstlane(total);
    share = max((total + fp.groups - 1) / fp.groups, 1);
    pos = g * share;
    pos_end = min(pos + share, total);
    bool found = false;
    for (int b0 = 0, before = 0; b0 < p.B && !found; b0 += 64) {
      const int own = b0 == 0 ? own0 : few_places(fp, seq_of(b0 + lane)), sum = b0 == 0 ? sum0 : running_sum(own);
      const unsigned long long past = __ballot(before + sum > pos);
      if (past) {
        const int first = __builtin_ctzll(past);
        b = b0 + first;
        start = before + __shfl(sum - own, first, 64);
        found = true;
      }
      before += __shfl(sum, 63, 64);
    }
    b = __builtin_amdgcn_readfirstlane(b);
    start = __builtin_amdgcn_readfirstlane(start);
  } else {                                                // a sequence for each workgroup of a head
    b = g;
    pos = 0;
    pos_end = 1 << 30;
    share = 1 << 30;
  }

  for (; pos < pos_end; ++b) {
  PagedSeq s;
  if (fp.groups && b < 64) {
    s.q0 = __builtin_amdgcn_readlane(mine.q0, b);
    s.n = __builtin_amdgcn_readlane(mine.n, b);
    s.kv = __builtin_amdgcn_readlane(mine.kv, b);
  } else {
    s = paged_seq(p, b);
  }
  const int places = few_places(fp, s);
  if (places == 0) {
    if (!fp.groups) return;
    continue;
  }
  const int rows = s.n * p.ratio.value;
  int tile_lo, tile_end;
  few_tiles(p, s, tile_lo, tile_end);
  const int seq_start = start, seq_end = start + places;
  const int t0 = tile_lo + max(pos - seq_start - fp.ahead, 0), t1 = min(tile_lo + min(pos_end, seq_end) - seq_start - fp.ahead, tile_end);
  int first_share, last_share;
  few_shares(fp, seq_start, places, share, first_share, last_share);
  const bool whole = first_share == last_share;         // this workgroup has the sequence's whole key range
  start = seq_end;
  pos = fp.groups ? min(pos_end, seq_end) : pos_end;
  if (g < first_share) continue;                         // only the places ahead of it lie in this share

  // Row i of the group (tile i / 32, column i % 32) is token i / ratio, head i % ratio of the group.
  uint4 qf[NQ][KSTEPS];
  int klo[NQ], khi[NQ];                                 // a row past the group's sees no key
#pragma unroll
  for (int qt = 0; qt < NQ; ++qt) {
    const int i = 32 * qt + l32;
    const bool valid = i < rows;
    const int tok = valid ? p.ratio.quotient(i) : 0, hs = valid ? i - tok * p.ratio.value : 0;
    const uint16_t* src = p.Q + (s.q0 + tok) * p.q_token + (h * p.ratio.value + hs) * p.q_head;
    // (codes: K is read 16 codes at a time, so the steps 2 j and 2 j + 1 share the columns 32 j + 16 lh .. + 15)
#pragma unroll
    for (int ks = 0; ks < KSTEPS; ++ks) {
      const int d = CODES ? 32 * (ks >> 1) + 16 * lh + 8 * (ks & 1) : 16 * ks + 8 * lh;
      qf[qt][ks] = valid && d < D ? *reinterpret_cast<const uint4*>(src + d) : make_uint4(0u, 0u, 0u, 0u);
    }
    klo[qt] = 0;
    khi[qt] = -1;
    if (valid) key_bounds(tok, s.n, s.kv, p.causal, p.window, klo[qt], khi[qt]);
  }
  int lo0, hi0, lo1, hi1;                               // bounds of the first and the last token
  key_bounds(0, s.n, s.kv, p.causal, p.window, lo0, hi0);
  key_bounds(s.n - 1, s.n, s.kv, p.causal, p.window, lo1, hi1);

  // ---- loader: the lane's 16-byte slot q * 64 + lane of a tile is (row slot / CHUNKS, physical chunk slot % CHUNKS).
  // D < DP: the chunks past a row's end are its first chunk again; they meet zeros of Q, and output columns that are not
  // stored.  (Where that chunk holds something not finite, 0 times it makes the row's result not finite: see the end.)
  const char* Kh = p.c.k + h * p.c.k_head;
  const char* Vh = p.c.v + h * p.c.v_head;
  const int row_chunks = D * G::ESZ / 16;
  uint32_t k_off[LD], v_off[LD];
#pragma unroll
  for (int q = 0; q < LD; ++q) {
    const int slot = q * 64 + lane, row = slot / CHUNKS, phys = slot % CHUNKS;
    const int kc = phys ^ k_swizzle<ROWB>(row), vc = phys ^ v_swizzle<ROWB, CODES>(row);
    k_off[q] = kc < row_chunks ? 16 * kc : 0;
    v_off[q] = vc < row_chunks ? 16 * vc : 0;
  }
  const int last = s.kv - 1;
  const int* table = p.table + (long)b * p.pages_per_seq;
  auto load_table = [&](int tile, int stage) __attribute__((always_inline)) {          // the pages of a tile's 32 keys
    const int entry = p.c.page_size.quotient(min(tile * G::BK + l32, last));
    if (lane < 32) gather4_to_lds(table + entry, __builtin_amdgcn_readfirstlane(wlds + G::TABLE_AT + stage * 128));
  };
  // A lane for a key, one half of the wave for K and one for V: where the rows of a tile start (its table stage has landed).
  // A scale lies where its row does, in its own strides; its offset is kept until the tile is loaded.
  long scale_at = 0;
  auto find_rows = [&](int tile, int stage) __attribute__((always_inline)) {
    const int key = min(tile * G::BK + l32, last), entry = p.c.page_size.quotient(key), place = key - entry * p.c.page_size.value;
    const int id = *reinterpret_cast<const int*>(wsm + G::TABLE_AT + stage * 128 + l32 * 4);
    const int page = (unsigned)id < (unsigned)p.c.pages ? id : 0;
    *reinterpret_cast<long*>(wsm + G::ROWS_AT + lane * 8) = lh ? p.c.v_at(page, place) : p.c.k_at(page, place);
    if constexpr (CODES) scale_at = p.c.scale_at(page, place);
  };
  auto load_tile_as = [&](auto nt_c, int stage) __attribute__((always_inline)) {
    constexpr bool NT = decltype(nt_c)::value;
#pragma unroll
    for (int q = 0; q < LD; ++q) {
      const char* row = wsm + G::ROWS_AT + (q * 64 + lane) / CHUNKS * 8;
      const uint32_t k_lds = __builtin_amdgcn_readfirstlane(wlds + stage * TILE + q * 1024);
      gather16_to_lds<NT>(Kh + *reinterpret_cast<const long*>(row) + k_off[q], k_lds);
      gather16_to_lds<NT>(Vh + *reinterpret_cast<const long*>(row + 256) + v_off[q], k_lds + 2 * TILE);
    }
    if constexpr (CODES)
      gather4_to_lds((lh ? p.c.v_scale : p.c.k_scale) + scale_at + h * p.c.s_head,
                     __builtin_amdgcn_readfirstlane(wlds + G::SCALE_AT + stage * 256));
  };
  auto load_tile = [&](int stage) __attribute__((always_inline)) {
    if (fp.once) load_tile_as(std::true_type{}, stage);
    else load_tile_as(std::false_type{}, stage);
  };

  // ---- LDS read addresses
  uint32_t k_rd[CODES ? KSTEPS / 2 : KSTEPS];
#pragma unroll
  for (int j = 0; j < (CODES ? KSTEPS / 2 : KSTEPS); ++j) k_rd[j] = l32 * ROWB + (((2 * j + lh) ^ k_swizzle<ROWB>(l32)) << 4);
  const int r16 = lane & 15, blk = (lane >> 4) & 1;
  uint32_t v_rd[DT];                                    // + 16 g ROWB for the key step g
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
    if constexpr (CODES) {                              // lane r of 16 supplies key r / 2 of the step's eight, columns 8 (r % 2)
      const int kk = r16 >> 1, key = (kk < 4 ? kk : kk + 4) + 4 * lh, col = dt * 32 + 16 * blk + 8 * (r16 & 1);
      v_rd[dt] = 2 * TILE + key * ROWB + (((col >> 4) ^ v_swizzle<ROWB, true>(key)) << 4) + (col & 15);
    } else {
      const int key = 4 * lh + (r16 >> 2), col = dt * 32 + 16 * blk + 4 * (r16 & 3);
      v_rd[dt] = 2 * TILE + key * ROWB + (((col >> 3) ^ v_swizzle<ROWB, false>(key)) << 4) + (col & 7) * 2;
    }
  }

  // ---- state
  f32x16 o_acc[NQ][DT];
  float m_run[NQ], l_run[NQ];
#pragma unroll
  for (int qt = 0; qt < NQ; ++qt) {
    m_run[qt] = FA_NEG;
    l_run[qt] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) o_acc[qt][dt][r] = 0.f;
  }
  // A score's exponent in base 2 is scale log2(e) s, folded into the exponential or applied before it.
  const float c = p.scale * 1.44269504088896340736f;
  const bool fold = folds(p);
  const SoftCap cap = fold ? SoftCap() : SoftCap(p, FAR);
  const float slope = fold || !(p.softcap > 0.f) ? c : cap.slope;
  const float cs = CODES ? 1.0f : fold ? c : cap.slope;  // what is left to multiply at the exponential

  // At the head of a step this tile's rows and the pages of the tile after the next are in flight, the next tile's row offsets
  // in LDS.  The step issues the next tile's rows, waits for everything older, looks up the rows of the tile after the next
  // and issues the pages of the one behind it: no wait is shorter than a step.
  const int W = G::WAVES;
  int t = t0 + wave, stage = 0;
  if (t < t1) {
    load_table(t, 0);
    load_table(min(t + W, t1 - 1), 1);
    wait_loads<0>();
    find_rows(t, 0);
    load_tile(0);
    find_rows(min(t + W, t1 - 1), 1);
    load_table(min(t + 2 * W, t1 - 1), 0);
  }
  for (; t < t1; t += W) {
    if (t + W < t1) {
      load_tile(stage ^ 1);
      wait_loads<TILE_LOADS>();
      if (t + 2 * W < t1) {
        find_rows(t + 2 * W, stage);
        load_table(min(t + 3 * W, t1 - 1), stage ^ 1);
      }
    } else {
      wait_loads<0>();
    }
    const float* scales = reinterpret_cast<const float*>(wsm + G::SCALE_AT + stage * 256);
    f32x16 sc[NQ];
#pragma unroll
    for (int qt = 0; qt < NQ; ++qt)
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[qt][r] = 0.f;
    if constexpr (CODES) {
#pragma unroll
      for (int j = 0; j < KSTEPS / 2; ++j) {
        const uint4 w = lds_read_b128(wsm, k_rd[j] + stage * TILE);
        const uint4 k0 = decode8<T, FMT>(make_uint2(w.x, w.y)), k1 = decode8<T, FMT>(make_uint2(w.z, w.w));
#pragma unroll
        for (int qt = 0; qt < NQ; ++qt) {
          sc[qt] = mfma_32x32x16<T>(k0, qf[qt][2 * j], sc[qt]);
          sc[qt] = mfma_32x32x16<T>(k1, qf[qt][2 * j + 1], sc[qt]);
        }
      }
    } else {
#pragma unroll
      for (int ks = 0; ks < KSTEPS; ++ks) {
        const uint4 kf = lds_read_b128(wsm, k_rd[ks] + stage * TILE);
#pragma unroll
        for (int qt = 0; qt < NQ; ++qt) sc[qt] = mfma_32x32x16<T>(kf, qf[qt][ks], sc[qt]);
      }
    }
    if constexpr (CODES) {                               // (a lane has read its scale when the first of them writes)
      const float vs = weight_scale(scales[32 + l32]);
      *reinterpret_cast<float*>(lh ? wsm + G::INVERSE_AT + 4 * l32 : wsm + G::SCALE_AT + stage * 256 + 128 + 4 * l32) =
          lh ? __builtin_amdgcn_rcpf(vs) : __builtin_amdgcn_logf(vs);
    }
    if constexpr (CODES) {
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const float4 x = *reinterpret_cast<const float4*>(scales + 8 * a + 4 * lh);
#pragma unroll
        for (int qt = 0; qt < NQ; ++qt) {
          sc[qt][4 * a + 0] *= x.x; sc[qt][4 * a + 1] *= x.y; sc[qt][4 * a + 2] *= x.z; sc[qt][4 * a + 3] *= x.w;
        }
      }
    }
    const int kv0 = t * G::BK;
    const bool need_mask = kv0 + G::BK - 1 > hi0 || kv0 < lo1;
    uint4 pf[NQ][2];
#pragma unroll
    for (int qt = 0; qt < NQ; ++qt) {
      if (!fold) {
        if constexpr (FAR) {
#pragma unroll
          for (int r = 0; r < 16; ++r) sc[qt][r] = far_exponent(sc[qt][r], c, cap.in, cap.top);
        } else if (p.softcap > 0.f) {
#pragma unroll
          for (int r = 0; r < 16; ++r) sc[qt][r] = cap.form(sc[qt][r]);
        } else if (!CODES) {
#pragma unroll
          for (int r = 0; r < 16; ++r) sc[qt][r] *= c;
        }
      }
      if constexpr (CODES && !LATE) {
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          const float4 x = *reinterpret_cast<const float4*>(scales + 32 + 8 * a + 4 * lh);
          sc[qt][4 * a + 0] = fmaf(sc[qt][4 * a + 0], slope, x.x); sc[qt][4 * a + 1] = fmaf(sc[qt][4 * a + 1], slope, x.y);
          sc[qt][4 * a + 2] = fmaf(sc[qt][4 * a + 2], slope, x.z); sc[qt][4 * a + 3] = fmaf(sc[qt][4 * a + 3], slope, x.w);
        }
      }
      if (need_mask) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int key = kv0 + 8 * (r >> 2) + 4 * lh + (r & 3);
          if (key > khi[qt] || key < klo[qt]) sc[qt][r] = FA_NEG;                 // (LATE: log2 vs is nothing beside it)
        }
      }
      float mx;
      if constexpr (LATE) {
        mx = FA_NEG;
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          const float4 x = *reinterpret_cast<const float4*>(scales + 32 + 8 * a + 4 * lh);
          mx = max3_raw(mx, sc[qt][4 * a + 0] + x.x, sc[qt][4 * a + 1] + x.y);
          mx = max3_raw(mx, sc[qt][4 * a + 2] + x.z, sc[qt][4 * a + 3] + x.w);
        }
      } else {
        mx = max3_raw(sc[qt][0], sc[qt][1], sc[qt][2]);
#pragma unroll
        for (int r = 3; r < 16; r += 2) mx = (r + 1 < 16) ? max3_raw(mx, sc[qt][r], sc[qt][r + 1]) : fmaxf(mx, sc[qt][r]);
      }
      mx = max_with_other_half(mx);
      const float m_new = fmaxf(m_run[qt], mx);
      if (__any(m_new > m_run[qt])) {
        const float corr = fast_exp2((m_run[qt] - m_new) * cs);
        l_run[qt] *= corr;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int r = 0; r < 16; ++r) o_acc[qt][dt][r] *= corr;
        m_run[qt] = m_new;
      }
      // (a row that has met no visible key keeps the sentinel: reference 0, so masked entries give P = 0)
      const float mc = m_new > 0.5f * FA_NEG ? fmaf(m_new, cs, -LIFT) : 0.f;
      float sum = 0.f;
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        if constexpr (LATE) {
#pragma unroll
          for (int a = 2 * g; a < 2 * g + 2; ++a) {
            const float4 x = *reinterpret_cast<const float4*>(scales + 32 + 8 * a + 4 * lh);
            sc[qt][4 * a + 0] = sc[qt][4 * a + 0] - mc + x.x; sc[qt][4 * a + 1] = sc[qt][4 * a + 1] - mc + x.y;
            sc[qt][4 * a + 2] = sc[qt][4 * a + 2] - mc + x.z; sc[qt][4 * a + 3] = sc[qt][4 * a + 3] - mc + x.w;
          }
        }
#pragma unroll
        for (int r = 8 * g; r < 8 * g + 8; ++r) {
          const float e = fast_exp2(LATE ? sc[qt][r] : CODES ? sc[qt][r] - mc : fmaf(sc[qt][r], cs, -mc));
          sc[qt][r] = e;
          if (!CODES) sum += e;
        }
        if constexpr (CODES) {
#pragma unroll
          for (int a = 2 * g; a < 2 * g + 2; ++a) {
            const float4 x = *reinterpret_cast<const float4*>(wsm + G::INVERSE_AT + 32 * a + 16 * lh);
            sum = fmaf(sc[qt][4 * a + 0], x.x, sum); sum = fmaf(sc[qt][4 * a + 1], x.y, sum);
            sum = fmaf(sc[qt][4 * a + 2], x.z, sum); sum = fmaf(sc[qt][4 * a + 3], x.w, sum);
          }
        }
        pf[qt][g].x = pack2<TV>(sc[qt][8 * g + 0], sc[qt][8 * g + 1]);
        pf[qt][g].y = pack2<TV>(sc[qt][8 * g + 2], sc[qt][8 * g + 3]);
        pf[qt][g].z = pack2<TV>(sc[qt][8 * g + 4], sc[qt][8 * g + 5]);
        pf[qt][g].w = pack2<TV>(sc[qt][8 * g + 6], sc[qt][8 * g + 7]);
      }
      l_run[qt] += sum;
    }
    // O^T += V^T P^T, 16 keys a step; a V fragment serves the NQ query tiles
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const uint32_t a = v_rd[dt] + stage * TILE + g * 16 * ROWB;
        uint4 vf;
        if constexpr (CODES) {
          vf = decode8<TV, FMT>(lds_read_tr8_b64(wsm + a));
        } else {
          const uint2 lo = lds_read_tr16_b64(wsm + a);
          const uint2 hi = lds_read_tr16_b64(wsm + a + 8 * ROWB);
          vf = make_uint4(lo.x, lo.y, hi.x, hi.y);
        }
#pragma unroll
        for (int qt = 0; qt < NQ; ++qt) {
          o_acc[qt][dt] = mfma_32x32x16<TV>(vf, pf[qt][g], o_acc[qt][dt]);
        }
      }
    stage ^= 1;
  }

  // ---- merge the waves' partials through LDS, one 32-row query tile at a time
  float* ml = reinterpret_cast<float*>(smem + G::ML_AT);      // m[WAVES][32] | l[WAVES][32] | m_tot[32] | l_tot[32] | flags[32]
  int* flags = reinterpret_cast<int*>(ml + (2 * G::WAVES + 2) * 32);
#pragma unroll
  for (int qt = 0; qt < NQ; ++qt) {
    if (32 * qt >= rows) break;
    __syncthreads();                                          // every wave is done with its tiles / the last pass
    const float l_wave = l_run[qt] + swap_half(l_run[qt]);
    if (lh == 0) {
      ml[wave * 32 + l32] = m_run[qt];
      ml[(G::WAVES + wave) * 32 + l32] = l_wave;
    }
    if (tid < 32) flags[tid] = 0;
    __syncthreads();
    float m_tot = FA_NEG;
#pragma unroll
    for (int w = 0; w < G::WAVES; ++w) m_tot = fmaxf(m_tot, ml[w * 32 + l32]);
    float l_tot = 0.f;
#pragma unroll
    for (int w = 0; w < G::WAVES; ++w) l_tot += ml[(G::WAVES + w) * 32 + l32] * fast_exp2((ml[w * 32 + l32] - m_tot) * cs);
    const float mine = fast_exp2((m_run[qt] - m_tot) * cs);   // both sentinels: 1, on accumulators that are 0
    if (wave == 0 && lh == 0) {
      ml[2 * G::WAVES * 32 + l32] = m_tot;
      ml[(2 * G::WAVES + 1) * 32 + l32] = l_tot;
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const int d = dt * 32 + 8 * a + 4 * lh;
        *reinterpret_cast<float4*>(wsm + l32 * G::PITCH + d * 4) =
            make_float4(o_acc[qt][dt][4 * a + 0] * mine, o_acc[qt][dt][4 * a + 1] * mine, o_acc[qt][dt][4 * a + 2] * mine,
                        o_acc[qt][dt][4 * a + 3] * mine);
      }
    __syncthreads();
    // every thread sums four columns of one row over the waves and stores them
    const int rows_here = min(32, rows - 32 * qt);
    for (int idx = tid; idx < rows_here * (DP / 4); idx += G::THREADS) {
      const int il = idx / (DP / 4), d = (idx - il * (DP / 4)) * 4;
      if (d >= D) continue;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < G::WAVES; ++w) {
        const float4 v = *reinterpret_cast<const float4*>(smem + w * G::WAVE_LDS + il * G::PITCH + d * 4);
        acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
      }
      const float mt = ml[2 * G::WAVES * 32 + il], lt = ml[(2 * G::WAVES + 1) * 32 + il];
      const float inv = lt == 0.f ? 0.f : 1.0f / lt;
      acc.x *= inv; acc.y *= inv; acc.z *= inv; acc.w *= inv;
      const int i = 32 * qt + il, tok = p.ratio.quotient(i), hq = h * p.ratio.value + i - tok * p.ratio.value;
      const long row = (long)(s.q0 + tok) * p.Hq + hq;
      const float lse = lt == 0.f ? -INFINITY : (mt * cs + (cap.base - LIFT) + __log2f(lt)) * 0.69314718055994530942f;
      if (whole) {
        if (!finite4(acc) || lt == 0.f) flags[il] = 1;
        store_o4<T>(p, s.q0 + tok, hq, d, acc);
        if (p.LSE && d == 0) p.LSE[row] = lse;
      } else {
        const long at = few_partial(fp, g, h, seq_start, share) + i;
        store_shared4(fp.part_o + at * D + d, acc);
        if (d == 0) store_shared(fp.part_lse + at, lse);
      }
    }
    if (whole) {
      // A value that is not finite in a key that a row does not see reached the row as 0 times that value, and scores as low as
      // the mask's sentinel count as masked: rows that are not finite, or have no weight, are formed again from the keys they see.
      __syncthreads();
      for (int il = wave; il < rows_here; il += G::WAVES) {
        if (!flags[il]) continue;
        const int i = 32 * qt + il, tok = p.ratio.quotient(i);
        paged_row<T, FMT>(p, b, s.q0 + tok, tok, s.n, s.kv, h * p.ratio.value + i - tok * p.ratio.value);
      }
    }
  }
  if (!whole && fp.arrived && arrive_last(fp.arrived + (long)b * H + h, last_share - first_share + 1, flags + 32)) {
    // O = sum_k w_k O_k / sum_k w_k, w_k = exp(LSE_k - max LSE); a thread for four columns of a row, eight partials fetched
    // together, a running maximum over the eights
    for (int i0 = 0; i0 < rows; i0 += 32) {
      if (tid < 32) flags[tid] = 0;
      __syncthreads();
      const int rows_here = min(32, rows - i0);
      for (int idx = tid; idx < rows_here * (DP / 4); idx += G::THREADS) {
        const int il = idx / (DP / 4), d = (idx - il * (DP / 4)) * 4, i = i0 + il;
        if (d >= D) continue;
        float mx = -INFINITY, wsum = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int k0 = first_share; k0 <= last_share; k0 += 8) {
          float l[8];
          float4 v[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            const long at = few_partial(fp, min(k0 + u, last_share), h, seq_start, share) + i;
            l[u] = load_shared(fp.part_lse + at);
            v[u] = load_shared4(fp.part_o + at * D + d);
          }
          float top = mx;
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            if (k0 + u > last_share) l[u] = -INFINITY;
            top = fmaxf(top, l[u]);
          }
          const float ref = top > -INFINITY ? top : 0.f, corr = __expf(mx - ref);
          acc.x *= corr; acc.y *= corr; acc.z *= corr; acc.w *= corr;
          wsum *= corr;
          mx = top;
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            const float w = __expf(l[u] - ref);
            acc.x += w * v[u].x; acc.y += w * v[u].y; acc.z += w * v[u].z; acc.w += w * v[u].w;
            wsum += w;
          }
        }
        const float inv = wsum == 0.f ? 0.f : 1.0f / wsum;
        acc.x *= inv; acc.y *= inv; acc.z *= inv; acc.w *= inv;
        const int tok = p.ratio.quotient(i), hq = h * p.ratio.value + i - tok * p.ratio.value;
        if (!finite4(acc) || !(wsum > 0.f)) flags[il] = 1;
        store_o4<T>(p, s.q0 + tok, hq, d, acc);
        if (p.LSE && d == 0) p.LSE[(long)(s.q0 + tok) * p.Hq + hq] = wsum == 0.f ? -INFINITY : mx + __logf(wsum);
      }
      __syncthreads();
      for (int il = wave; il < rows_here; il += G::WAVES) {
        if (!flags[il]) continue;
        const int i = i0 + il, tok = p.ratio.quotient(i);
        paged_row<T, FMT>(p, b, s.q0 + tok, tok, s.n, s.kv, h * p.ratio.value + i - tok * p.ratio.value);
      }
      __syncthreads();
    }
  }
  __syncthreads();                                           // the next sequence's tiles overwrite what was merged
  }
}

}  // namespace tsr950
