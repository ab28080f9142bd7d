// Attention over a paged cache for sequences with many new tokens (chunks of prompts).
//
// The contiguous forward kernel's arithmetic (flash_attn.h: transposed products, lane-local softmax rows) on other rows and
// other loads:
//
// - The 32 query rows of an MFMA tile are (token, head of the group) pairs, heads fastest: a workgroup's rows are the group's
//   Hq / heads query heads of neighbouring tokens.  One walk over K and V serves them all, a causal mask cuts the walk at
//   the block's last token rather than at a block of 256 tokens, and a chunk of 20 tokens fills a tile as one of 256 does.
// - Workgroups find their sequence themselves: blockIdx.x counts the blocks of all sequences in order, KV heads fastest; a
//   wave adds up the sequences' blocks 64 at a time.  blockIdx.y is the part of the block's key range.
// - K and V rows come through the page table: two tiles ahead one wave looks up the pages of a tile's 64 keys, a lane for
//   a key, and leaves the rows' addresses in LDS, where every thread that loads a piece of a row finds it.  Any page size
//   costs the same.  16-bit pages go straight into LDS; codes go through registers, become 16-bit values there, once for the whole
//   workgroup, and are written to the same LDS layout; K's scales multiply the scores and V's the probabilities, in f32.
//
// Bound by the softmax's vector work beside the MFMAs, as the contiguous kernel (matrix pipes busy 44 % of the cycles; 278 us there,
// 293 here for B 4, 2048 tokens on 3000 keys, D 128).  Measured (Hq 32, Hkv 8, D 128, bf16): four sequences of 2048 tokens on 2048
// to 4096 keys 281 to 306 us from card to card = 856 to 930 TFLOP/s; 512 tokens on 16384 keys, split in four, 147 to 160 us with the merge; over
// e4m3 codes 12 % longer (the decoding), at D 256 530 TFLOP/s (one wave to a SIMD).
#pragma once
#include <type_traits>
#include "paged_few.h"

namespace tsr950 {

// With codes the second product is in bf16 (a probability times V's scale needs its range; codes are exact in it).  A bf16
// program rounds its result as coarsely; for an f16 program the probabilities' remainders go through a second product, which
// keeps 16 bits of them: error of the f32 result 1.7e-3 without, 3e-6 with it.  (The few-rows kernel's weights in f16 take 25 registers
// more here, which spilled: B 4, 2048 tokens on 3000 e4m3 keys, bf16 332 us, 446 with them; f16 433 and 446.)
template <class T, int FMT> constexpr bool splits_p() { return FMT != kStorage && std::is_same<T, F16>::value; }
// What eight values lost when they were packed to bf16, packed.
__device__ __forceinline__ uint4 remainder8(const f32x16& x, int r0, const uint4& packed) {
  auto low = [](uint32_t w) { return __builtin_bit_cast(float, w << 16); };
  auto high = [](uint32_t w) { return __builtin_bit_cast(float, w & 0xffff0000u); };
  return make_uint4(pack2<BF16>(x[r0] - low(packed.x), x[r0 + 1] - high(packed.x)),
                    pack2<BF16>(x[r0 + 2] - low(packed.y), x[r0 + 3] - high(packed.y)),
                    pack2<BF16>(x[r0 + 4] - low(packed.z), x[r0 + 5] - high(packed.z)),
                    pack2<BF16>(x[r0 + 6] - low(packed.w), x[r0 + 7] - high(packed.w)));
}

// W waves of 32 rows each.  DP = 256 takes four waves, one to a SIMD: a wave's 128 output, 64 Q and 32 score registers do not
// fit beside a second wave's.
template <int DP, int W> struct TileGeom {
  static constexpr int THREADS = W * 64, BQ = W * 32;
  static constexpr int TILE = FA_BKV * DP * 2;           // bytes of one K (or V) stage
  static constexpr int PITCH = DP * 4 + 16;              // epilogue staging row, f32
  static constexpr int BODY = 4 * TILE > W * 32 * PITCH ? 4 * TILE : W * 32 * PITCH;
  static constexpr int ROWS_AT = BODY;                   // four stages of 64 K row addresses, then as many of V
  static constexpr int SCALE_AT = ROWS_AT + 8 * 512;     // four stages of 64 K scales, four of 64 V scales
  static constexpr int SMEM(bool codes) { return SCALE_AT + (codes ? 8 * 256 : 0); }
};

// 16 bytes at an address that was kept as a number: not a flat load, which would wait for LDS as well.
__device__ __forceinline__ uint4 load_global16(const char* from) {
  return __builtin_bit_cast(uint4, *(const __attribute__((address_space(1))) i32x4*)from);
}

struct PagedTileParams {
  PagedParams p;
  float* part_o;            // [nsplit][total_q * Hq][D] normalised partial O; null where no walk is split
  float* part_lse;          // [nsplit][total_q * Hq]
  int nsplit, min_rows;     // sequences with at most min_rows rows a KV head are another kernel's
};

// Blocks of `block` rows of a sequence.
__device__ __forceinline__ int tile_blocks(const PagedTileParams& tp, int n, int block) {
  const int rows = n * tp.p.ratio.value;
  return rows > tp.min_rows ? (rows + block - 1) / block : 0;
}

// The 64-key tiles [lo, lo + count) of a block's rows, and the share of one of the nsplit workgroups that divide them.
__device__ __forceinline__ void tile_range(const PagedTileParams& tp, const PagedSeq& s, int first_row, int block, int& lo, int& count,
                                           int& share) {
  const PagedParams& p = tp.p;
  const int rows = s.n * p.ratio.value;
  int lo0, hi0, lo1, hi1;
  key_bounds(p.ratio.quotient(first_row), s.n, s.kv, p.causal, p.window, lo0, hi0);
  key_bounds(p.ratio.quotient(min(first_row + block, rows) - 1), s.n, s.kv, p.causal, p.window, lo1, hi1);
  lo = lo0 / FA_BKV;
  count = hi1 >= lo0 ? hi1 / FA_BKV + 1 - lo : 0;
  share = (count + tp.nsplit - 1) / tp.nsplit;
}

// What workgroup `index` serves: KV head, sequence, first row (blocks with the longest walks first).  The sequences' blocks are
// added up 64 at a time.
__device__ __forceinline__ bool find_block(const PagedTileParams& tp, int index, int block, int& h, int& b, int& r0, PagedSeq& s) {
  const PagedParams& p = tp.p;
  const int lane = threadIdx.x & 63;
  int at = index / p.c.heads;
  h = index - at * p.c.heads;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    const PagedSeq mine = b0 + lane < p.B ? paged_seq(p, b0 + lane) : PagedSeq{0, 0, 0};
    const int own = tile_blocks(tp, mine.n, block), sum = running_sum(own);
    const unsigned long long past = __ballot(sum > at);
    if (past) {
      const int first = __builtin_ctzll(past);
      b = b0 + first;
      at -= __builtin_amdgcn_readlane(sum - own, first);
      s = PagedSeq{__builtin_amdgcn_readlane(mine.q0, first), __builtin_amdgcn_readlane(mine.n, first), __builtin_amdgcn_readlane(mine.kv, first)};
      r0 = (tile_blocks(tp, s.n, block) - 1 - at) * block;
      return true;
    }
    at -= __builtin_amdgcn_readlane(sum, 63);
  }
  return false;
}

// EXT 0: the scale is folded into the exponential.  1: a soft cap, or a scale that is not well above zero: scores become exponents
// before the mask.  2: the same for a cap over kPlainCap.
template <class T, int FMT, int DP, int W, int EXT>
__global__ __launch_bounds__((TileGeom<DP, W>::THREADS), (DP > 128 ? 1 : 2)) void paged_tile_kernel(const PagedTileParams tp) {
  using G = TileGeom<DP, W>;
  using TV = typename std::conditional<FMT == kStorage, T, BF16>::type;
  constexpr bool CODES = FMT != kStorage;
  constexpr bool SPLIT = splits_p<T, FMT>();
  constexpr float LIFT = weight_lift<TV>();
  constexpr int THREADS = G::THREADS, BQ = G::BQ, KT = FA_BKV / 32, KSTEPS = DP / 16;
  constexpr int DT = DP / 32, ROWB = DP * 2, CHUNKS = DP / 8, TILE = G::TILE;
  // pieces of 16 bytes from memory: 8 values, or 16 codes
  constexpr int PIECES = CODES ? DP / 16 : CHUNKS;
  constexpr int LD = (FA_BKV * PIECES + THREADS - 1) / THREADS;
  constexpr bool SPARE = FA_BKV * PIECES < THREADS;              // DP = 64 codes: four of eight waves have no piece
  const PagedParams& p = tp.p;

  extern __shared__ __attribute__((aligned(16))) char smem[];    // K stages 0, 1, V stages 0, 1, tables, scales
  const uint32_t lds0 = (uint32_t)(uintptr_t)(TSR_LDS char*)smem;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, lh = lane >> 5;
  const int D = p.c.D, split = blockIdx.y;

  int h, b, r0;
  PagedSeq s;
  if (!find_block(tp, blockIdx.x, BQ, h, b, r0, s)) return;
  const int rows = s.n * p.ratio.value;
  int tile_base, ntiles, share;
  tile_range(tp, s, r0, BQ, tile_base, ntiles, share);
  if (tp.nsplit > 1) {
    const int from = split * share;
    if (from >= ntiles) return;                          // (nothing left for this part: the merge counts the parts the same way)
    tile_base += from;
    ntiles = min(share, ntiles - from);
  }

  // Eight waves: w and w + 4 share a SIMD; the upper half takes its row blocks in reverse, so that each SIMD has the same
  // work under a causal mask.
  const int rblk = wave < W / 2 || W < 8 ? wave : W + W / 2 - 1 - wave;
  const int rw = r0 + rblk * 32;                         // first row of the wave
  auto token_of = [&](int row) { return p.ratio.quotient(row); };

  int nt_w = 0, t_w0 = 0;
  int wlo_first = 0, whi_first = 0, wlo_last = 0, whi_last = 0;
  if (rw < rows) {
    key_bounds(token_of(rw), s.n, s.kv, p.causal, p.window, wlo_first, whi_first);
    key_bounds(token_of(min(rw + 32, rows) - 1), s.n, s.kv, p.causal, p.window, wlo_last, whi_last);
    nt_w = min(max((whi_last + FA_BKV) / FA_BKV - tile_base, 0), ntiles);
    t_w0 = min(max(wlo_first / FA_BKV - tile_base, 0) & ~1, nt_w);
  }

  // ---- loader.  Piece P = (wave * LD + q) * 64 + lane of a tile is (row P / PIECES, piece P % PIECES).  In LDS a row's
  // 16-byte chunks are XOR-swizzled (k_swizzle, v_swizzle).
  const char* Kh = p.c.k + h * p.c.k_head;
  const char* Vh = p.c.v + h * p.c.v_head;
  const int row_pieces = D / (CODES ? 16 : 8), last = s.kv - 1;
  const int* table = p.table + (long)b * p.pages_per_seq;
  // What a thread keeps of a piece: the row's place among the addresses (of piece q: 64 / PIECES rows further for each), the
  // piece's offset in the row, and, for codes, where the 16 values of its first piece go.
  uint32_t k_off[LD], v_off[LD];
  const uint32_t row_at = (wave * LD * 64 + lane) / PIECES % FA_BKV * 8;
#pragma unroll
  for (int q = 0; q < LD; ++q) {
    const int P = (wave * LD + q) * 64 + lane, row = P / PIECES % FA_BKV;
    const int phys = P % PIECES;
    // (D < DP: the pieces past a row's end are its first piece again.  They meet zeros of Q, and output columns that are not
    // stored; where that piece holds something not finite, 0 times it makes the row's result not finite: see the end.)
    auto piece_off = [&](int piece) { return 16u * (piece < row_pieces ? piece : 0); };
    if constexpr (CODES) {
      k_off[q] = v_off[q] = piece_off(phys);
    } else {                                             // the LDS slot is the physical chunk: the swizzle is in the address
      k_off[q] = piece_off(phys ^ k_swizzle<ROWB>(row));
      v_off[q] = piece_off(phys ^ v_swizzle<ROWB, false>(row));
    }
  }
  // (piece q's row lies ROW_STEP q behind: K's swizzle is row % 16 where there is more than one piece, V's has the period 4)
  constexpr int ROW_STEP = 64 / PIECES;
  static_assert(!CODES || LD == 1 || (ROWB >= 256 && ROW_STEP % 4 == 0), "swizzles by XOR");
  uint32_t k_to = 0, v_to = 0;
  if constexpr (CODES) {
    const int row = row_at / 8, chunk = 2 * (lane % PIECES);
    k_to = row * ROWB + ((chunk ^ k_swizzle<ROWB>(row)) << 4);                   // (the second eight: the next chunk, address ^ 16)
    v_to = 2 * TILE + row * ROWB + ((chunk ^ v_swizzle<ROWB, false>(row)) << 4);
  }
  // The first wave, a lane for a key: the page of a tile's keys, then its rows' addresses (and its scales' offset, kept until
  // they are loaded, a step later).  Rows past the last key repeat the last key's row.
  constexpr int ROWS_AT = G::ROWS_AT, SCALE_AT = G::SCALE_AT;
  int page_entry = 0, page_place = 0;
  long scales_at = 0;
  auto find_page = [&](int tile, int& entry_of, int& place_of) __attribute__((always_inline)) {
    const int key = min(tile * FA_BKV + lane, last), entry = p.c.page_size.quotient(key);
    place_of = key - entry * p.c.page_size.value;
    entry_of = table[entry];
  };
  auto find_rows = [&](int tile, int entry_of, int place_of) __attribute__((always_inline)) {
    const int page = (unsigned)entry_of < (unsigned)p.c.pages ? entry_of : 0;
    *reinterpret_cast<long*>(smem + ROWS_AT + (tile & 3) * 512 + lane * 8) = (long)Kh + p.c.k_at(page, place_of);
    *reinterpret_cast<long*>(smem + ROWS_AT + 2048 + (tile & 3) * 512 + lane * 8) = (long)Vh + p.c.v_at(page, place_of);
    if constexpr (CODES) scales_at = p.c.scale_at(page, place_of);
  };
  // The scales of a tile's 64 keys, of the tile whose rows were found last.
  auto load_scales = [&](int tile) __attribute__((always_inline)) {
    if (CODES && wave == 0) {
      const uint32_t to = __builtin_amdgcn_readfirstlane(lds0 + SCALE_AT + (tile & 3) * 256);
      gather4_to_lds(p.c.k_scale + h * p.c.s_head + scales_at, to);
      gather4_to_lds(p.c.v_scale + h * p.c.s_head + scales_at, to + 1024);
    }
  };
  uint4 k_reg[LD], v_reg[LD];                            // codes on their way
  auto load_k = [&](int tile, int stage) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < LD; ++q) {
      const char* from = reinterpret_cast<const char*>(*reinterpret_cast<const long*>(smem + ROWS_AT + (tile & 3) * 512 + row_at + q * (512 / PIECES)) + k_off[q]);
      if constexpr (CODES) {
        k_reg[q] = load_global16(from);
      } else {
        gather16_to_lds(from, __builtin_amdgcn_readfirstlane(lds0 + stage * TILE + (wave * LD + q) * 1024));
      }
    }
  };
  auto load_v = [&](int tile, int stage) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < LD; ++q) {
      const char* from = reinterpret_cast<const char*>(*reinterpret_cast<const long*>(smem + ROWS_AT + 2048 + (tile & 3) * 512 + row_at + q * (512 / PIECES)) + v_off[q]);
      if constexpr (CODES) {
        v_reg[q] = load_global16(from);
      } else {
        gather16_to_lds(from, __builtin_amdgcn_readfirstlane(lds0 + (2 + stage) * TILE + (wave * LD + q) * 1024));
      }
    }
  };
  // Codes: decode and write what load_k / load_v fetched.
  const bool spare = SPARE && wave * LD * 64 >= FA_BKV * PIECES;
  auto store_k = [&](int stage) __attribute__((always_inline)) {
    if constexpr (CODES) {
      if (spare) return;
#pragma unroll
      for (int q = 0; q < LD; ++q) {
        const uint32_t to = k_to ^ q * ROW_STEP * 16;
        lds_write_b128(smem, to + stage * TILE + q * ROW_STEP * ROWB, decode8<T, FMT>(make_uint2(k_reg[q].x, k_reg[q].y)));
        lds_write_b128(smem, (to ^ 16) + stage * TILE + q * ROW_STEP * ROWB, decode8<T, FMT>(make_uint2(k_reg[q].z, k_reg[q].w)));
      }
    }
  };
  auto store_v = [&](int stage) __attribute__((always_inline)) {
    if constexpr (CODES) {
      if (spare) return;
#pragma unroll
      for (int q = 0; q < LD; ++q) {
        lds_write_b128(smem, v_to + stage * TILE + q * ROW_STEP * ROWB, decode8<TV, FMT>(make_uint2(v_reg[q].x, v_reg[q].y)));
        lds_write_b128(smem, (v_to ^ 16) + stage * TILE + q * ROW_STEP * ROWB, decode8<TV, FMT>(make_uint2(v_reg[q].z, v_reg[q].w)));
      }
    }
  };

  // The pages of the first tiles, then Q: all of these loads are on their way together.
  int first_entry[2] = {}, first_place[2] = {};
  if (wave == 0 && ntiles > 0) {
#pragma unroll
    for (int i = 0; i < 2; ++i) find_page(tile_base + min(i, ntiles - 1), first_entry[i], first_place[i]);
  }
  // ---- Q fragments: lane (row l32, half lh) holds columns 16 ks + 8 lh .. + 7
  uint4 qf[KSTEPS];
  int klo, khi;
  {
    const int row = min(rw + l32, rows - 1), tok = token_of(row), hq = h * p.ratio.value + row - tok * p.ratio.value;
    const uint16_t* src = p.Q + (s.q0 + tok) * p.q_token + hq * p.q_head + 8 * lh;
#pragma unroll
    for (int ks = 0; ks < KSTEPS; ++ks)
      qf[ks] = 16 * ks < D ? *reinterpret_cast<const uint4*>(src + 16 * ks) : make_uint4(0u, 0u, 0u, 0u);
    key_bounds(tok, s.n, s.kv, p.causal, p.window, klo, khi);
  }

  // ---- state
  f32x16 o_acc[DT];
  float m_run = FA_NEG, l_run = 0.f;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) o_acc[dt][r] = 0.f;
  const float c = p.scale * 1.44269504088896340736f;
  const SoftCap cap = EXT ? SoftCap(p, EXT == 2) : SoftCap();
  const float cs = EXT ? cap.slope : c;                  // see folds()

  // ---- LDS read addresses: of step ks k_rd ^ 32 ks, of output columns 32 dt .. v_rd ^ 64 dt (chunk numbers are swizzled by
  // XOR, a row's chunks fill a power of two).  At DP 256 formed at each read: kept, they were what the compiler spilled, and a
  // reload waits for every load on its way (B 6, 65 tokens on 2329 keys, soft cap, 97 us kept, 57 so; int8 67 and 56).  At DP 128
  // they fit and forming them costs 11 %.
  const uint32_t k_rd = l32 * ROWB + ((lh ^ k_swizzle<ROWB>(l32)) << 4);
  uint32_t v_rd;
  {
    const int r16 = lane & 15, key = 4 * lh + (r16 >> 2), col = 16 * ((lane >> 4) & 1) + 4 * (r16 & 3);
    v_rd = 2 * TILE + key * ROWB + (((col >> 3) ^ v_swizzle<ROWB, false>(key)) << 4) + (col & 7) * 2;
  }
  auto here = [](uint32_t at) __attribute__((always_inline)) {
    if constexpr (DP == 256) asm volatile("" : "+v"(at));
    return at;
  };
  const char* scales = smem + G::SCALE_AT + 16 * lh;

  auto scores = [&](f32x16 (&sc)[KT], int stage) __attribute__((always_inline)) {
    const uint32_t at = here(k_rd);
#pragma unroll
    for (int ks = 0; ks < KSTEPS; ++ks)
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        const uint4 kf = lds_read_b128(smem, (at ^ 32 * ks) + stage * TILE + kt * 32 * ROWB);
        if (ks == 0) {
          f32x16 z;
#pragma unroll
          for (int r = 0; r < 16; ++r) z[r] = 0.f;
          sc[kt] = mfma_32x32x16<T>(kf, qf[ks], z);
        } else {
          sc[kt] = mfma_32x32x16<T>(kf, qf[ks], sc[kt]);
        }
      }
  };

  // The loads of step t: K and V of tile t + 1 into the stages that the step before released, the pages of tile t + 2.
  auto begin_loads = [&](int t, int par) __attribute__((always_inline)) {
    const int tile = tile_base + t;
    if (t + 1 < ntiles) {
      load_k(tile + 1, par ^ 1);
      load_v(tile + 1, par ^ 1);
      load_scales(tile + 1);
    }
    if (wave == 0 && t + 2 < ntiles) find_page(tile + 2, page_entry, page_place);
  };
  auto end_loads = [&](int t, int par) __attribute__((always_inline)) {
    if (t + 1 < ntiles) {
      store_k(par ^ 1);
      store_v(par ^ 1);
    }
    if (wave == 0 && t + 2 < ntiles) find_rows(tile_base + t + 2, page_entry, page_place);
    fa_wait_loads();
    __syncthreads();
  };

  // One tile.  (Forming the next tile's scores under this one's softmax, as the contiguous kernel does, gained nothing beside
  // two waves to a SIMD and cost the registers: B 4, 2048 tokens on 3000 keys 311 us with it, 301 without, e4m3 376 and 332.)
  auto step = [&](auto par_c, int t) __attribute__((always_inline)) {
    constexpr int PAR = decltype(par_c)::value;
    const int tile = tile_base + t;
    begin_loads(t, PAR);
    f32x16 sc[KT];
    scores(sc, PAR);
    const int kv0 = tile * FA_BKV;
    const char* ts = scales + (tile & 3) * 256;
    if constexpr (CODES) {
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          const float4 x = *reinterpret_cast<const float4*>(ts + kt * 128 + a * 32);
          sc[kt][4 * a + 0] *= x.x; sc[kt][4 * a + 1] *= x.y; sc[kt][4 * a + 2] *= x.z; sc[kt][4 * a + 3] *= x.w;
        }
    }
    if constexpr (EXT != 0) {
      if constexpr (EXT == 2) {
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int r = 0; r < 16; ++r) sc[kt][r] = far_exponent(sc[kt][r], c, cap.in, cap.top);
      } else if (p.softcap > 0.f) {
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int r = 0; r < 16; ++r) sc[kt][r] = cap.form(sc[kt][r]);
      } else {
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int r = 0; r < 16; ++r) sc[kt][r] *= c;
      }
    }
    if ((kv0 + FA_BKV - 1 > whi_first) || (kv0 < wlo_last)) {
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int key = kv0 + kt * 32 + 8 * (r >> 2) + 4 * lh + (r & 3);
          if (key > khi || key < klo) sc[kt][r] = FA_NEG;
        }
    }
    float mx = max3_raw(sc[0][0], sc[0][1], sc[0][2]);
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int r = (kt == 0 ? 3 : 0); r < 16; r += 2) mx = (r + 1 < 16) ? max3_raw(mx, sc[kt][r], sc[kt][r + 1]) : fmaxf(mx, sc[kt][r]);
    mx = max_with_other_half(mx);
    const float m_new = fmaxf(m_run, mx);
    if (__any(m_new > m_run)) {
      const float corr = fast_exp2((m_run - m_new) * cs);
      l_run *= corr;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o_acc[dt][r] *= corr;
      m_run = m_new;
    }
    // (a row that has met no visible key yet keeps the sentinel: reference 0, its masked entries underflow to P = 0)
    const float mc = m_new > 0.5f * FA_NEG ? fmaf(m_new, cs, -LIFT) : 0.f;
    constexpr int NU = 2 * KT, AHEAD = SPLIT ? 1 : 3;      // (units of P held before their product)
    uint4 pf[NU], pl[NU];
    float sum[2] = {0.f, 0.f};
    auto unit = [&](int i) __attribute__((always_inline)) {
      const int g = i & 1, kt = i >> 1;
#pragma unroll
      for (int r = 8 * g; r < 8 * g + 8; ++r) {
        const float e = fast_exp2(fmaf(sc[kt][r], cs, -mc));
        sc[kt][r] = e;
        sum[g] += e;
      }
      if constexpr (CODES) {
#pragma unroll
        for (int a = 2 * g; a < 2 * g + 2; ++a) {
          const float4 x = *reinterpret_cast<const float4*>(ts + 1024 + kt * 128 + a * 32);
          sc[kt][4 * a + 0] *= x.x; sc[kt][4 * a + 1] *= x.y; sc[kt][4 * a + 2] *= x.z; sc[kt][4 * a + 3] *= x.w;
        }
      }
      pf[i].x = pack2<TV>(sc[kt][8 * g + 0], sc[kt][8 * g + 1]);
      pf[i].y = pack2<TV>(sc[kt][8 * g + 2], sc[kt][8 * g + 3]);
      pf[i].z = pack2<TV>(sc[kt][8 * g + 4], sc[kt][8 * g + 5]);
      pf[i].w = pack2<TV>(sc[kt][8 * g + 6], sc[kt][8 * g + 7]);
      if constexpr (SPLIT) pl[i] = remainder8(sc[kt], 8 * g, pf[i]);
    };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) unit(i);
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      const int kt = i >> 1, g = i & 1;
      const uint32_t at = here(v_rd);
      uint4 vf[DT];
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const uint32_t a = (at ^ 64 * dt) + PAR * TILE + (kt * 32 + g * 16) * ROWB;
        const uint2 lo = lds_read_tr16_b64(smem + a);
        const uint2 hi = lds_read_tr16_b64(smem + a + 8 * ROWB);
        vf[dt] = make_uint4(lo.x, lo.y, hi.x, hi.y);
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        o_acc[dt] = mfma_32x32x16<TV>(vf[dt], pf[i], o_acc[dt]);
        if constexpr (SPLIT) o_acc[dt] = mfma_32x32x16<TV>(vf[dt], pl[i], o_acc[dt]);
      }
      if (i + AHEAD < NU) unit(i + AHEAD);
    }
    l_run += sum[0] + sum[1];
    end_loads(t, PAR);
  };
  using P0 = std::integral_constant<int, 0>;
  using P1 = std::integral_constant<int, 1>;

  // ---- prologue: the rows of tiles 0 and 1, then K(0), V(0)
  if (ntiles > 0) {
    if (wave == 0) {
      find_rows(tile_base, first_entry[0], first_place[0]);
      load_scales(tile_base);
      if (ntiles > 1) find_rows(tile_base + 1, first_entry[1], first_place[1]);
    }
    __syncthreads();
    load_k(tile_base, 0);
    load_v(tile_base, 0);
    store_k(0);
    store_v(0);
  }
  fa_wait_loads();
  __syncthreads();
  // A wave outside of its own range keeps the loads going.
  auto idle_step = [&](int t) __attribute__((always_inline)) {
    begin_loads(t, t & 1);
    end_loads(t, t & 1);
  };
  int t = 0;
  for (; t < t_w0; ++t) idle_step(t);                    // (t_w0 is even)
  for (; t + 2 <= nt_w; t += 2) {
    step(P0{}, t);
    step(P1{}, t + 1);
  }
  if (t < nt_w) {
    step(P0{}, t);
    ++t;
  }
  for (; t < ntiles; ++t) idle_step(t);

  // The arguments once more, through a pointer the compiler cannot see through: what only the end needs does not
  // occupy scalar registers during the walk (it spilled a hundred of them otherwise).
  const PagedTileParams late = late_params<PagedTileParams>();
  // ---- epilogue: a wave's 32 x D tile passes through its slice of the idle LDS, so that whole rows are stored
  const bool whole = late.nsplit == 1;
  const long total_rows = (long)late.p.total_q * late.p.Hq;
  float l = l_run + swap_half(l_run);
  if (khi < klo) l = 0.f;                                // no visible key: O = 0, LSE = -inf
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  float odd = 0.f;                                       // NaN where a value of the row is not finite
  char* stage = smem + wave * 32 * G::PITCH;
  const bool halves = whole && late.p.out_storage;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const int d = dt * 32 + 8 * a + 4 * lh;
      const float v0 = o_acc[dt][4 * a + 0] * inv, v1 = o_acc[dt][4 * a + 1] * inv;
      const float v2 = o_acc[dt][4 * a + 2] * inv, v3 = o_acc[dt][4 * a + 3] * inv;
      odd = fmaf(v0, 0.f, fmaf(v1, 0.f, fmaf(v2, 0.f, fmaf(v3, 0.f, odd))));
      if (halves) *reinterpret_cast<uint2*>(stage + l32 * G::PITCH + d * 2) = make_uint2(pack2<T>(v0, v1), pack2<T>(v2, v3));
      else *reinterpret_cast<float4*>(stage + l32 * G::PITCH + d * 4) = make_float4(v0, v1, v2, v3);
    }
  auto row_of = [&](int row, int& tok, int& hq) {
    tok = late.p.ratio.quotient(row);
    hq = h * late.p.ratio.value + row - tok * late.p.ratio.value;
  };
  if (lh == 0 && rw + l32 < rows) {
    int tok, hq;
    row_of(rw + l32, tok, hq);
    const float lse = l == 0.f ? -INFINITY : (m_run * cs + (cap.base - LIFT) + __log2f(l)) * 0.69314718055994530942f;
    const long at_row = (long)(s.q0 + tok) * late.p.Hq + hq;
    if (!whole) late.part_lse[split * total_rows + at_row] = lse;
    else if (late.p.LSE) late.p.LSE[at_row] = lse;
  }
  const int esz = halves ? 2 : 4, per_row = D * esz / 16, rows_here = min(32, rows - rw);
  for (int idx = lane; idx < rows_here * per_row; idx += 64) {
    const int r = idx / per_row, piece = idx - r * per_row;
    const uint4 v = *reinterpret_cast<const uint4*>(stage + r * G::PITCH + piece * 16);
    int tok, hq;
    row_of(rw + r, tok, hq);
    char* to = whole ? reinterpret_cast<char*>(late.p.O) + ((s.q0 + tok) * late.p.o_token + hq * late.p.o_head) * esz
                     : reinterpret_cast<char*>(late.part_o + (split * total_rows + (long)(s.q0 + tok) * late.p.Hq + hq) * D);
    *reinterpret_cast<uint4*>(to + piece * 16) = v;
  }
  if (whole) {
    // rows that a hidden key's value reached as 0 times something not finite, and those whose scores are all as low as the mask's
    // sentinel: again, from the keys they see
    unsigned long long mask = __ballot(!(odd == 0.f) || l == 0.f);
    mask = (mask | mask >> 32) & 0xffffffffull;
    while (mask) {
      const int r = __builtin_ctzll(mask);
      mask &= mask - 1;
      if (rw + r >= rows) break;
      int tok, hq;
      row_of(rw + r, tok, hq);
      paged_row<T, FMT>(late.p, b, s.q0 + tok, tok, s.n, s.kv, hq);
    }
  }
}

}  // namespace tsr950
