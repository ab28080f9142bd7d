// Attention of a ragged batch of new tokens over a paged cache: what its kernels share.
#pragma once
#include "flash_attn.h"
#include "kv_cache.h"

namespace tsr950 {

struct PagedParams {
  KvCache c;
  const uint16_t* Q;                    // (total_q, Hq, D) through q_token, q_head
  void* O;                              // the same through o_token, o_head; f32 or the storage type
  float* LSE;                           // [total_q, Hq] or null
  long q_token, q_head, o_token, o_head;
  const int* table;                     // [B, pages_per_seq]
  const int* q_offsets;                 // [B + 1]
  const int* kv_lens;                   // [B]
  int pages_per_seq, B, Hq, total_q, max_q, max_kv;
  Divisor ratio;                        // Hq / heads
  float scale, softcap;
  int causal, window, out_storage;
};

// One sequence of the batch: its new tokens are rows q0 .. q0 + n - 1 of Q, its keys 0 .. kv - 1.  Device values are held
// to the bounds the host was given, so that no index leaves the arrays.
struct PagedSeq {
  int q0, n, kv;
};
__device__ __forceinline__ PagedSeq paged_seq(const PagedParams& p, int b) {
  PagedSeq s;
  s.q0 = min(max(p.q_offsets[b], 0), p.total_q);
  s.n = min(max(min(p.q_offsets[b + 1], p.total_q) - s.q0, 0), p.max_q);
  s.kv = min(max(p.kv_lens[b], 0), p.max_kv);
  return s;
}

// The kernel's arguments (a single struct) read again from where the launch put them.
template <class P> __device__ __forceinline__ P late_params() {
  uint64_t at = (uint64_t)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(at));
  P p;
  const auto* from = (const __attribute__((address_space(4))) uint32_t*)at;
  static_assert(sizeof(P) % 4 == 0, "dwords");
  uint32_t words[sizeof(P) / 4];
#pragma unroll
  for (unsigned i = 0; i < sizeof(P) / 4; ++i) words[i] = from[i];
  __builtin_memcpy(&p, words, sizeof(P));
  return p;
}

// Whether the scale may be folded into the exponential, the running maximum being taken over the raw scores: no soft cap,
// and a scale that leaves the mask's sentinel far below every score.
__host__ __device__ inline bool folds(const PagedParams& p) { return p.scale > 1e-6f && !(p.softcap > 0.f); }

// The soft cap  cap tanh(scale s / cap) = cap - 2 cap / (1 + e^(2 scale s / cap)): a walk carries form(s) = -1 / (1 + ..), whose
// multiplier 2 cap log2(e) goes into the exponential's FMA and whose constant only the LSE needs (base).  B 4, 2048 tokens on
// 3000 keys, cap 30: 457 us with those two FMAs in the walk, 433 without; and 357 with the choice between cap and plain scale made once a
// tile, not at each score (296 without a cap).  A cap under 1e-8 is one of 1e-8, no score being off by
// more than that: the mask's sentinel times the slope has to stay far below every score.  Caps over kPlainCap (far): the walk carries the
// exponent itself, from far_exponent.
struct SoftCap {
  float in = 0.f, top = 0.f, slope = 1.0f, base = 0.f;
  __device__ __forceinline__ SoftCap() {}
  __device__ __forceinline__ SoftCap(const PagedParams& p, bool far) {
    if (!(p.softcap > 0.f)) return;
    const float cap = far ? fminf(p.softcap, 2.0e38f) : fmaxf(p.softcap, 1e-8f);
    in = 2.0f * 1.44269504088896340736f * p.scale / cap;
    top = 1.44269504088896340736f * cap;
    if (far) return;
    slope = 2.0f * top;
    base = top;
  }
  __device__ __forceinline__ float form(float s) const { return __builtin_amdgcn_rcpf(-1.0f - __builtin_amdgcn_exp2f(s * in)); }
};

// The page of a table entry, one of the cache's whatever the entry says.
__device__ __forceinline__ int paged_page(const PagedParams& p, int b, int entry) {
  const int page = p.table[(long)b * p.pages_per_seq + entry];
  return (unsigned)page < (unsigned)p.c.pages ? page : 0;
}

// One new token and query head by one wave, from the definition: 64 keys at a time, a lane forms one key's score in f32,
// the running maximum and sum are reductions over the wave, and each lane sums every 64th column of the output. 
template <class T, int FMT>
__device__ __forceinline__ void paged_row(const PagedParams& p, int b, int token, int i, int n, int kv, int hq) {
  const int lane = threadIdx.x & 63, h = p.ratio.quotient(hq), D = p.c.D;
  int lo, hi;
  key_bounds(i, n, kv, p.causal, p.window, lo, hi);
  const uint16_t* q = p.Q + token * p.q_token + hq * p.q_head;
  float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int k0 = lo; k0 <= hi; k0 += 64) {
    const int key = k0 + lane;
    float x = -INFINITY, vs = 0.f;
    long v_at = 0;
    if (key <= hi) {
      const int entry = p.c.page_size.quotient(key), place = key - entry * p.c.page_size.value, page = paged_page(p, b, entry);
      const char* kp = p.c.k + p.c.k_at(page, place) + h * p.c.k_head;
      v_at = p.c.v_at(page, place) + h * p.c.v_head;
      float dot = 0.f;
      if constexpr (FMT == kStorage) {
        for (int d = 0; d < D; ++d) dot += from_storage<T>(q[d]) * from_storage<T>(reinterpret_cast<const uint16_t*>(kp)[d]);
      } else {
        for (int d = 0; d < D; d += 4) {
          const float4 c = decode4<FMT>(*reinterpret_cast<const uint32_t*>(kp + d));
          dot += from_storage<T>(q[d]) * c.x + from_storage<T>(q[d + 1]) * c.y + from_storage<T>(q[d + 2]) * c.z +
                 from_storage<T>(q[d + 3]) * c.w;
        }
        const long at = p.c.scale_at(page, place) + h * p.c.s_head;
        dot *= p.c.k_scale[at];
        vs = p.c.v_scale[at];
      }
      x = dot * p.scale;
      if (p.softcap > 0.f) x = p.softcap * tanhf(x / p.softcap);
    }
    float mn = x;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mn = fmaxf(mn, __shfl_xor(mn, o, 64));
    mn = fmaxf(mn, m);
    const float ref = mn > -INFINITY ? mn : 0.f;
    const float e = __expf(x - ref);
    float sum = e;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    const float corr = __expf(m - ref);
    l = l * corr + sum;
#pragma unroll
    for (int c = 0; c < 4; ++c) acc[c] *= corr;
    m = mn;
    const int keys = min(64, hi - k0 + 1);
    for (int j = 0; j < keys; ++j) {
      const float w = __shfl(FMT == kStorage ? e : e * vs, j, 64);
      const long at = ((long)__shfl((int)(v_at >> 32), j, 64) << 32) | (unsigned)__shfl((int)v_at, j, 64);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int d = lane + 64 * c;
        if (d >= D) continue;
        float v;
        if constexpr (FMT == kStorage) v = from_storage<T>(reinterpret_cast<const uint16_t*>(p.c.v + at)[d]);
        else v = decode4<FMT>(reinterpret_cast<const uint8_t*>(p.c.v + at)[d]).x;
        acc[c] += w * v;
      }
    }
  }
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int d = lane + 64 * c;
    if (d >= D) continue;
    const float o = l == 0.f ? 0.f : acc[c] / l;
    const long at = token * p.o_token + hq * p.o_head + d;
    if (p.out_storage) reinterpret_cast<uint16_t*>(p.O)[at] = to_storage<T>(o);
    else reinterpret_cast<float*>(p.O)[at] = o;
  }
  if (p.LSE && lane == 0) p.LSE[(long)token * p.Hq + hq] = l == 0.f ? -INFINITY : m + __logf(l);
}

}  // namespace tsr950
