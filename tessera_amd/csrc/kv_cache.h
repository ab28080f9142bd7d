// The paged key/value cache: how a kernel finds a token's row, and the 8-bit formats.
//
// K and V are each `pages` pages of `page_size` slots with `heads` rows of D values; any order of the three outer
// dimensions is served through strides.  Format kStorage holds 16-bit values; kInt8 and kE4m3 hold codes with one f32
// scale for each (slot, head): value = code * scale.
#pragma once
#include <algorithm>
#include <type_traits>
#include "../../include/tessera_gfx950.h"
#include "common.h"

namespace tsr950 {

constexpr int kStorage = 0, kInt8 = 1, kE4m3 = 2;

// t / divisor for 0 <= t < 2^31 as a multiplication: with 2^l the power of two not under the divisor and
// mul = ceil(2^(31 + l) / divisor), t * mul / 2^(31 + l) passes the true quotient by less than t / 2^31 / divisor, which is
// too little to reach the next whole number.
struct Divisor {
  uint32_t mul;
  int shift;       // -1: the divisor is 1
  int value;
  Divisor() = default;
  explicit Divisor(int d) : mul(0), shift(-1), value(d) {
    if (d <= 1) return;
    int l = 1;
    while ((1u << l) < (uint32_t)d) ++l;
    mul = (uint32_t)(((1ull << (31 + l)) + (uint32_t)d - 1) / (uint32_t)d);
    shift = l - 1;
  }
  __device__ __forceinline__ int quotient(int t) const { return shift < 0 ? t : (int)(__umulhi((uint32_t)t, mul) >> shift); }
};

struct KvCache {
  char *k, *v;
  float *k_scale, *v_scale;
  uint32_t k_page, k_slot, v_page, v_slot;                  // bytes, below 2^31
  long k_head, v_head;
  uint32_t s_page, s_slot;                                  // elements of both scale arrays
  long s_head;
  int pages, heads, D;
  Divisor page_size;

  __device__ __forceinline__ long k_at(int page, int place) const {
    return (long)((uint64_t)(uint32_t)page * k_page + (uint64_t)(uint32_t)place * k_slot);
  }
  __device__ __forceinline__ long v_at(int page, int place) const {
    return (long)((uint64_t)(uint32_t)page * v_page + (uint64_t)(uint32_t)place * v_slot);
  }
  __device__ __forceinline__ long scale_at(int page, int place) const {
    return (long)((uint64_t)(uint32_t)page * s_page + (uint64_t)(uint32_t)place * s_slot);
  }
};

inline KvCache device_view(const tessera_gfx950_kv_cache& c) {
  const int esz = c.format == kStorage ? 2 : 1;
  KvCache d{};
  d.k = static_cast<char*>(c.k);
  d.v = static_cast<char*>(c.v);
  d.k_scale = c.k_scale;
  d.v_scale = c.v_scale;
  d.k_page = (uint32_t)(c.k_strides[0] * esz); d.k_slot = (uint32_t)(c.k_strides[1] * esz); d.k_head = c.k_strides[2] * esz;
  d.v_page = (uint32_t)(c.v_strides[0] * esz); d.v_slot = (uint32_t)(c.v_strides[1] * esz); d.v_head = c.v_strides[2] * esz;
  d.s_page = (uint32_t)c.scale_strides[0]; d.s_slot = (uint32_t)c.scale_strides[1]; d.s_head = c.scale_strides[2];
  d.pages = c.num_pages;
  d.heads = c.num_heads;
  d.D = c.head_dim;
  d.page_size = Divisor(c.page_size);
  return d;
}

// Whether a cache cannot be served: sizes, the 16-byte grid of rows and pointers (every row is moved 16 or 8 bytes at a
// time), strides under a row (whether rows overlap otherwise matters to a write: rows_overlap), strides of 2 GiB and more (a page's and a slot's offsets are 32 by 32 bit products).  Slot
// numbers fit 31 bits.
inline bool bad_cache(const tessera_gfx950_kv_cache* c) {
  if (!c || !c->k || !c->v || c->format < kStorage || c->format > kE4m3) return true;
  if (c->num_pages <= 0 || c->page_size <= 0 || c->num_heads <= 0) return true;
  if ((int64_t)c->num_pages * c->page_size > 0x7fffffff) return true;
  if (c->head_dim <= 0 || c->head_dim % 16 != 0 || c->head_dim > 256) return true;
  const int per16 = c->format == kStorage ? 8 : 16;         // elements in 16 bytes
  if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15) return true;
  const int size[3] = {c->num_pages, c->page_size, c->num_heads};
  const int64_t most = 0x7fffffff / (c->format == kStorage ? 2 : 1);
  for (int i = 0; i < 3; ++i) {
    if (c->k_strides[i] > most || c->v_strides[i] > most) return true;
    if (c->k_strides[i] < 0 || c->v_strides[i] < 0 || c->k_strides[i] % per16 || c->v_strides[i] % per16) return true;
    if (size[i] > 1 && (c->k_strides[i] < c->head_dim || c->v_strides[i] < c->head_dim)) return true;
  }
  if (c->format == kStorage) return false;
  if (!c->k_scale || !c->v_scale) return true;
  if ((reinterpret_cast<uintptr_t>(c->k_scale) | reinterpret_cast<uintptr_t>(c->v_scale)) & 3) return true;
  for (int i = 0; i < 3; ++i)
    if (c->scale_strides[i] < 0 || c->scale_strides[i] > 0x7fffffff || (size[i] > 1 && c->scale_strides[i] < 1)) return true;
  return false;
}

// Whether rows of `width` elements share elements: taken by their strides, each has to be at least what the smaller ones span.  (Orders that
// interleave without that, strides 2 and 3 of two each, are taken to overlap.)
inline bool rows_overlap(const int64_t strides[3], const int size[3], int width) {
  int order[3] = {0, 1, 2};
  std::sort(order, order + 3, [&](int a, int b) { return strides[a] < strides[b]; });
  int64_t span = width;
  for (int i : order) {
    if (size[i] == 1) continue;
    if (strides[i] < span) return true;
    span += strides[i] * (size[i] - 1);                  // (under 2^31 before the last, 2^62 there)
  }
  return false;
}
// Whether a write to a cache that is not bad would put rows, or scales, on top of each other.
inline bool overlapping_cache(const tessera_gfx950_kv_cache& c) {
  const int size[3] = {c.num_pages, c.page_size, c.num_heads};
  return rows_overlap(c.k_strides, size, c.head_dim) || rows_overlap(c.v_strides, size, c.head_dim) ||
         (c.format != kStorage && rows_overlap(c.scale_strides, size, 1));
}

// Four codes (one dword) as f32.
template <int FMT> __device__ __forceinline__ float4 decode4(uint32_t w) {
  if constexpr (FMT == kInt8) {
    return make_float4((float)(int8_t)(w), (float)(int8_t)(w >> 8), (float)(int8_t)(w >> 16), (float)(int8_t)(w >> 24));
  } else {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    return make_float4(lo[0], lo[1], hi[0], hi[1]);
  }
}

// Eight codes as eight values of the 16-bit type T: exact, as e4m3 numbers and the whole numbers to 128 have at most 8
// significant bits and lie in the normal range of both types.  e4m3 by the packed conversion with scale 1.
template <class T, int FMT> __device__ __forceinline__ uint4 decode8(uint2 w) {
  if constexpr (FMT == kE4m3) {
    auto two = [](uint32_t c, auto high) -> uint32_t {
      if constexpr (std::is_same<T, BF16>::value)
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, 1.0f, decltype(high)::value));
      else
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c, 1.0f, decltype(high)::value));
    };
    return make_uint4(two(w.x, std::false_type{}), two(w.x, std::true_type{}), two(w.y, std::false_type{}), two(w.y, std::true_type{}));
  } else {
    const float4 a = decode4<kInt8>(w.x), b = decode4<kInt8>(w.y);
    return make_uint4(pack2<T>(a.x, a.y), pack2<T>(a.z, a.w), pack2<T>(b.x, b.y), pack2<T>(b.z, b.w));
  }
}

}  // namespace tsr950
