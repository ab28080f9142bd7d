// C ABI: writing new tokens' K and V into a paged cache and reading slots back.
#include <algorithm>
#include "kv_cache.h"
#include "host_util.h"

namespace tsr950 {
namespace {

// Contiguous sides of a copy: element (t, h, d) of K at t * k_token + h * k_head + d.
struct Rows {
  long k_token, k_head, v_token, v_head;       // elements
};

// x / scale, correctly rounded, from the correctly rounded reciprocal: the product is off by less than two units in the last
// place, one step q + (x - q scale) / scale with the remainder exact in an FMA brings it within one, a second one to the
// nearest (Markstein, IBM Journal of Research and Development 34, 1990).  Exact remainders need |x| > 2^-100 or so, the
// nearest quotient one that is normal: below, the code is zero either way (scale >= 1e-12).  The compiler's own division
// takes twice the instructions, and they bounded the kernel: 8192 tokens x 8 heads x 128 into int8 14.4 -> 12.8 us.
__device__ __forceinline__ float divide(float x, float scale, float reciprocal) {
  float q = x * reciprocal;
  q = fmaf(fmaf(-q, scale, x), reciprocal, q);
  return fmaf(fmaf(-q, scale, x), reciprocal, q);
}

// Codes and scale of a row held by G lanes, 8 values each (zeros past its end).  The maximum is taken over the magnitudes' bit
// patterns, which order as the magnitudes do and put a NaN on top: a row that holds an infinity or a NaN gets a scale that
// is not finite, and nothing finite is read back from it.
template <class T, int FMT, int G>
__device__ __forceinline__ uint2 quantise_row(const uint4& x, float& scale) {
  typedef __attribute__((ext_vector_type(2))) unsigned short u16x2;
  auto magnitudes = [](uint32_t w) { return __builtin_bit_cast(u16x2, w & 0x7fff7fffu); };
  const u16x2 m = __builtin_elementwise_max(__builtin_elementwise_max(magnitudes(x.x), magnitudes(x.y)),
                                            __builtin_elementwise_max(magnitudes(x.z), magnitudes(x.w)));
  unsigned top = m[0] > m[1] ? m[0] : m[1];
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) {
    const unsigned other = __shfl_xor(top, o, 64);
    top = top > other ? top : other;
  }
  constexpr float TOP = FMT == kInt8 ? 127.0f : 448.0f;
  scale = from_storage<T>((uint16_t)top) * (1.0f / TOP);
  if (scale < 1e-12f) scale = 1e-12f;                                     // (a NaN stays)
  const float reciprocal = __fdiv_rn(1.0f, scale);
  const uint32_t in[4] = {x.x, x.y, x.z, x.w};
  uint32_t out[2];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    float q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint16_t bits = (uint16_t)(in[2 * w + i / 2] >> (16 * (i & 1)));
      q[i] = fminf(fmaxf(divide(from_storage<T>(bits), scale, reciprocal), -TOP), TOP);
    }
    if constexpr (FMT == kInt8) {
      uint32_t packed = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) packed |= (uint32_t)(uint8_t)(int8_t)__builtin_rintf(q[i]) << (8 * i);
      out[w] = packed;
    } else {
      const int packed = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
      out[w] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], packed, true);
    }
  }
  return make_uint2(out[0], out[1]);
}

// One (token, head) row of K and of V by G lanes, 8 values each; G is the power of two at or over D / 8, so that a row's
// maximum is a reduction inside G neighbouring lanes.  Bound by memory: both rows are on their way together.
template <class T, int FMT, int G>
__global__ __launch_bounds__(256) void kv_write_kernel(const KvCache c, const uint16_t* __restrict__ k,
                                                       const uint16_t* __restrict__ v, const Rows src,
                                                       const int64_t* __restrict__ slots, const Divisor heads, int rows) {
  const int sub = threadIdx.x & (G - 1);
  const int row = blockIdx.x * (256 / G) + threadIdx.x / G;
  if (row >= rows) return;
  const int t = heads.quotient(row), h = row - t * heads.value;
  const int64_t slot = slots[t];
  const bool on = 8 * sub < c.D;
  uint4 x = make_uint4(0u, 0u, 0u, 0u), y = x;
  if (on) {
    x = *reinterpret_cast<const uint4*>(k + t * src.k_token + h * src.k_head + 8 * sub);
    y = *reinterpret_cast<const uint4*>(v + t * src.v_token + h * src.v_head + 8 * sub);
  }
  if (slot < 0 || slot >= (int64_t)c.pages * c.page_size.value) return;   // (the row's lanes leave together)
  const int page = c.page_size.quotient((int)slot), place = (int)slot - page * c.page_size.value;
  char* k_to = c.k + c.k_at(page, place) + h * c.k_head;
  char* v_to = c.v + c.v_at(page, place) + h * c.v_head;
  if constexpr (FMT == kStorage) {
    if (!on) return;
    *reinterpret_cast<uint4*>(k_to + 16 * sub) = x;
    *reinterpret_cast<uint4*>(v_to + 16 * sub) = y;
  } else {
    float k_scale, v_scale;
    const uint2 kc = quantise_row<T, FMT, G>(x, k_scale), vc = quantise_row<T, FMT, G>(y, v_scale);
    if (sub == 0) {
      const long at = c.scale_at(page, place) + h * c.s_head;
      c.k_scale[at] = k_scale;
      c.v_scale[at] = v_scale;
    }
    if (!on) return;
    *reinterpret_cast<uint2*>(k_to + 8 * sub) = kc;
    *reinterpret_cast<uint2*>(v_to + 8 * sub) = vc;
  }
}

// The way back: f32(code) * scale, rounded once to the storage type; zeros for a slot outside the cache.
template <class T, int FMT, int G>
__global__ __launch_bounds__(256) void kv_read_kernel(const KvCache c, uint16_t* __restrict__ k, uint16_t* __restrict__ v,
                                                      const Rows dst, const int64_t* __restrict__ slots,
                                                      const Divisor heads, int rows) {
  const int sub = threadIdx.x & (G - 1);
  const int row = blockIdx.x * (256 / G) + threadIdx.x / G;
  if (row >= rows || 8 * sub >= c.D) return;
  const int t = heads.quotient(row), h = row - t * heads.value;
  const int64_t slot = slots[t];
  uint4 x = make_uint4(0u, 0u, 0u, 0u), y = x;
  if (slot >= 0 && slot < (int64_t)c.pages * c.page_size.value) {
    const int page = c.page_size.quotient((int)slot), place = (int)slot - page * c.page_size.value;
    const char* k_from = c.k + c.k_at(page, place) + h * c.k_head;
    const char* v_from = c.v + c.v_at(page, place) + h * c.v_head;
    if constexpr (FMT == kStorage) {
      x = *reinterpret_cast<const uint4*>(k_from + 16 * sub);
      y = *reinterpret_cast<const uint4*>(v_from + 16 * sub);
    } else {
      const uint2 kc = *reinterpret_cast<const uint2*>(k_from + 8 * sub), vc = *reinterpret_cast<const uint2*>(v_from + 8 * sub);
      const long at = c.scale_at(page, place) + h * c.s_head;
      const float k_scale = c.k_scale[at], v_scale = c.v_scale[at];
      auto values = [](const uint2& codes, float scale) {
        const float4 a = decode4<FMT>(codes.x), b = decode4<FMT>(codes.y);
        return make_uint4(pack2<T>(a.x * scale, a.y * scale), pack2<T>(a.z * scale, a.w * scale), pack2<T>(b.x * scale, b.y * scale),
                          pack2<T>(b.z * scale, b.w * scale));
      };
      x = values(kc, k_scale);
      y = values(vc, v_scale);
    }
  }
  *reinterpret_cast<uint4*>(k + t * dst.k_token + h * dst.k_head + 8 * sub) = x;
  *reinterpret_cast<uint4*>(v + t * dst.v_token + h * dst.v_head + 8 * sub) = y;
}

// The contiguous side: strides in elements on the 16-byte grid, rows that do not overlap where they are written.
bool bad_rows(const void* k, const void* v, const int64_t* st, int D, int T, int heads, bool written) {
  if (!k || !v || !st || ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15)) return true;
  for (int i = 0; i < 4; ++i) {
    if (st[i] < 0 || st[i] % 8) return true;
    if (written && (i & 1 ? heads : T) > 1 && st[i] < D) return true;
  }
  return false;
}

template <class T, int FMT, int G>
int launch_rows(bool write, const KvCache& c, const void* k, const void* v, const Rows& r, const int64_t* slots, int rows,
                hipStream_t s) {
  const dim3 grid((unsigned)ceil_div(rows, 256 / G));
  const Divisor heads(c.heads);
  if (write) {
    hipLaunchKernelGGL((kv_write_kernel<T, FMT, G>), grid, dim3(256), 0, s, c, static_cast<const uint16_t*>(k),
                       static_cast<const uint16_t*>(v), r, slots, heads, rows);
  } else {
    hipLaunchKernelGGL((kv_read_kernel<T, FMT, G>), grid, dim3(256), 0, s, c,
                       static_cast<uint16_t*>(const_cast<void*>(k)), static_cast<uint16_t*>(const_cast<void*>(v)), r, slots,
                       heads, rows);
  }
  return launch_status();
}
template <class T, int FMT>
int launch_rows_for(bool write, const KvCache& c, const void* k, const void* v, const Rows& r, const int64_t* slots,
                    int rows, hipStream_t s) {
  if (c.D <= 64) return launch_rows<T, FMT, 8>(write, c, k, v, r, slots, rows, s);
  if (c.D <= 128) return launch_rows<T, FMT, 16>(write, c, k, v, r, slots, rows, s);
  return launch_rows<T, FMT, 32>(write, c, k, v, r, slots, rows, s);
}

template <class T>
int cache_rows(bool write, const tessera_gfx950_kv_cache* cache, const void* k, const void* v, const int64_t* strides,
               const int64_t* slots, int tokens, void* stream) {
  if (bad_cache(cache) || tokens < 0 || (write && overlapping_cache(*cache))) return kBadShape;
  if (tokens == 0) return probe_device();
  if (!slots || bad_rows(k, v, strides, cache->head_dim, tokens, cache->num_heads, !write)) return kBadShape;
  // (rows are 32-bit numbers, and so are a launch's threads, up to 32 for a row)
  const int64_t rows64 = (int64_t)tokens * cache->num_heads;
  if (rows64 > 0x7fffff00 || rows64 * (cache->head_dim <= 64 ? 8 : cache->head_dim <= 128 ? 16 : 32) > 0xffffff00) return kBadShape;
  if (int rc = probe_device(); rc != kOk) return rc;
  const KvCache c = device_view(*cache);
  const Rows r{(long)strides[0], (long)strides[1], (long)strides[2], (long)strides[3]};
  const int rows = (int)rows64;
  switch (cache->format) {
    case kStorage: return launch_rows_for<T, kStorage>(write, c, k, v, r, slots, rows, as_stream(stream));
    case kInt8: return launch_rows_for<T, kInt8>(write, c, k, v, r, slots, rows, as_stream(stream));
    default: return launch_rows_for<T, kE4m3>(write, c, k, v, r, slots, rows, as_stream(stream));
  }
}

}  // namespace
}  // namespace tsr950

using namespace tsr950;

extern "C" {

int tessera_gfx950_kv_cache_write_f16_dev(const tessera_gfx950_kv_cache* cache, const void* K, const void* V,
                                          const int64_t* strides, const int64_t* slots, int T, void* stream) {
  return cache_rows<F16>(true, cache, K, V, strides, slots, T, stream);
}
int tessera_gfx950_kv_cache_write_bf16_dev(const tessera_gfx950_kv_cache* cache, const void* K, const void* V,
                                           const int64_t* strides, const int64_t* slots, int T, void* stream) {
  return cache_rows<BF16>(true, cache, K, V, strides, slots, T, stream);
}
int tessera_gfx950_kv_cache_read_f16_dev(const tessera_gfx950_kv_cache* cache, const int64_t* slots, void* K, void* V,
                                         const int64_t* strides, int T, void* stream) {
  return cache_rows<F16>(false, cache, K, V, strides, slots, T, stream);
}
int tessera_gfx950_kv_cache_read_bf16_dev(const tessera_gfx950_kv_cache* cache, const int64_t* slots, void* K, void* V,
                                          const int64_t* strides, int T, void* stream) {
  return cache_rows<BF16>(false, cache, K, V, strides, slots, T, stream);
}

}  // extern "C"
