// What the kernels on a paged cache share: page lookup with its checks, and the rows of an e4m3 cache.
// Device code, but for the view.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../../include/qmm_decode.h"
#include "qmm_internal.h"

namespace qmm {

// A checked qmm_paged_cache as the kernels take it.
struct CacheView {
  uint8_t* k;
  uint8_t* v;
  uint8_t* k_exp;
  uint8_t* v_exp;
  const int32_t* table;
  int64_t table_stride;
  int64_t pages;
  int32_t table_width;
  int32_t page_shift;
  int32_t kv_heads;
};

__device__ __forceinline__ void report_index(int* status) { atomicCAS(status, 0, QMM_DEVICE_BAD_INDEX); }

// Page of a position, or -1 (reported): no such entry, or a page that the cache does not have.
__device__ __forceinline__ int64_t page_of(const CacheView& c, int seq, int pos, int* status) {
  const int entry = pos >> c.page_shift;
  if (pos < 0 || entry >= c.table_width) {
    report_index(status);
    return -1;
  }
  const int page = __ldg(c.table + seq * c.table_stride + entry);
  if (page < 0 || page >= c.pages) {
    report_index(status);
    return -1;
  }
  return page;
}

// ---- rows of an e4m3 cache ----
// The exponent e of a row whose largest magnitude is `big` (finite): the smallest whole number with big <= 448 * 2^e, 448 = 1.75 * 2^8.
__device__ __forceinline__ int row_exponent(float big) {
  const uint32_t bits = __float_as_uint(big);          // 1.m * 2^(x - 127); what is smaller than 2^-126 has a row of the least exponent
  const int e = static_cast<int>(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return bits == 0 ? 0 : e < -117 ? -117 : e > 119 ? 119 : e;
}

__device__ __forceinline__ uint32_t e4m3_pair(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// What turns a row's codes into bf16, as two factors (pairs of bf16): a code's bits as a bf16 are its value times 2^-120, subnormal codes
// among them (subnormal bf16 operands are taken as they are). The second factor is 1 but for rows above 57344.
struct RowFactors {
  uint32_t first, second;
};
__device__ __forceinline__ RowFactors row_factors(uint32_t exp_byte) {
  const int e = static_cast<int>(exp_byte) - 127;
  const int a = e > 7 ? 127 : 120 + e;
  const uint32_t f = exp_byte == 255 ? 0x7fc0u : static_cast<uint32_t>(a + 127) << 7;
  const uint32_t g = static_cast<uint32_t>((exp_byte != 255 && e > 7 ? e - 7 : 0) + 127) << 7;
  return {f | f << 16, g | g << 16};
}

__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// Sixteen codes -> sixteen bf16. Of a byte s eeee mmm the upper byte of the bf16 is s0000eee and the lower one emmm0000, made for four codes at a time.
__device__ __forceinline__ void row_values(const uint32_t (&codes)[4], const RowFactors& f, uint32_t (&out)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = codes[i], upper = ((w & 0x80808080u) | ((w >> 4) & 0x7f7f7f7fu)) & 0x87878787u, lower = (w << 4) & 0xf0f0f0f0u;
    out[2 * i] = mul_bf16x2(__byte_perm(upper, lower, 0x1504), f.first);
    out[2 * i + 1] = mul_bf16x2(__byte_perm(upper, lower, 0x3726), f.first);
  }
  if (f.second != 0x3f803f80u) {
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = mul_bf16x2(out[i], f.second);
  }
}

// ... without the power of two: code I of two words, as bf16 (2^120 brings the exponent there; subnormal codes among them), and as f16, which holds a code as it is.
template <int I>
__device__ __forceinline__ uint32_t code_pair(uint32_t a, uint32_t b) {
  const uint32_t x = __byte_perm(a, b, (4 + I) << 12 | I << 4);         // (what stands in the lower bytes is masked off)
  return mul_bf16x2(((x >> 4) & 0x07f007f0u) | (x & 0x80008000u), 0x7b807b80u);
}
__device__ __forceinline__ uint32_t code_half2(uint32_t two) {         // the lower two
  uint32_t h;
  asm("{ .reg .b16 l, u; mov.b32 {l, u}, %1; cvt.rn.f16x2.e4m3x2 %0, l; }" : "=r"(h) : "r"(two));
  return h;
}
template <int I>
__device__ __forceinline__ uint32_t code_half2(uint32_t a, uint32_t b) {
  return code_half2(__byte_perm(a, b, (4 + I) << 4 | I));
}
__device__ __forceinline__ float row_scale(uint32_t exp_byte) {
  return __uint_as_float(exp_byte == 255 ? 0x7fc00000u : exp_byte == 0 ? 0x00400000u : exp_byte << 23);
}

// ---- 16-bit floats ----
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

}  // namespace qmm
