// What the kernels of the paged cache share: where a token lies, and the 4-bit values.
#pragma once

#include <cuda_fp16.h>
#include <string.h>

#include "common.cuh"

namespace bma {

constexpr int kStatusAppend = 801, kStatusRead = 802, kStatusPaged = 803;   // a position outside the table, or a page outside the cache
constexpr int kPagedHeadDim = 128;

// Page and slot of position `pos` of sequence b; page -1 where the table does not cover it or names no page of the cache.
__device__ __forceinline__ int page_of(const bma_paged_cache& c, int b, int64_t pos, int& slot) {
  if (pos < 0 || pos >= (int64_t)c.width * c.page_size) return -1;
  const int i = (int)pos / c.page_size;   // (width * page_size < 2^31, checked on the host)
  slot = (int)pos - i * c.page_size;
  const int page = __ldg(c.page_table + (int64_t)b * c.table_stride + i);
  return page >= 0 && page < c.pages ? page : -1;
}

// The newest tokens of sequence b that are real, of the T given, and the position of the first.
struct NewTokens {
  int count;
  int64_t first;
};
__device__ __forceinline__ NewTokens new_tokens(const int32_t* lengths, const int32_t* new_lengths, int b, int T) {
  const int64_t len = __ldg(lengths + b);
  int n = new_lengths ? min(max(__ldg(new_lengths + b), 0), T) : T;
  return {n, len - n};
}

// ---- e2m1 ---------------------------------------------------------------------------------------------------------------
// Two values as a byte, to the nearest, ties to the even code, at most 6; `lo` goes into the lower half.
__device__ __forceinline__ uint32_t to_e2m1x2(float lo, float hi) {
  uint16_t r;
  asm("{ .reg .b8 b; cvt.rn.satfinite.e2m1x2.f32 b, %1, %2; mov.b16 %0, {b, 0}; }" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// The four pairs of values of eight codes, as half2: r[i] = values 2i and 2i + 1.
__device__ __forceinline__ void from_e2m1x8(uint32_t codes, uint32_t (&r)[4]) {
  asm("{ .reg .b8 a, b, c, d;\n mov.b32 {a, b, c, d}, %4;\n cvt.rn.f16x2.e2m1x2 %0, a;\n cvt.rn.f16x2.e2m1x2 %1, b;\n"
      " cvt.rn.f16x2.e2m1x2 %2, c;\n cvt.rn.f16x2.e2m1x2 %3, d; }"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(codes));
}
// 2^(byte - 127); 255 is NaN, 0 the subnormal 2^-127
__device__ __forceinline__ float e8m0_value(uint32_t byte) {
  return byte == 255 ? __uint_as_float(0x7fffffffu) : byte == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23);
}

// Host-side checks of a cache description.
inline int validate_cache(const bma_paged_cache* c) {
  BMA_REQUIRE(c && c->k && c->v && c->page_table, BMA_ERR_ARG);
  BMA_REQUIRE(c->pages > 0 && c->page_size > 0 && c->Hkv > 0 && c->d > 0 && c->B > 0 && c->width > 0, BMA_ERR_ARG);
  BMA_REQUIRE(c->dtype == BMA_DTYPE_F32 || c->dtype == BMA_DTYPE_BF16 || c->dtype == BMA_DTYPE_MXFP4, BMA_ERR_UNSUPPORTED);
  BMA_REQUIRE(c->d <= kPagedHeadDim && c->d % (c->dtype == BMA_DTYPE_MXFP4 ? 32 : 8) == 0, BMA_ERR_UNSUPPORTED);
  BMA_REQUIRE((int64_t)c->width * c->page_size < (1ll << 31) - 4096 && c->B <= 65535 && c->Hkv <= 65535, BMA_ERR_LIMIT);
  const int64_t unit = c->dtype == BMA_DTYPE_F32 ? 4 : c->dtype == BMA_DTYPE_BF16 ? 8 : 16;   // rows start on 16 bytes: copies are that wide
  BMA_REQUIRE(((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15) == 0, BMA_ERR_UNSUPPORTED);
  BMA_REQUIRE(c->stride_page % unit == 0 && c->stride_slot % unit == 0 && c->stride_head % unit == 0, BMA_ERR_UNSUPPORTED);
  BMA_REQUIRE(c->stride_page >= 0 && c->stride_slot >= 0 && c->stride_head >= 0, BMA_ERR_ARG);      // (negative offsets stand for no place)
  BMA_REQUIRE(c->dtype != BMA_DTYPE_MXFP4 || (c->k_scale && c->v_scale), BMA_ERR_ARG);
  BMA_REQUIRE(c->dtype != BMA_DTYPE_MXFP4 || (c->scale_stride_page >= 0 && c->scale_stride_slot >= 0 && c->scale_stride_head >= 0), BMA_ERR_ARG);
  return BMA_OK;
}

}  // namespace bma
