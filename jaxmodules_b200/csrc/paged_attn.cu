// Attention of the newest tokens of every sequence over a paged cache.
#include "paged.cuh"

namespace bma {
namespace {

constexpr int kRows = 16, kKeys = 32;

__device__ __forceinline__ float held_value(const bma_paged_cache& c, bool v, int64_t at, int64_t scale_at, int h, int i) {
  const void* p = v ? c.v : c.k;
  if (c.dtype == BMA_DTYPE_F32) return static_cast<const float*>(p)[at + h * c.stride_head + i];
  if (c.dtype == BMA_DTYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[at + h * c.stride_head + i]);
  const uint8_t code = static_cast<const uint8_t*>(p)[at + h * c.stride_head + i / 2] >> (i & 1 ? 4 : 0);
  uint32_t pairs[4];
  from_e2m1x8(code & 15, pairs);
  return __low2float(*reinterpret_cast<const __half2*>(&pairs[0])) * e8m0_value((v ? c.v_scale : c.k_scale)[scale_at + h * c.scale_stride_head + i / 32]);
}

// One CTA: a sequence, a kv head, and up to 16 of the rows (token, query head of the group), one pass over the keys.
__global__ void __launch_bounds__(128) paged_rows_kernel(const __grid_constant__ bma_paged_cache c, const __grid_constant__ bma_paged_attn_args a, int* status) {
  __shared__ float q[kRows][kPagedHeadDim], kv[kKeys][kPagedHeadDim + 1], p[kRows][kKeys + 1], shift[kRows];
  const int G = a.Hq / c.Hkv, rows = a.T * G;
  const int h = blockIdx.y, b = blockIdx.z, r0 = blockIdx.x * kRows, n = min(kRows, rows - r0);
  const NewTokens news = new_tokens(a.lengths, a.new_lengths, b, a.T);
  auto position = [&](int r) -> int64_t { const int t = (r0 + r) / G; return t < news.count ? news.first + t : -1; };
  auto value = [&](const bma_tensor& t, int r, int i) { return (int64_t)b * t.stride_b + ((r0 + r) / G) * t.stride_l + (h * G + (r0 + r) % G) * t.stride_h + i; };
  for (int i = threadIdx.x; i < n * c.d; i += 128) {
    const int r = i / c.d;
    const int64_t at = value(a.q, r, i % c.d);
    q[r][i % c.d] = a.q.dtype == BMA_DTYPE_F32 ? static_cast<const float*>(a.q.ptr)[at] : __bfloat162float(static_cast<const __nv_bfloat16*>(a.q.ptr)[at]);
  }
  int64_t lo = 0, hi = 0;
  for (int r = 0; r < n; ++r) {
    const int64_t at = position(r);
    if (at >= 0) hi = at + 1;
    if (r == 0 && a.window >= 0 && at > a.window) lo = at - a.window;
  }
  float m = -INFINITY, l = 0.f, o[kRows];     // statistics: threads r < n; the sums of column threadIdx.x: all rows
  for (int r = 0; r < kRows; ++r) o[r] = 0.f;
  for (int64_t k0 = lo; k0 < hi; k0 += kKeys) {
    const int keys = (int)min((int64_t)kKeys, hi - k0);
    for (int side = 0; side < 2; ++side) {
      __syncthreads();
      for (int j = threadIdx.x / 32; j < keys; j += 4) {
        int slot = 0;
        const int page = page_of(c, b, k0 + j, slot);
        if (page < 0 && threadIdx.x % 32 == 0) report_device_error(status, kStatusPaged);
        const int64_t at = (int64_t)page * c.stride_page + (int64_t)slot * c.stride_slot, sat = (int64_t)page * c.scale_stride_page + (int64_t)slot * c.scale_stride_slot;
        for (int i = threadIdx.x % 32; i < c.d; i += 32) kv[j][i] = page < 0 ? 0.f : held_value(c, side, at, sat, h, i);
      }
      __syncthreads();
      if (side == 0) {
        for (int i = threadIdx.x; i < n * kKeys; i += 128) {
          const int r = i / kKeys, j = i % kKeys;
          const int64_t at = position(r), key = k0 + j;
          float s = 0.f;
          if (j < keys)
            for (int x = 0; x < c.d; ++x) s = fmaf(q[r][x], kv[j][x], s);
          p[r][j] = j < keys && key <= at && (a.window < 0 || key >= at - a.window) ? s * a.scale : -INFINITY;
        }
        __syncthreads();
        if (threadIdx.x < n) {
          const int r = threadIdx.x;
          float top = m;
          for (int j = 0; j < kKeys; ++j) top = fmaxf(top, p[r][j]);
          const float base = top == -INFINITY ? 0.f : top;
          shift[r] = expf(m - base);
          float sum = 0.f;          // (a tile's sums first: short chains)
          for (int j = 0; j < kKeys; ++j) {
            const bool seen = p[r][j] != -INFINITY;
            p[r][j] = seen ? expf(p[r][j] - base) : -1.f;      // (a key that is not seen adds nothing, whatever its value)
            if (seen) sum += p[r][j];
          }
          l = fmaf(l, shift[r], sum);
          m = top;
        }
      } else if (threadIdx.x < c.d) {
        for (int r = 0; r < n; ++r) {
          float sum = 0.f;
          for (int j = 0; j < keys; ++j)
            if (!(p[r][j] < 0.f)) sum = fmaf(p[r][j], kv[j][threadIdx.x], sum);
          o[r] = fmaf(o[r], shift[r], sum);
        }
      }
    }
  }
  __syncthreads();
  if (threadIdx.x < n) {
    shift[threadIdx.x] = l > 0.f || l != l ? 1.f / l : 0.f;
    const int t = (r0 + threadIdx.x) / G, head = h * G + (r0 + threadIdx.x) % G;
    if (a.lse) a.lse[((int64_t)b * a.Hq + head) * a.T + t] = l > 0.f || l != l ? m + logf(l) : -INFINITY;
  }
  __syncthreads();
  if (threadIdx.x < c.d)
    for (int r = 0; r < n; ++r) {
      const int64_t at = value(a.o, r, threadIdx.x);
      const float x = o[r] * shift[r];
      if (a.o.dtype == BMA_DTYPE_F32) static_cast<float*>(a.o.ptr)[at] = x;
      else static_cast<__nv_bfloat16*>(a.o.ptr)[at] = __float2bfloat16_rn(x);
    }
}

int validate_paged(const bma_paged_cache* c, const bma_paged_attn_args* a) {
  int rc = validate_cache(c);
  if (rc != BMA_OK) return rc;
  BMA_REQUIRE(a && a->T > 0 && a->Hq > 0 && a->lengths, BMA_ERR_ARG);
  BMA_REQUIRE(a->Hq % c->Hkv == 0, BMA_ERR_ARG);
  BMA_REQUIRE(a->Hq <= 65535 && (int64_t)a->T * a->Hq < (1ll << 30), BMA_ERR_LIMIT);
  BMA_REQUIRE(a->q.ptr && a->o.ptr, BMA_ERR_ARG);
  BMA_REQUIRE(a->q.dtype == (c->dtype == BMA_DTYPE_F32 ? BMA_DTYPE_F32 : BMA_DTYPE_BF16), BMA_ERR_UNSUPPORTED);
  BMA_REQUIRE(a->o.dtype == BMA_DTYPE_F32 || a->o.dtype == BMA_DTYPE_BF16, BMA_ERR_UNSUPPORTED);
  return BMA_OK;
}

}  // namespace
}  // namespace bma

using namespace bma;

extern "C" {

size_t bma_paged_attn_workspace_bytes(const bma_paged_cache* cache, const bma_paged_attn_args* args) { return 0; }

int bma_paged_attn(const bma_paged_cache* cache, const bma_paged_attn_args* args, void* workspace, size_t workspace_bytes, bma_stream_t stream) {
  int rc = validate_paged(cache, args);
  if (rc != BMA_OK) return rc;
  int* status = device_status_ptr();
  BMA_REQUIRE(status != nullptr, BMA_ERR_CUDA);
  const dim3 grid(ceil_div(args->T * (args->Hq / cache->Hkv), kRows), cache->Hkv, cache->B);
  paged_rows_kernel<<<grid, 128, 0, static_cast<cudaStream_t>(stream)>>>(*cache, *args, status);
  count_launches(1);
  BMA_CUDA_TRY(cudaGetLastError());
  return BMA_OK;
}

}
