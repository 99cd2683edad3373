// Norm and rotation of query and key heads, and what moves whole heads into and out of the pages of a cache.
//
// All of these read every value once and write every result once: they are bound by memory, for heads of few rows to a token by instructions, for a few tokens by the
// launch.  Measured: forward and backward of 4 x 4096 tokens of 64 heads of 128 bfloat16 values 248 us, 82 % of the copy rate; prompts of 8 sequences of up to 2500
// tokens, 8 heads, appended in 30 us (2.8 TB/s); contexts of 16 sequences of up to 5001 tokens read back in 85 us, 94 %.
//
// Rotation.  Component pairs are (i, i + dim/2) or (2i, 2i + 1).  A lane holds two 16-byte chunks of a head that hold both halves of its pairs
// (chunks u and u + dim/2 of a head, or chunks 2u and 2u + 1), so that no value crosses lanes; only the sum of squares does.  A head of 128
// bfloat16 values takes 8 lanes, a warp four heads at a time.  Cosine and sine of a token are taken once by the warp, through shared memory, and
// with the weights of a side make four factors of a pair, which serve all heads of that side: out = x * F + y * G, two values to an instruction.
// (Taken by every lane for itself, with weights applied first, forward and backward of 4 x 4096 tokens of 64 heads of 128 took 144 and 208 us,
// bound by instructions, three times as many.)
//
// The angle position * frequency is kept as a fraction of a turn in 64-bit integers: frequency / 2 pi as a multiple of 2^-64, times the
// position, modulo 2^64.  That is exact but for the rounding of the frequency (2^-53 of it in float64), however far the position; in float32 a
// position of 10^5 would leave 0.004 of the angle open.  The upper 32 bits then go through sincospi in float32.
//
// Tensors whose rows no 16-byte access fits, and heads whose halves begin in the middle of a chunk, go through the kernels' narrow form, a value at a time.
#include "paged.cuh"

namespace bma {
namespace {

constexpr int kHeadsThreads = 128, kHeadsWarps = kHeadsThreads / 32;
constexpr int kHeadsCtas = 8;       // at most so many CTAs to an SM, each over its share of the tokens (two waves)

template <typename T> struct Bits16;   // values of a 16-byte chunk
template <> struct Bits16<float> { static constexpr int n = 4; };
template <> struct Bits16<__nv_bfloat16> { static constexpr int n = 8; };

// frequency / 2 pi as a multiple of 2^-64, modulo 1
__device__ __forceinline__ unsigned long long step_of(double frequency) {
  double turns = frequency * 0.15915494309189533577;
  turns -= floor(turns);
  return __double2ull_rz(turns * 18446744073709551616.0);
}
// cosine and sine of position * frequency, times `magnitude`
__device__ __forceinline__ void turn_of(unsigned long long step, long long position, float magnitude, float& c, float& s) {
  const long long phase = (long long)((unsigned long long)position * step);
  sincospif((float)(int)(phase >> 32) * 4.656612873077392578125e-10f, &s, &c);   // half turns in [-1, 1]
  c *= magnitude;
  s *= magnitude;
}

// How the lanes of a warp lie on heads: `tpr` lanes (a power of two) to a head, each with a unit of two chunks (the narrow form: four units, a value to a chunk).
struct HeadMap {
  int tpr, chunks, half_chunks, dim, layout;   // half_chunks: dim / 2 in chunks (HALF layout)
};

__device__ __forceinline__ void unit_chunks(const HeadMap& m, int u, int& ca, int& cb) {
  if (m.layout == BMA_ROTARY_INTERLEAVED) { ca = 2 * u; cb = 2 * u + 1; }
  else if (u < m.half_chunks) { ca = u; cb = u + m.half_chunks; }
  else { ca = 2 * u; cb = 2 * u + 1; }   // (what is not rotated: chunks from 2 * half_chunks on)
}

// The narrow form's unit: one pair, and how it is turned.
constexpr int kUnits = 4;      // to a lane: 32 lanes hold 256 components
struct Turn {
  float c, s;
  bool live;             // the pair is rotated
  __device__ __forceinline__ void make(const HeadMap& m, const double* frequencies, int u, long long position, float magnitude) {
    c = 1.f;
    s = 0.f;
    live = 2 * u < m.dim;
    if (live) turn_of(step_of(__ldg(frequencies + u)), position, magnitude, c, s);
  }
  // BACK: by the negative angle
  template <bool BACK>
  __device__ __forceinline__ void apply(float& x, float& y) const {
    const float sn = BACK ? -s : s;
    const float p = x * c - y * sn, q = y * c + x * sn;
    if (live) { x = p; y = q; }
  }
};

// A lane's values of a head, all of them asked for at once; zeros where there are none.
template <typename T>
__device__ __forceinline__ void load_units(const T* head, bool there, const int (&ca)[kUnits], const int (&cb)[kUnits], int d, float (&a)[kUnits], float (&b)[kUnits]) {
  T x[kUnits], y[kUnits];
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    x[i] = y[i] = from_float<T>(0.f);
    if (there) {
      if (ca[i] < d) x[i] = head[ca[i]];
      if (cb[i] < d) y[i] = head[cb[i]];
    }
  }
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    a[i] = to_float(x[i]);
    b[i] = to_float(y[i]);
  }
}

__device__ __forceinline__ float group_sum(float x, int tpr) {
  for (int o = tpr >> 1; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

__device__ __forceinline__ float weight_at(const void* w, int dtype, int i) {
  return dtype == BMA_DTYPE_F32 ? __ldg(static_cast<const float*>(w) + i) : __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
}

// One side (q, k or v) of a launch: where its heads come from and go to.
struct Side {
  bma_tensor in, out;
  const void* weight;
  int heads;
  int turned;
  int before;            // heads of the sides before
};

// Division of numbers below 2^31 by one that a launch fixes: n * m >> 31 + s with m = ceil(2^(31 + s) / d), 2^s >= d, whose error n / 2^31 * d' / d < 1 / d is too
// small to reach the next whole number.
struct Divider {
  uint32_t m, s, d;
  __device__ __forceinline__ int operator()(int n) const { return d == 1 ? n : (int)(((uint64_t)(uint32_t)n * m) >> 31 >> s); }
};
inline Divider divider(int d) {
  Divider r{0, 0, (uint32_t)d};
  while ((1u << r.s) < r.d) ++r.s;
  r.m = (uint32_t)((((uint64_t)1 << (31 + r.s)) + r.d - 1) / r.d);
  return r;
}

struct HeadsParams {
  Side side[3];          // q, k, v
  Divider by_length, by_slabs;
  int B, L, d, slabs, slab_heads;
  HeadMap map;
  const double* frequencies;
  float magnitude, eps;
  int weight_dtype;
  const void* positions;
  int position_bytes;
  int64_t position_stride_b, position_stride_l;
  int back;              // rotate by the negative angle (the backward pass of a rotation alone)
  // appending
  bma_paged_cache cache;
  const int32_t *lengths, *new_lengths;
  int* status;
};

enum { kRotate = 0, kAppend = 1, kAppend4 = 2 };

template <typename P>
__device__ __forceinline__ long long position_of(const P& p, int b, int t) {
  if (!p.positions) return t;
  const int64_t at = b * p.position_stride_b + t * p.position_stride_l;
  return p.position_bytes == 8 ? __ldg(static_cast<const long long*>(p.positions) + at) : (long long)__ldg(static_cast<const int*>(p.positions) + at);
}
// Whether token t of those given of sequence b is real; its position, and its offsets in the cache (negative where there is no place for it)
__device__ __forceinline__ bool token_place(const HeadsParams& p, int b, int t, int lane, long long& position, int64_t& held, int64_t& held_scale) {
  const NewTokens n = new_tokens(p.lengths, p.new_lengths, b, p.L);
  position = n.first + t;
  if (t >= n.count) return false;
  int slot = 0;
  const int page = page_of(p.cache, b, position, slot);
  if (page < 0) {
    if (lane == 0) report_device_error(p.status, kStatusAppend);
    held = -1;
  } else {
    held = (int64_t)page * p.cache.stride_page + (int64_t)slot * p.cache.stride_slot;
    held_scale = (int64_t)page * p.cache.scale_stride_page + (int64_t)slot * p.cache.scale_stride_slot;
  }
  return true;
}

// e2m1 codes and powers of two of a warp's heads, whose values lie in shared memory: each lane takes 8 values, four lanes 32.
__device__ __forceinline__ void store_4bit(const float* row, bool there, int d, int tpr, int u, uint8_t* codes, uint8_t* scales) {
  for (int p = u; p - u < kPagedHeadDim / 8; p += tpr) {       // (every lane of the warp goes round as often)
    float x[8];
    float top = 0.f;
    bool nan = false;
    const bool in = p * 8 < d;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = in ? row[p * 8 + i] : 0.f;
      nan |= x[i] != x[i];
      top = fmaxf(top, fabsf(x[i]));
    }
    top = nan ? __uint_as_float(0x7fffffffu) : top;
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      const float t = __shfl_xor_sync(0xffffffffu, top, o);
      top = top != top || t != t ? __uint_as_float(0x7fffffffu) : fmaxf(top, t);
    }
    // smallest e with top <= 6 * 2^e = 1.5 * 2^(e + 2): from the exponent and the mantissa of top
    const uint32_t bits = __float_as_uint(top);
    int e = (int)(bits >> 23) - 127 - ((bits & 0x7fffffu) <= 0x400000u ? 2 : 1);
    e = min(max(e, -127), 126);
    const float inv = __uint_as_float((uint32_t)(127 - e) << 23);      // 2^-e, e from -127 (2^127) to 126
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w |= to_e2m1x2(x[2 * i] * inv, x[2 * i + 1] * inv) << (8 * i);
    if (there && in) {
      *reinterpret_cast<uint32_t*>(codes + p * 4) = w;
      if ((p & 3) == 0) scales[p >> 2] = top != top ? 255 : (uint8_t)(e + 127);
    }
  }
}

// The narrow form.  A warp takes one token and a slab of its heads (all sides counted through), `tpr` lanes to a head, a value at a time.
template <typename T, int KIND>
__global__ void __launch_bounds__(kHeadsThreads) heads_kernel(const __grid_constant__ HeadsParams p) {
  __shared__ float rows[KIND == kAppend4 ? kHeadsWarps : 1][KIND == kAppend4 ? 8 : 1][KIND == kAppend4 ? kPagedHeadDim + 4 : 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t item = (int64_t)blockIdx.x * kHeadsWarps + warp;
  const int64_t token = item / p.slabs;
  const int slab = (int)(item - token * p.slabs);
  const int b = (int)(token / p.L), t = (int)(token - (int64_t)b * p.L);
  if (b >= p.B) return;
  const int tpr = p.map.tpr, group = lane / tpr, u0 = lane & (tpr - 1), groups = 32 / tpr;

  long long position = t;
  bool real = true;
  int64_t held = 0, held_scale = 0;      // offsets of the token in the cache
  if constexpr (KIND == kRotate) position = position_of(p, b, t);
  else real = token_place(p, b, t, lane, position, held, held_scale);

  Turn turns[kUnits];
  int ca[kUnits], cb[kUnits];
  const bool turned = p.map.dim > 0;
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    unit_chunks(p.map, u0 + i * tpr, ca[i], cb[i]);
    if (turned) turns[i].make(p.map, p.frequencies, u0 + i * tpr, position, p.magnitude);
  }
  const int slab_begin = slab * p.slab_heads, slab_end = slab_begin + p.slab_heads;
  const float inv_d = 1.f / (float)p.d;

#pragma unroll 1
  for (int si = 0; si < (KIND == kRotate ? 2 : 3); ++si) {
    const Side& side = p.side[si];
    const int lo = max(slab_begin - side.before, 0), hi = min(slab_end - side.before, side.heads);
    if (lo >= hi) continue;
    const bool cached = KIND != kRotate && si > 0;
    if (cached && (!real || held < 0)) continue;
    const T* in = static_cast<const T*>(side.in.ptr) + b * side.in.stride_b + t * side.in.stride_l;
    T* out = static_cast<T*>(side.out.ptr) + b * side.out.stride_b + t * side.out.stride_l;
    int64_t out_head = side.out.stride_h;
    if (cached) {
      out = static_cast<T*>(si == 1 ? p.cache.k : p.cache.v) + held;      // (a 4-bit cache is not written through this)
      out_head = p.cache.stride_head;
    }
    const bool normed = side.weight != nullptr;
    float wa[kUnits], wb[kUnits];
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      wa[i] = normed && ca[i] < p.map.chunks ? weight_at(side.weight, p.weight_dtype, ca[i]) : 0.f;
      wb[i] = normed && cb[i] < p.map.chunks ? weight_at(side.weight, p.weight_dtype, cb[i]) : 0.f;
    }
#pragma unroll 1
    for (int h = lo + group; h - group < hi; h += groups) {
      float xa[kUnits], xb[kUnits];
      float sum = 0.f;
      load_units(in + h * side.in.stride_h, h < hi && real, ca, cb, p.map.chunks, xa, xb);
      if (normed) {
#pragma unroll
        for (int i = 0; i < kUnits; ++i) sum = fmaf(xa[i], xa[i], fmaf(xb[i], xb[i], sum));
        const float inv = rsqrtf(group_sum(sum, tpr) * inv_d + p.eps);
#pragma unroll
        for (int i = 0; i < kUnits; ++i) { xa[i] *= inv * wa[i]; xb[i] *= inv * wb[i]; }
      }
      if (turned && side.turned) {
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
          if (p.back) turns[i].template apply<true>(xa[i], xb[i]);
          else turns[i].template apply<false>(xa[i], xb[i]);
        }
      }
      if (KIND == kAppend4 && cached) {
        float* row = rows[warp][group];
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
          if (ca[i] < p.map.chunks) row[ca[i]] = xa[i];
          if (cb[i] < p.map.chunks) row[cb[i]] = xb[i];
        }
        __syncwarp();
        uint8_t* codes = static_cast<uint8_t*>(si == 1 ? p.cache.k : p.cache.v) + held + h * p.cache.stride_head;
        uint8_t* scales = (si == 1 ? p.cache.k_scale : p.cache.v_scale) + held_scale + h * p.cache.scale_stride_head;
        store_4bit(row, h < hi, p.d, tpr, u0, codes, scales);
      } else if (h < hi) {
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {      // (zeros for a token that is not real)
          if (ca[i] < p.map.chunks) out[h * out_head + ca[i]] = from_float<T>(real ? xa[i] : 0.f);
          if (cb[i] < p.map.chunks) out[h * out_head + cb[i]] = from_float<T>(real ? xb[i] : 0.f);
        }
      }
    }
  }
}

// Backward of norm and rotation.  With g' = the cotangent turned back, x^ = x * inv and the norm's weight w:
//   dx = inv * (g' w - x^ mean(g' w x^)),  dw = sum over tokens and heads of g' x^.
// The first `q_ctas` CTAs take q, the others k; each warp goes over tokens and keeps its share of dw in registers, the CTAs' shares go to
// `partial` [CTAs, d] and are added up by weight_sum_kernel in a fixed order.
struct BackParams {
  Side side[2];          // in: x, out: dx
  bma_tensor g[2];
  int B, L, d, q_ctas;
  HeadMap map;
  const double* frequencies;
  float magnitude, eps;
  int weight_dtype;
  const void* positions;
  int position_bytes;
  int64_t position_stride_b, position_stride_l;
  float* partial;
};

template <typename T>
__global__ void __launch_bounds__(kHeadsThreads, 4) rotate_back_kernel(const __grid_constant__ BackParams p) {
  __shared__ float sums[kHeadsWarps][256];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int tpr = p.map.tpr, group = lane / tpr, u0 = lane & (tpr - 1), groups = 32 / tpr;
  const int si = (int)blockIdx.x < p.q_ctas ? 0 : 1;
  const int cta = si ? blockIdx.x - p.q_ctas : blockIdx.x, ctas = si ? gridDim.x - p.q_ctas : p.q_ctas;
  const Side& side = p.side[si];
  const bma_tensor& g = p.g[si];
  const float inv_d = 1.f / (float)p.d;
  int ca[kUnits], cb[kUnits];
  float wa[kUnits], wb[kUnits], da[kUnits], db[kUnits];
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    unit_chunks(p.map, u0 + i * tpr, ca[i], cb[i]);
    wa[i] = ca[i] < p.map.chunks ? weight_at(side.weight, p.weight_dtype, ca[i]) : 0.f;
    wb[i] = cb[i] < p.map.chunks ? weight_at(side.weight, p.weight_dtype, cb[i]) : 0.f;
    da[i] = db[i] = 0.f;
  }
  const int64_t tokens = (int64_t)p.B * p.L;
#pragma unroll 1
  for (int64_t token = (int64_t)cta * kHeadsWarps + warp; token < tokens; token += (int64_t)ctas * kHeadsWarps) {
    const int b = (int)(token / p.L), t = (int)(token - (int64_t)b * p.L);
    const long long position = position_of(p, b, t);
    Turn turns[kUnits];
    const bool turned = p.map.dim > 0;
    if (turned) {
#pragma unroll
      for (int i = 0; i < kUnits; ++i) turns[i].make(p.map, p.frequencies, u0 + i * tpr, position, p.magnitude);
    }
    const T* in = static_cast<const T*>(side.in.ptr) + b * side.in.stride_b + t * side.in.stride_l;
    const T* gin = static_cast<const T*>(g.ptr) + b * g.stride_b + t * g.stride_l;
    T* out = static_cast<T*>(side.out.ptr) + b * side.out.stride_b + t * side.out.stride_l;
#pragma unroll 1
    for (int h = group; h - group < side.heads; h += groups) {
      const bool there = h < side.heads;
      float fa[kUnits], fb[kUnits], ea[kUnits], eb[kUnits];
      float sum = 0.f, dot = 0.f;
      load_units(in + h * side.in.stride_h, there, ca, cb, p.map.chunks, fa, fb);
      load_units(gin + h * g.stride_h, there, ca, cb, p.map.chunks, ea, eb);
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        if (turned) turns[i].template apply<true>(ea[i], eb[i]);
        sum = fmaf(fa[i], fa[i], fmaf(fb[i], fb[i], sum));
        dot = fmaf(ea[i] * wa[i], fa[i], fmaf(eb[i] * wb[i], fb[i], dot));
      }
      for (int o = tpr >> 1; o; o >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
        dot += __shfl_xor_sync(0xffffffffu, dot, o);
      }
      const float inv = rsqrtf(sum * inv_d + p.eps), m = dot * inv * inv_d;     // m = mean(g' w x^)
      if (!there) continue;
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        const float ha = fa[i] * inv, hb = fb[i] * inv;
        da[i] = fmaf(ea[i], ha, da[i]);
        db[i] = fmaf(eb[i], hb, db[i]);
        if (ca[i] < p.map.chunks) out[h * side.out.stride_h + ca[i]] = from_float<T>(inv * (ea[i] * wa[i] - ha * m));
        if (cb[i] < p.map.chunks) out[h * side.out.stride_h + cb[i]] = from_float<T>(inv * (eb[i] * wb[i] - hb * m));
      }
    }
  }
  // the groups of a warp, the warps of the CTA
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    for (int o = tpr; o < 32; o <<= 1) {
      da[i] += __shfl_xor_sync(0xffffffffu, da[i], o);
      db[i] += __shfl_xor_sync(0xffffffffu, db[i], o);
    }
    if (group == 0) {
      if (ca[i] < p.map.chunks) sums[warp][ca[i]] = da[i];
      if (cb[i] < p.map.chunks) sums[warp][cb[i]] = db[i];
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < p.d; c += kHeadsThreads) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kHeadsWarps; ++w) s += sums[w][c];
    p.partial[(int64_t)blockIdx.x * p.d + c] = s;
  }
}

// ---- 16-byte chunks -----------------------------------------------------------------------------------------------------
// A lane's unit of a head: VEC pairs of neighbouring values (as float2), those of chunk `ca`, then those of chunk `cb`.
template <typename T>
struct Unit {
  static constexpr int VEC = Bits16<T>::n;
  uint4 a, b;
  __device__ __forceinline__ void load(const T* p, int ca, int cb, int chunks) {
    a = b = make_uint4(0, 0, 0, 0);
    if (ca < chunks) a = *reinterpret_cast<const uint4*>(p + ca * VEC);
    if (cb < chunks) b = *reinterpret_cast<const uint4*>(p + cb * VEC);
  }
  __device__ __forceinline__ void zero() { a = b = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void get(float2 (&v)[VEC]) const {
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      if constexpr (VEC == 8) v[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
      else v[i] = make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    }
  }
  __device__ __forceinline__ void set(const float2 (&v)[VEC]) {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      if constexpr (VEC == 8) {
        const __nv_bfloat162 h = __float22bfloat162_rn(v[i]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        w[2 * i] = __float_as_uint(v[i].x);
        w[2 * i + 1] = __float_as_uint(v[i].y);
      }
    }
    a = make_uint4(w[0], w[1], w[2], w[3]);
    b = make_uint4(w[4], w[5], w[6], w[7]);
  }
  __device__ __forceinline__ void store(T* p, int ca, int cb, int chunks) const {
    if (ca < chunks) *reinterpret_cast<uint4*>(p + ca * VEC) = a;
    if (cb < chunks) *reinterpret_cast<uint4*>(p + cb * VEC) = b;
  }
};
__device__ __forceinline__ float2 swapped(float2 v) { return make_float2(v.y, v.x); }
__device__ __forceinline__ float2 twice(float x) { return make_float2(x, x); }

// 64-bit steps of the pairs (a CTA makes them once), and a warp's cosines and sines of a token, a gap after every unit's, so that lanes read from different banks.
constexpr int kPairs = 128;
template <int VEC>
constexpr int kTurns = kPairs / VEC * (VEC + 1);
__device__ __forceinline__ void make_steps(unsigned long long* steps, const double* frequencies, int pairs) {
  for (int i = threadIdx.x; i < pairs; i += blockDim.x) steps[i] = step_of(__ldg(frequencies + i));
  __syncthreads();
}
template <int VEC>
__device__ __forceinline__ void make_turns(float2* turns, const unsigned long long* steps, int pairs, long long position, float magnitude, int lane) {
  __syncwarp();            // (those of the last token have been read)
  for (int i = lane; i < pairs; i += 32) {
    float c, s;
    turn_of(steps[i], position, magnitude, c, s);
    turns[i + i / VEC] = make_float2(c, s);
  }
  __syncwarp();
}

// Bits of the unit's pairs of components that are rotated: component pairs u * VEC and up are (value j of chunk a, value j of chunk b) in the HALF layout,
// else neighbours.
template <int VEC>
__device__ __forceinline__ uint32_t live_pairs(int u, int pairs) {
  const int n = min(max(pairs - u * VEC, 0), VEC);
  return (1u << n) - 1u;
}

// The rows ahead of a warp: the heads of a token that it takes at once, item by item and side by side as it will come to them.  Each lane copies its own
// 32 bytes of them into its own place in shared memory, where it alone reads them: kAhead rows are on their way without a register or a barrier.
constexpr int kAhead = 4;      // (a power of two)
template <typename T, int KIND>
struct RowsAhead {
  static constexpr int kSides = KIND == kRotate ? 2 : 3;
  int item, items, stride;           // items of this warp: item, item + stride, ...
  int b, t, begin;                   // its token, first head
  int si, h, hi;                     // next rows: heads h + group below hi of side si
  const T* at;                       // this lane's head of them
  int64_t step;                      // to the next rows
  int to;
  bool real;

  __device__ __forceinline__ void start(const HeadsParams& p, int first, int all, int by, int group, int groups) {
    item = first;
    items = all;
    stride = by;
    to = 0;
    h = hi = 0;
    if (open(p)) next(p, group, groups);
  }
  __device__ __forceinline__ bool open(const HeadsParams& p) {
    if (item >= items) return false;
    const int token = p.by_slabs(item);
    begin = (item - token * p.slabs) * p.slab_heads;
    b = p.by_length(token);
    t = token - b * p.L;
    real = KIND == kRotate || t < new_tokens(p.lengths, p.new_lengths, b, p.L).count;
    si = -1;
    return true;
  }
  // To the next side that has rows; item >= items: there is none.
  __device__ __forceinline__ void next(const HeadsParams& p, int group, int groups) {
    do {
      while (real && ++si < kSides) {
        const Side& side = p.side[si];
        h = max(begin - side.before, 0);
        hi = min(begin + p.slab_heads - side.before, side.heads);
        if (h >= hi) continue;
        at = static_cast<const T*>(side.in.ptr) + b * side.in.stride_b + t * side.in.stride_l + (h + group) * side.in.stride_h;
        step = groups * side.in.stride_h;
        return;
      }
      item += stride;
    } while (open(p));
  }
  // Asks for the next rows, if there are any.  `ring`: the shared address of this lane's place, 2 * kAhead chunks, 512 bytes apart; A, B: it has chunks a and b.
  __device__ __forceinline__ void fetch(const HeadsParams& p, uint32_t ring, int group, int groups, int ca, int cb, bool A, bool B) {
    constexpr int VEC = Bits16<T>::n;
    if (item < items) {
      const bool there = h + group < hi;
      const uint32_t dst = ring + to * 1024;
      if (there && A) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(at + ca * VEC) : "memory");
      if (there && B) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + 512), "l"(at + cb * VEC) : "memory");
      to = (to + 1) & (kAhead - 1);
      at += step;
      h += groups;
      if (h >= hi) next(p, group, groups);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
};

// The same work as heads_kernel's.  FULL: every component is rotated.
template <typename T, int LAYOUT, bool FULL, int KIND>
__global__ void __launch_bounds__(kHeadsThreads, 4) heads_wide_kernel(const __grid_constant__ HeadsParams p) {
  constexpr int VEC = Bits16<T>::n;
  constexpr bool HALF = LAYOUT == BMA_ROTARY_HALF;
  __shared__ unsigned long long steps[kPairs];
  __shared__ float2 turns[kHeadsWarps][kTurns<VEC>];
  __shared__ uint4 rings[kHeadsWarps][kAhead][2][32];
  __shared__ __align__(16) float weights[2][2 * kPairs];
  __shared__ float rows[KIND == kAppend4 ? kHeadsWarps : 1][KIND == kAppend4 ? 8 : 1][KIND == kAppend4 ? kPagedHeadDim + 4 : 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int tpr = p.map.tpr, group = lane / tpr, u = lane & (tpr - 1), groups = 32 / tpr, chunks = p.map.chunks;
  const int pairs = p.map.dim / 2;
  int ca, cb;
  unit_chunks(p.map, u, ca, cb);
  const uint32_t live = live_pairs<VEC>(u, pairs);
  const float inv_d = 1.f / (float)p.d;
  const bool A = ca < chunks, B = cb < chunks;
  const int items = p.B * p.L * p.slabs, first_item = blockIdx.x * kHeadsWarps + warp, stride = gridDim.x * kHeadsWarps;      // (below 2^31: launch_heads)
  uint4* ring = &rings[warp][0][0][lane];
  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
  RowsAhead<T, KIND> ahead;
  ahead.start(p, first_item, items, stride, group, groups);
#pragma unroll
  for (int i = 0; i < kAhead - 1; ++i) ahead.fetch(p, ring_at, group, groups, ca, cb, A, B);
  for (int i = threadIdx.x; i < 2 * p.d; i += kHeadsThreads) {
    const int si = i >= p.d, k = i - si * p.d;
    const void* w = p.side[si].weight;
    weights[si][k] = w ? weight_at(w, p.weight_dtype, k) : 1.f;
  }
  make_steps(steps, p.frequencies, pairs);
  int from = 0;
#pragma unroll 1
  for (int item = first_item; item < items; item += stride) {
    const int token = p.by_slabs(item);
    const int slab_begin = (item - token * p.slabs) * p.slab_heads, slab_end = slab_begin + p.slab_heads;
    const int b = p.by_length(token), t = token - b * p.L;
    long long position = t;
    bool real = true;
    int64_t held = 0, held_scale = 0;      // offsets of the token in the cache
    if constexpr (KIND == kRotate) position = position_of(p, b, t);
    else real = token_place(p, b, t, lane, position, held, held_scale);
    if (pairs && real) make_turns<VEC>(turns[warp], steps, pairs, position, p.back ? -p.magnitude : p.magnitude, lane);
#pragma unroll 1
    for (int si = 0; si < (KIND == kRotate ? 2 : 3); ++si) {
      const Side& side = p.side[si];
      const int lo = max(slab_begin - side.before, 0), hi = min(slab_end - side.before, side.heads);
      if (lo >= hi) continue;
      const bool cached = KIND != kRotate && si > 0;
      T* out = static_cast<T*>(side.out.ptr) + b * side.out.stride_b + t * side.out.stride_l;
      int64_t out_head = side.out.stride_h;
      if (cached) {
        out = static_cast<T*>(si == 1 ? p.cache.k : p.cache.v) + held;      // (a 4-bit cache is not written through this)
        out_head = p.cache.stride_head;
      }
      out += (lo + group) * out_head;
      if (KIND != kRotate && !real) {       // zeros for queries of tokens that are not real
        Unit<T> zero;
        zero.zero();
        if (!cached)
          for (int h = lo + group; h < hi; h += groups, out += groups * out_head) zero.store(out, ca, cb, chunks);
        continue;
      }
      const bool normed = side.weight != nullptr, plain = !normed && !side.turned;
      // out = v * F + (the other half of the pair) * G
      float2 F[VEC], G[VEC];
      if (!plain) {
        float2 w[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) w[i] = make_float2(1.f, 1.f);
        if (normed) {
#pragma unroll
          for (int i = 0; i < VEC / 2; ++i) {
            if (A) w[i] = *reinterpret_cast<const float2*>(&weights[si][ca * VEC + 2 * i]);
            if (B) w[VEC / 2 + i] = *reinterpret_cast<const float2*>(&weights[si][cb * VEC + 2 * i]);
          }
        }
        float2 cs[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          cs[j] = make_float2(1.f, 0.f);
          if (side.turned && (FULL || live >> j & 1) && u * VEC + j < pairs) cs[j] = turns[warp][u * (VEC + 1) + j];
          if (p.back) cs[j].x = (FULL || live >> j & 1) ? -cs[j].x : cs[j].x;      // (-magnitude gave -cos and -sin)
        }
        if constexpr (HALF) {
#pragma unroll
          for (int i = 0; i < VEC / 2; ++i) {
            const float2 c = make_float2(cs[2 * i].x, cs[2 * i + 1].x), s = make_float2(cs[2 * i].y, cs[2 * i + 1].y);
            F[i] = __fmul2_rn(c, w[i]);
            F[VEC / 2 + i] = __fmul2_rn(c, w[VEC / 2 + i]);
            G[i] = __fmul2_rn(make_float2(-s.x, -s.y), w[VEC / 2 + i]);
            G[VEC / 2 + i] = __fmul2_rn(s, w[i]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            F[j] = __fmul2_rn(twice(cs[j].x), w[j]);
            G[j] = __fmul2_rn(make_float2(-cs[j].y, cs[j].y), swapped(w[j]));
          }
        }
      }
      const int64_t out_step = groups * out_head;
#pragma unroll 1
      for (int h = lo + group; h - group < hi; h += groups, out += out_step) {
        ahead.fetch(p, ring_at, group, groups, ca, cb, A, B);
        asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
        Unit<T> x;
        x.zero();
        if (h < hi && A) x.a = ring[from * 64];
        if (h < hi && B) x.b = ring[from * 64 + 32];
        from = (from + 1) & (kAhead - 1);
        float2 v[VEC];
        if (!plain || KIND == kAppend4) x.get(v);
        if (!plain) {
          float2 o[VEC];
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            float2 other = HALF ? v[(i + VEC / 2) % VEC] : swapped(v[i]);
            // what is not rotated takes nothing of its neighbour, not even a zero times infinity
            if (!FULL && !(HALF ? live != 0 : live >> i & 1)) other = make_float2(0.f, 0.f);
            o[i] = __ffma2_rn(v[i], F[i], __fmul2_rn(other, G[i]));
          }
          if (normed) {
            float2 sum = make_float2(0.f, 0.f);
#pragma unroll
            for (int i = 0; i < VEC; ++i) sum = __ffma2_rn(v[i], v[i], sum);
            const float2 inv = twice(rsqrtf(group_sum(sum.x + sum.y, tpr) * inv_d + p.eps));
#pragma unroll
            for (int i = 0; i < VEC; ++i) o[i] = __fmul2_rn(o[i], inv);
          }
          if (KIND == kAppend4 && cached) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[i] = o[i];
          } else x.set(o);
        }
        if (KIND != kRotate && cached && held < 0) continue;
        if (KIND == kAppend4 && cached) {
          float* row = rows[warp][group];
          __syncwarp();
#pragma unroll
          for (int i = 0; i < VEC / 2; ++i) {
            if (ca < chunks) *reinterpret_cast<float2*>(row + ca * VEC + 2 * i) = v[i];
            if (cb < chunks) *reinterpret_cast<float2*>(row + cb * VEC + 2 * i) = v[VEC / 2 + i];
          }
          __syncwarp();
          uint8_t* codes = static_cast<uint8_t*>(si == 1 ? p.cache.k : p.cache.v) + held + h * p.cache.stride_head;
          uint8_t* scales = (si == 1 ? p.cache.k_scale : p.cache.v_scale) + held_scale + h * p.cache.scale_stride_head;
          store_4bit(row, h < hi, p.d, tpr, u, codes, scales);
        } else if (h < hi) x.store(out, ca, cb, chunks);
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// The same work as rotate_back_kernel's.  (Four CTAs to an SM: 128 registers, for which bfloat16 spills 8 to 40 bytes.)
template <typename T, int LAYOUT, bool FULL>
__global__ void __launch_bounds__(kHeadsThreads, 4) rotate_back_wide_kernel(const __grid_constant__ BackParams p) {
  constexpr int VEC = Bits16<T>::n;
  constexpr bool HALF = LAYOUT == BMA_ROTARY_HALF;
  constexpr int CS = HALF ? VEC / 2 : VEC;
  __shared__ unsigned long long steps[kPairs];
  __shared__ float2 turns[kHeadsWarps][kTurns<VEC>];
  __shared__ uint4 rings[kHeadsWarps][kAhead][4][32];       // (the sums of the warps lie there at the end)
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int tpr = p.map.tpr, group = lane / tpr, u = lane & (tpr - 1), groups = 32 / tpr, chunks = p.map.chunks;
  const int si = (int)blockIdx.x < p.q_ctas ? 0 : 1;
  const int cta = si ? blockIdx.x - p.q_ctas : blockIdx.x, ctas = si ? gridDim.x - p.q_ctas : p.q_ctas;
  const Side& side = p.side[si];
  const bma_tensor& g = p.g[si];
  const float inv_d = 1.f / (float)p.d;
  const int pairs = p.map.dim / 2, heads = side.heads;
  int ca, cb;
  unit_chunks(p.map, u, ca, cb);
  const bool A = ca < chunks, B = cb < chunks;
  const uint32_t live = live_pairs<VEC>(u, pairs);
  const int tokens = p.B * p.L, stride = ctas * kHeadsWarps;       // (below 2^30: rotate_backward)

  // rows on their way, as in RowsAhead: four chunks, of x and of the cotangent
  uint4* ring = &rings[warp][0][0][lane];
  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
  const int64_t x_step = groups * side.in.stride_h, g_step = groups * g.stride_h;
  const T *ax = nullptr, *ag = nullptr;
  int next_token = cta * kHeadsWarps + warp, next_head = 0, to = 0;
  auto open = [&] {
    if (next_token >= tokens) return;
    const int b = next_token / p.L, t = next_token - b * p.L;
    ax = static_cast<const T*>(side.in.ptr) + b * side.in.stride_b + t * side.in.stride_l + group * side.in.stride_h;
    ag = static_cast<const T*>(g.ptr) + b * g.stride_b + t * g.stride_l + group * g.stride_h;
  };
  auto fetch = [&] {
    if (next_token < tokens) {
      const uint32_t dst = ring_at + to * 2048;
      if (next_head + group < heads) {
        if (A) {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(ax + ca * VEC) : "memory");
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + 1024), "l"(ag + ca * VEC) : "memory");
        }
        if (B) {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + 512), "l"(ax + cb * VEC) : "memory");
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + 1536), "l"(ag + cb * VEC) : "memory");
        }
      }
      to = (to + 1) & (kAhead - 1);
      ax += x_step;
      ag += g_step;
      next_head += groups;
      if (next_head >= heads) {
        next_head = 0;
        next_token += stride;
        open();
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  open();
#pragma unroll
  for (int i = 0; i < kAhead - 1; ++i) fetch();
  make_steps(steps, p.frequencies, pairs);

  float2 w[VEC], dw[VEC];
  {
    const auto at = [&](int chunk, int j) { return chunk < chunks ? weight_at(side.weight, p.weight_dtype, chunk * VEC + j) : 0.f; };
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      w[i] = make_float2(at(ca, 2 * i), at(ca, 2 * i + 1));
      w[VEC / 2 + i] = make_float2(at(cb, 2 * i), at(cb, 2 * i + 1));
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) dw[i] = make_float2(0.f, 0.f);
  }
  int from = 0;
#pragma unroll 1
  for (int token = cta * kHeadsWarps + warp; token < tokens; token += stride) {
    const int b = token / p.L, t = token - b * p.L;
    // cosines and sines of the unit's values: HALF, of pairs 2i and 2i + 1 and the sines with the other sign, too; else of both values of pair i, the sine
    // with its sign
    float2 c[CS], s[CS], ns[CS];
    if (pairs) make_turns<VEC>(turns[warp], steps, pairs, position_of(p, b, t), p.magnitude, lane);
#pragma unroll
    for (int i = 0; i < CS; ++i) {
      const auto at = [&](int j) { return (FULL || live >> j & 1) && u * VEC + j < pairs ? turns[warp][u * (VEC + 1) + j] : make_float2(1.f, 0.f); };
      if constexpr (HALF) {
        const float2 x = at(2 * i), y = at(2 * i + 1);
        c[i] = make_float2(x.x, y.x);
        s[i] = make_float2(x.y, y.y);
        ns[i] = make_float2(-x.y, -y.y);
      } else {
        const float2 x = at(i);
        c[i] = twice(x.x);
        s[i] = make_float2(x.y, -x.y);
      }
    }
    T* out = static_cast<T*>(side.out.ptr) + b * side.out.stride_b + t * side.out.stride_l + group * side.out.stride_h;
    const int64_t out_step = groups * side.out.stride_h;
#pragma unroll 1
    for (int h = group; h - group < heads; h += groups, out += out_step) {
      fetch();
      asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
      const bool there = h < heads;
      Unit<T> x, y;
      x.zero();
      y.zero();
      if (there && A) { x.a = ring[from * 128]; y.a = ring[from * 128 + 64]; }
      if (there && B) { x.b = ring[from * 128 + 32]; y.b = ring[from * 128 + 96]; }
      from = (from + 1) & (kAhead - 1);
      float2 v[VEC], e[VEC], f[VEC];
      x.get(v);
      y.get(e);
      float2 sum = make_float2(0.f, 0.f), dot = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        float2 other = HALF ? e[(i + VEC / 2) % VEC] : swapped(e[i]);
        if (!FULL && !(HALF ? live != 0 : live >> i & 1)) other = make_float2(0.f, 0.f);
        if constexpr (HALF) {
          const int k = i % (VEC / 2);
          f[i] = __ffma2_rn(e[i], c[k], __fmul2_rn(other, i < VEC / 2 ? s[k] : ns[k]));
        } else f[i] = __ffma2_rn(e[i], c[i], __fmul2_rn(other, s[i]));
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        e[i] = __fmul2_rn(f[i], v[i]);                 // g' x
        f[i] = __fmul2_rn(f[i], w[i]);
        sum = __ffma2_rn(v[i], v[i], sum);
        dot = __ffma2_rn(e[i], w[i], dot);
      }
      float sum1 = sum.x + sum.y, dot1 = dot.x + dot.y;
      for (int o = tpr >> 1; o; o >>= 1) {
        sum1 += __shfl_xor_sync(0xffffffffu, sum1, o);
        dot1 += __shfl_xor_sync(0xffffffffu, dot1, o);
      }
      const float inv = there ? rsqrtf(sum1 * inv_d + p.eps) : 0.f;
      const float2 inv2 = twice(inv), m = twice(-(dot1 * inv * inv_d) * inv * inv);    // -inv^2 mean(g' w x^)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        dw[i] = __ffma2_rn(e[i], inv2, dw[i]);
        f[i] = __ffma2_rn(v[i], m, __fmul2_rn(f[i], inv2));
      }
      if (there) {
        y.set(f);
        y.store(out, ca, cb, chunks);
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  float (*sums)[256] = reinterpret_cast<float (*)[256]>(&rings[0][0][0][0]);
  // the groups of a warp, the warps of the CTA
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    for (int o = tpr; o < 32; o <<= 1) {
      dw[i].x += __shfl_xor_sync(0xffffffffu, dw[i].x, o);
      dw[i].y += __shfl_xor_sync(0xffffffffu, dw[i].y, o);
    }
    const int chunk = i < VEC / 2 ? ca : cb;
    if (group == 0 && chunk < chunks) *reinterpret_cast<float2*>(&sums[warp][chunk * VEC + 2 * (i % (VEC / 2))]) = dw[i];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < p.d; i += kHeadsThreads) {
    float x = 0.f;
#pragma unroll
    for (int k = 0; k < kHeadsWarps; ++k) x += sums[k][i];
    p.partial[(int64_t)blockIdx.x * p.d + i] = x;
  }
}

// dw of q (blockIdx.y 0) and k: columns of `partial` added up, 32 columns to a CTA, 32 rows at a time.
__global__ void __launch_bounds__(1024) weight_sum_kernel(const float* partial, int q_ctas, int k_ctas, int d, void* dq, void* dk, int dtype) {
  __shared__ float sums[32][33];
  const bool k = blockIdx.y;
  const float* rows = partial + (k ? (int64_t)q_ctas * d : 0);
  const int n = k ? k_ctas : q_ctas, c = blockIdx.x * 32 + threadIdx.x;
  void* out = k ? dk : dq;
  if (!n || !out) return;
  float s = 0.f;
  if (c < d)
    for (int r = threadIdx.y; r < n; r += 32) s += rows[(int64_t)r * d + c];
  sums[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  s = sums[threadIdx.x][threadIdx.y];       // column blockIdx.x * 32 + threadIdx.y
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const int col = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && col < d) {
    if (dtype == BMA_DTYPE_F32) static_cast<float*>(out)[col] = s;
    else static_cast<__nv_bfloat16*>(out)[col] = __float2bfloat16_rn(s);
  }
}

// Pages back to dense rows: a thread moves 16 bytes of the output (8 values of a 4-bit cache) of keys and of values at a time.  A CTA takes kReadTokens
// neighbouring tokens of a sequence, whose places it looks up at once, so that what then follows are loads that do not wait for one another.
constexpr int kReadTokens = 16;
template <int DTYPE>
__global__ void __launch_bounds__(256) read_kv_kernel(const __grid_constant__ bma_paged_cache c, const int32_t* lengths, int L, const bma_tensor k, const bma_tensor v,
                                                      int* status) {
  using T = typename std::conditional<DTYPE == BMA_DTYPE_F32, float, __nv_bfloat16>::type;
  constexpr int VEC = Bits16<T>::n;
  __shared__ int64_t held[kReadTokens], held_scale[kReadTokens];       // negative: nothing there
  const int per_head = c.d / VEC, per_token = c.Hkv * per_head;
  const int runs = (L + kReadTokens - 1) / kReadTokens, b = blockIdx.x / runs, t0 = (blockIdx.x - b * runs) * kReadTokens;
  const int tid = threadIdx.y * blockDim.x + threadIdx.x, n = min(kReadTokens, L - t0);
  if (tid < n) {
    int slot = 0, page = -1;
    if (t0 + tid < __ldg(lengths + b)) {
      page = page_of(c, b, t0 + tid, slot);
      if (page < 0) report_device_error(status, kStatusRead);
    }
    held[tid] = page < 0 ? -1 : (int64_t)page * c.stride_page + (int64_t)slot * c.stride_slot;
    held_scale[tid] = page < 0 ? -1 : (int64_t)page * c.scale_stride_page + (int64_t)slot * c.scale_stride_slot;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < per_token; i += blockDim.x) {
    const int h = i / per_head, at = (i - h * per_head) * VEC;
    T* to_k = static_cast<T*>(k.ptr) + b * k.stride_b + t0 * k.stride_l + h * k.stride_h + at;
    T* to_v = static_cast<T*>(v.ptr) + b * v.stride_b + t0 * v.stride_l + h * v.stride_h + at;
    const int64_t in_token = h * c.stride_head + (DTYPE == BMA_DTYPE_MXFP4 ? at / 2 : at), scale_in_token = h * c.scale_stride_head + at / 32;
#pragma unroll 4
    for (int t = threadIdx.y; t < n; t += blockDim.y) {
      uint4 x[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
      const int64_t from = held[t];
      if (from >= 0) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          if constexpr (DTYPE == BMA_DTYPE_MXFP4) {
            const uint32_t codes = __ldg(reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(s ? c.v : c.k) + from + in_token));
            const float f = e8m0_value(__ldg((s ? c.v_scale : c.k_scale) + held_scale[t] + scale_in_token));
            uint32_t pairs[4], w[4];
            from_e2m1x8(codes, pairs);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&pairs[j]));
              const __nv_bfloat162 r = __floats2bfloat162_rn(y.x * f, y.y * f);       // (exact: two significant bits)
              w[j] = *reinterpret_cast<const uint32_t*>(&r);
            }
            x[s] = make_uint4(w[0], w[1], w[2], w[3]);
          } else {
            x[s] = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(s ? c.v : c.k) + from + in_token));
          }
        }
      }
      *reinterpret_cast<uint4*>(to_k + t * k.stride_l) = x[0];
      *reinterpret_cast<uint4*>(to_v + t * v.stride_l) = x[1];
    }
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------------
int validate_rotary(const bma_rotary& r, int d) {
  BMA_REQUIRE(r.dim >= 0 && r.dim % 2 == 0 && r.dim <= d, BMA_ERR_ARG);
  BMA_REQUIRE(r.dim == 0 || r.frequencies, BMA_ERR_ARG);
  BMA_REQUIRE(r.layout == BMA_ROTARY_HALF || r.layout == BMA_ROTARY_INTERLEAVED, BMA_ERR_ARG);
  BMA_REQUIRE((!r.q_weight && !r.k_weight) || r.weight_dtype == BMA_DTYPE_F32 || r.weight_dtype == BMA_DTYPE_BF16, BMA_ERR_UNSUPPORTED);
  return BMA_OK;
}

bool wide_tensor(const bma_tensor& t, int vec) {
  return (reinterpret_cast<uintptr_t>(t.ptr) & 15) == 0 && t.stride_b % vec == 0 && t.stride_l % vec == 0 && t.stride_h % vec == 0;
}

// 16-byte chunks where every tensor allows them and no pair of the HALF layout has its halves in the middle of chunks
bool wide_heads(const bma_rotary& r, int d, int vec) { return d % vec == 0 && (r.layout == BMA_ROTARY_INTERLEAVED || (r.dim / 2) % vec == 0); }

HeadMap head_map(const bma_rotary& r, int d, int vec, int least) {
  HeadMap m{};
  m.chunks = ceil_div(d, vec);
  m.half_chunks = r.dim / 2 / vec;
  m.dim = r.dim;
  m.layout = r.layout;
  m.tpr = least;
  while (m.tpr < 32 && m.tpr < (m.chunks + 1) / 2) m.tpr *= 2;
  return m;
}

// Warps of a launch take a token and `slab_heads` of its heads: all of them where there are tokens enough for 16 warps an SM, fewer
// (down to one pass of the warp) where there are not.
void cut_heads(HeadsParams& p, int64_t tokens, int heads, int pass) {
  const int64_t want = ceil_div(device_sms(current_device()) * 16, (int)std::min<int64_t>(tokens, 1 << 20));
  p.slab_heads = (int)std::max<int64_t>(pass, ceil_div(heads, (int)want));
  p.slab_heads = ceil_div(p.slab_heads, pass) * pass;
  p.slabs = ceil_div(heads, p.slab_heads);
}

template <typename T, int KIND>
int launch_heads(HeadsParams& p, const bma_rotary& r, bool wide, cudaStream_t st) {
  const int vec = wide ? Bits16<T>::n : 1;
  p.map = head_map(r, p.d, vec, KIND == kAppend4 ? 4 : 1);
  const int64_t tokens = (int64_t)p.B * p.L;
  const int heads = p.side[0].heads + p.side[1].heads + p.side[2].heads;
  cut_heads(p, tokens, heads, 32 / p.map.tpr);
  p.side[1].before = p.side[0].heads;
  p.side[2].before = p.side[0].heads + p.side[1].heads;
  BMA_REQUIRE(tokens * p.slabs < (1ll << 30), BMA_ERR_LIMIT);
  p.by_length = divider(p.L);
  p.by_slabs = divider(p.slabs);
  int64_t ctas = (tokens * p.slabs + kHeadsWarps - 1) / kHeadsWarps;
  if (wide) {
    ctas = std::min<int64_t>(ctas, (int64_t)device_sms(current_device()) * kHeadsCtas);
    const bool full = r.dim == p.d;
#define BMA_WIDE(LAYOUT, FULL) heads_wide_kernel<T, LAYOUT, FULL, KIND><<<(unsigned)ctas, kHeadsThreads, 0, st>>>(p)
    if (r.layout == BMA_ROTARY_HALF) { if (full) BMA_WIDE(BMA_ROTARY_HALF, true); else BMA_WIDE(BMA_ROTARY_HALF, false); }
    else { if (full) BMA_WIDE(BMA_ROTARY_INTERLEAVED, true); else BMA_WIDE(BMA_ROTARY_INTERLEAVED, false); }
#undef BMA_WIDE
  } else heads_kernel<T, KIND><<<(unsigned)ctas, kHeadsThreads, 0, st>>>(p);
  count_launches(1);
  BMA_CUDA_TRY(cudaGetLastError());
  return BMA_OK;
}

int validate_heads(const bma_tensor& t, int dtype) {
  BMA_REQUIRE(t.ptr, BMA_ERR_ARG);
  BMA_REQUIRE(t.dtype == BMA_DTYPE_F32 || t.dtype == BMA_DTYPE_BF16, BMA_ERR_UNSUPPORTED);
  BMA_REQUIRE(t.dtype == dtype, BMA_ERR_UNSUPPORTED);
  return BMA_OK;
}

int validate_rotate(const bma_rotate_args* a) {
  BMA_REQUIRE(a, BMA_ERR_ARG);
  BMA_REQUIRE(a->B > 0 && a->L > 0 && a->Hq > 0 && a->Hkv >= 0 && a->d > 0, BMA_ERR_ARG);
  BMA_REQUIRE(a->d <= 256, BMA_ERR_UNSUPPORTED);
  BMA_REQUIRE(a->Hq <= 65535 && a->Hkv <= 65535, BMA_ERR_LIMIT);
  BMA_REQUIRE(!a->positions || a->position_bytes == 4 || a->position_bytes == 8, BMA_ERR_ARG);
  return validate_rotary(a->rotary, a->d);
}

HeadsParams rotate_params(const bma_rotate_args& a) {
  HeadsParams p{};
  p.B = a.B; p.L = a.L; p.d = a.d;
  p.frequencies = a.rotary.frequencies;
  p.magnitude = a.rotary.magnitude; p.eps = a.rotary.eps;
  p.weight_dtype = a.rotary.weight_dtype;
  p.positions = a.positions; p.position_bytes = a.position_bytes;
  p.position_stride_b = a.position_stride_b; p.position_stride_l = a.position_stride_l;
  return p;
}

// CTAs of the backward pass with weights: (q, k), in proportion to their heads; a side without a norm goes through heads_kernel.
// Four CTAs of four warps run on an SM.
void back_ctas(const bma_rotate_args& a, int& q, int& k) {
  const int hq = a.rotary.q_weight ? a.Hq : 0, hk = a.rotary.k_weight ? a.Hkv : 0;
  const int64_t tokens = (int64_t)a.B * a.L;
  const int64_t most = (tokens + kHeadsWarps - 1) / kHeadsWarps;
  const int64_t all = (int64_t)device_sms(current_device()) * 4;
  q = hq ? (int)std::max<int64_t>(1, std::min(most, all * hq / (hq + hk))) : 0;
  k = hk ? (int)std::max<int64_t>(1, std::min(most, all * hk / (hq + hk))) : 0;
}

}  // namespace

int rotate_forward(const bma_rotate_args* a, cudaStream_t st) {
  int rc = validate_rotate(a);
  if (rc != BMA_OK) return rc;
  if ((rc = validate_heads(a->q, a->q.dtype)) || (rc = validate_heads(a->q_out, a->q.dtype))) return rc;
  if (a->Hkv && ((rc = validate_heads(a->k, a->q.dtype)) || (rc = validate_heads(a->k_out, a->q.dtype)))) return rc;
  HeadsParams p = rotate_params(*a);
  p.side[0] = {a->q, a->q_out, a->rotary.q_weight, a->Hq, 1, 0};
  p.side[1] = {a->k, a->k_out, a->rotary.k_weight, a->Hkv, 1};
  const int vec = a->q.dtype == BMA_DTYPE_F32 ? 4 : 8;
  const bool wide = wide_heads(a->rotary, a->d, vec) && wide_tensor(a->q, vec) && wide_tensor(a->q_out, vec) &&
                    (!a->Hkv || (wide_tensor(a->k, vec) && wide_tensor(a->k_out, vec)));
  return a->q.dtype == BMA_DTYPE_F32 ? launch_heads<float, kRotate>(p, a->rotary, wide, st) : launch_heads<__nv_bfloat16, kRotate>(p, a->rotary, wide, st);
}

size_t rotate_back_bytes(const bma_rotate_args* a) {
  if (validate_rotate(a) != BMA_OK) return 0;
  int q, k;
  back_ctas(*a, q, k);
  return (size_t)(q + k) * a->d * sizeof(float);
}

int rotate_backward(const bma_rotate_args* a, void* workspace, size_t bytes, cudaStream_t st) {
  int rc = validate_rotate(a);
  if (rc != BMA_OK) return rc;
  const bool qn = a->rotary.q_weight, kn = a->Hkv && a->rotary.k_weight;
  const int dtype = a->q_out.dtype;
  if ((rc = validate_heads(a->q_out, dtype)) || (rc = validate_heads(a->dq, dtype)) || (qn && (rc = validate_heads(a->q, dtype)))) return rc;
  if (a->Hkv && ((rc = validate_heads(a->k_out, dtype)) || (rc = validate_heads(a->dk, dtype)) || (kn && (rc = validate_heads(a->k, dtype))))) return rc;
  BMA_REQUIRE((!qn || a->dq_weight) && (!kn || a->dk_weight), BMA_ERR_ARG);
  const int vec = dtype == BMA_DTYPE_F32 ? 4 : 8;
  const bool fits = wide_heads(a->rotary, a->d, vec);
  const bool q_wide = wide_tensor(a->q_out, vec) && wide_tensor(a->dq, vec) && (!qn || wide_tensor(a->q, vec));
  const bool k_wide = wide_tensor(a->k_out, vec) && wide_tensor(a->dk, vec) && (!kn || wide_tensor(a->k, vec));
  if (qn || kn) {
    BMA_REQUIRE(workspace && bytes >= rotate_back_bytes(a) && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0, BMA_ERR_WORKSPACE);
    BackParams p{};
    p.side[0] = {a->q, a->dq, a->rotary.q_weight, qn ? a->Hq : 0, 1};
    p.side[1] = {a->k, a->dk, a->rotary.k_weight, kn ? a->Hkv : 0, 1};
    p.g[0] = a->q_out; p.g[1] = a->k_out;
    p.B = a->B; p.L = a->L; p.d = a->d;
    p.frequencies = a->rotary.frequencies;
    p.magnitude = a->rotary.magnitude; p.eps = a->rotary.eps;
    p.weight_dtype = a->rotary.weight_dtype;
    p.positions = a->positions; p.position_bytes = a->position_bytes;
    p.position_stride_b = a->position_stride_b; p.position_stride_l = a->position_stride_l;
    p.partial = static_cast<float*>(workspace);
    int k_ctas;
    back_ctas(*a, p.q_ctas, k_ctas);
    BMA_REQUIRE((int64_t)a->B * a->L < (1ll << 30), BMA_ERR_LIMIT);
    const bool wide = fits && (!qn || q_wide) && (!kn || k_wide);
    p.map = head_map(a->rotary, a->d, wide ? vec : 1, 1);
    const unsigned ctas = (unsigned)(p.q_ctas + k_ctas);
    const bool full = a->rotary.dim == a->d, half = a->rotary.layout == BMA_ROTARY_HALF;
#define BMA_BACK(T)                                                                                                       \
  do {                                                                                                                    \
    if (!wide) rotate_back_kernel<T><<<ctas, kHeadsThreads, 0, st>>>(p);                                            \
    else if (half && full) rotate_back_wide_kernel<T, BMA_ROTARY_HALF, true><<<ctas, kHeadsThreads, 0, st>>>(p);          \
    else if (half) rotate_back_wide_kernel<T, BMA_ROTARY_HALF, false><<<ctas, kHeadsThreads, 0, st>>>(p);                 \
    else if (full) rotate_back_wide_kernel<T, BMA_ROTARY_INTERLEAVED, true><<<ctas, kHeadsThreads, 0, st>>>(p);           \
    else rotate_back_wide_kernel<T, BMA_ROTARY_INTERLEAVED, false><<<ctas, kHeadsThreads, 0, st>>>(p);                    \
  } while (0)
    if (dtype == BMA_DTYPE_F32) BMA_BACK(float);
    else BMA_BACK(__nv_bfloat16);
#undef BMA_BACK
    weight_sum_kernel<<<dim3(ceil_div(a->d, 32), 2), dim3(32, 32), 0, st>>>(p.partial, p.q_ctas, k_ctas, a->d, a->dq_weight, a->dk_weight, a->rotary.weight_dtype);
    count_launches(2);
    BMA_CUDA_TRY(cudaGetLastError());
  }
  if (!qn || (a->Hkv && !kn)) {      // sides without a norm: the rotation by the negative angle
    HeadsParams p = rotate_params(*a);
    p.back = 1;
    if (!qn) p.side[0] = {a->q_out, a->dq, nullptr, a->Hq, 1};
    if (a->Hkv && !kn) p.side[1] = {a->k_out, a->dk, nullptr, a->Hkv, 1};
    const bool wide = fits && (qn || q_wide) && (!p.side[1].heads || k_wide);
    return dtype == BMA_DTYPE_F32 ? launch_heads<float, kRotate>(p, a->rotary, wide, st) : launch_heads<__nv_bfloat16, kRotate>(p, a->rotary, wide, st);
  }
  return BMA_OK;
}

int append_kv(const bma_paged_cache* c, const bma_append_args* a, cudaStream_t st) {
  int rc = validate_cache(c);
  if (rc != BMA_OK) return rc;
  BMA_REQUIRE(a && a->T > 0 && a->Hq >= 0 && a->lengths, BMA_ERR_ARG);
  BMA_REQUIRE(a->Hq <= 65535, BMA_ERR_LIMIT);
  if ((rc = validate_rotary(a->rotary, c->d))) return rc;
  const int dtype = c->dtype == BMA_DTYPE_MXFP4 ? a->k.dtype : c->dtype;
  if ((rc = validate_heads(a->k, dtype)) || (rc = validate_heads(a->v, dtype))) return rc;
  if (a->Hq && ((rc = validate_heads(a->q, dtype)) || (rc = validate_heads(a->q_out, dtype)))) return rc;
  HeadsParams p{};
  p.B = c->B; p.L = a->T; p.d = c->d;
  p.frequencies = a->rotary.frequencies;
  p.magnitude = a->rotary.magnitude; p.eps = a->rotary.eps;
  p.weight_dtype = a->rotary.weight_dtype;
  p.side[0] = {a->q, a->q_out, a->rotary.q_weight, a->Hq, 1, 0};
  p.side[1] = {a->k, {}, a->rotary.k_weight, c->Hkv, 1};
  p.side[2] = {a->v, {}, nullptr, c->Hkv, 0};
  p.cache = *c;
  p.lengths = a->lengths; p.new_lengths = a->new_lengths;
  BMA_REQUIRE((p.status = device_status_ptr()) != nullptr, BMA_ERR_CUDA);
  const int vec = dtype == BMA_DTYPE_F32 ? 4 : 8;
  const bool wide = wide_heads(a->rotary, c->d, vec) && wide_tensor(a->k, vec) && wide_tensor(a->v, vec) &&
                    (!a->Hq || (wide_tensor(a->q, vec) && wide_tensor(a->q_out, vec)));
  if (c->dtype == BMA_DTYPE_MXFP4)
    return dtype == BMA_DTYPE_F32 ? launch_heads<float, kAppend4>(p, a->rotary, wide, st) : launch_heads<__nv_bfloat16, kAppend4>(p, a->rotary, wide, st);
  return dtype == BMA_DTYPE_F32 ? launch_heads<float, kAppend>(p, a->rotary, wide, st) : launch_heads<__nv_bfloat16, kAppend>(p, a->rotary, wide, st);
}

int read_kv(const bma_paged_cache* c, const int32_t* lengths, int L, const bma_tensor* k, const bma_tensor* v, cudaStream_t st) {
  int rc = validate_cache(c);
  if (rc != BMA_OK) return rc;
  BMA_REQUIRE(lengths && L > 0 && k && v, BMA_ERR_ARG);
  BMA_REQUIRE(L < (1ll << 31) - 4096, BMA_ERR_LIMIT);      // (as many as a table may cover; rounded up to kReadTokens it fits an int)
  const int dtype = c->dtype == BMA_DTYPE_F32 ? BMA_DTYPE_F32 : BMA_DTYPE_BF16, vec = dtype == BMA_DTYPE_F32 ? 4 : 8;
  if ((rc = validate_heads(*k, dtype)) || (rc = validate_heads(*v, dtype))) return rc;
  BMA_REQUIRE(wide_tensor(*k, vec) && wide_tensor(*v, vec), BMA_ERR_UNSUPPORTED);
  int* status = device_status_ptr();
  BMA_REQUIRE(status != nullptr, BMA_ERR_CUDA);
  const int per_token = c->Hkv * c->d / vec;
  const int x = per_token >= 256 ? 256 : ((per_token + 31) & ~31), y = 256 / x;
  const int64_t ctas = (int64_t)c->B * ((L + kReadTokens - 1) / kReadTokens);
  BMA_REQUIRE(ctas < (1ll << 31), BMA_ERR_LIMIT);
  const dim3 block(x, y);
  if (c->dtype == BMA_DTYPE_F32) read_kv_kernel<BMA_DTYPE_F32><<<(unsigned)ctas, block, 0, st>>>(*c, lengths, L, *k, *v, status);
  else if (c->dtype == BMA_DTYPE_BF16) read_kv_kernel<BMA_DTYPE_BF16><<<(unsigned)ctas, block, 0, st>>>(*c, lengths, L, *k, *v, status);
  else read_kv_kernel<BMA_DTYPE_MXFP4><<<(unsigned)ctas, block, 0, st>>>(*c, lengths, L, *k, *v, status);
  count_launches(1);
  BMA_CUDA_TRY(cudaGetLastError());
  return BMA_OK;
}

}  // namespace bma

using namespace bma;

extern "C" {
int bma_rotate(const bma_rotate_args* args, bma_stream_t stream) { return rotate_forward(args, static_cast<cudaStream_t>(stream)); }
size_t bma_rotate_bwd_workspace_bytes(const bma_rotate_args* args) { return rotate_back_bytes(args); }
int bma_rotate_bwd(const bma_rotate_args* args, void* workspace, size_t workspace_bytes, bma_stream_t stream) {
  return rotate_backward(args, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}
int bma_append_kv(const bma_paged_cache* cache, const bma_append_args* args, bma_stream_t stream) {
  return append_kv(cache, args, static_cast<cudaStream_t>(stream));
}
int bma_read_kv(const bma_paged_cache* cache, const int32_t* lengths, int32_t L, const bma_tensor* k, const bma_tensor* v, bma_stream_t stream) {
  return read_kv(cache, lengths, L, k, v, static_cast<cudaStream_t>(stream));
}
}
