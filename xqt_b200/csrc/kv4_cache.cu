// A paged cache of keys and values in 4 bits: writing vectors into it and reading them back.
//
// One vector (a key or value of one token and head) is held as codes c of 4 bits and a pair (scale s, minimum m) in the
// activation type T:  m = min x,  s = T((max x - min x) / 15), 1 where that is 0,  c = clamp(rint((x - m) / s), 0, 15),
// and stands for c * s + m.  The codes are taken against the rounded s, so its rounding costs nothing but the clamp.  A vector
// that holds an infinity or a NaN (or whose range overflows) gets s = m = NaN and stands for NaN.
//
//   codes  uint8 [pages, 2 (key, value), heads, page_size, dim / 2]   low nibble = even channel
//   params T     [pages, 2, heads, page_size, 2]                      (scale, minimum)
//
// A head's tokens of one page are contiguous in both, so attention fetches them with one bulk copy each.  Both kernels are bound
// by HBM (2 * dim bytes in, dim / 2 + 4 out, or the reverse); 8 channels a lane: one 16-byte access to the vector, one
// 4-byte access to the codes.
#include <type_traits>

#include "common.cuh"

namespace xqt_b200 {

namespace {

__device__ __forceinline__ long long slot_of(const void* slots, int wide, int token) {
  return wide ? reinterpret_cast<const long long*>(slots)[token] : (long long)reinterpret_cast<const int*>(slots)[token];
}

struct CacheArgs {
  const void* x[2];                 // keys, values (append)
  void* out[2];                     // keys, values (gather)
  long long x_token[2], x_head[2];  // strides of x, in elements
  uint8_t* codes;
  void* params;
  const void* slots;
  long long capacity;               // pages * page_size
  int wide_slots, tokens, heads, page_size, page_shift;
};

template <typename T>
struct Pair;
template <>
struct Pair<__half> {
  using type = __half2;
};
template <>
struct Pair<__nv_bfloat16> {
  using type = __nv_bfloat162;
};
__device__ __forceinline__ float2 floats(__half2 v) { return __half22float2(v); }
__device__ __forceinline__ float2 floats(__nv_bfloat162 v) { return __bfloat1622float2(v); }
__device__ __forceinline__ __half2 lows(__half2 a, __half2 b) { return __lows2half2(a, b); }
__device__ __forceinline__ __nv_bfloat162 lows(__nv_bfloat162 a, __nv_bfloat162 b) { return __lows2bfloat162(a, b); }
__device__ __forceinline__ __half2 highs(__half2 a, __half2 b) { return __highs2half2(a, b); }
__device__ __forceinline__ __nv_bfloat162 highs(__nv_bfloat162 a, __nv_bfloat162 b) { return __highs2bfloat162(a, b); }
__device__ __forceinline__ __half2 rounded(float a, float b, __half) { return __floats2half2_rn(a, b); }
__device__ __forceinline__ __nv_bfloat162 rounded(float a, float b, __nv_bfloat16) { return __floats2bfloat162_rn(a, b); }

// One vector per group of DIM / 8 lanes, two groups' worth of vectors per thread.  Minimum and maximum on packed pairs as they come, the minimum
// negated so that both are maxima, NaN kept.  The division is a product with the reciprocal, which is off by less than 2^-19 of a code: the
// quotients that close to half a code are divided.
template <typename T, int DIM>
__global__ void __launch_bounds__(256) kv4_append_kernel(const CacheArgs a) {
  constexpr int LANES = DIM / 8, kBatch = 2, kGroups = 256 / LANES;
  constexpr float kHalf = 0.5f - 1.0f / 65536.0f, kMagic = 12582912.0f, kMost = 3.402823466e38f;     // kMagic: 1.5 * 2^23, rounds to whole numbers
  constexpr float kNormal = std::is_same<T, __half>::value ? 6.103515625e-05f : 1e-30f;
  using P = typename Pair<T>::type;
  const int lane = threadIdx.x % LANES;
  const unsigned first = blockIdx.x * (kBatch * kGroups) + threadIdx.x / LANES, count = 2u * a.tokens * a.heads;
  uint4 raw[kBatch];
  long long at[kBatch];
#pragma unroll
  for (int b = 0; b < kBatch; ++b) {
    const unsigned vec = first + b * kGroups;
    at[b] = -1;
    raw[b] = make_uint4(0, 0, 0, 0);
    if (vec < count) {
      const unsigned row = vec / (unsigned)a.heads;                // token and which
      const int head = (int)(vec - row * a.heads), which = row & 1, token = (int)(row >> 1);
      const long long slot = slot_of(a.slots, a.wide_slots, token);
      if (slot >= 0 && slot < a.capacity) {
        const T* src = which ? reinterpret_cast<const T*>(a.x[1]) + token * a.x_token[1] + head * a.x_head[1]
                             : reinterpret_cast<const T*>(a.x[0]) + token * a.x_token[0] + head * a.x_head[0];
        raw[b] = *reinterpret_cast<const uint4*>(src + 8 * lane);
        at[b] = (((slot >> a.page_shift) * 2 + which) * a.heads + head) * a.page_size + (slot & (a.page_size - 1));
      }
    }
  }
#pragma unroll
  for (int b = 0; b < kBatch; ++b) {
    const P* const e = reinterpret_cast<const P*>(&raw[b]);
    const P high2 = __hmax2_nan(__hmax2_nan(e[0], e[1]), __hmax2_nan(e[2], e[3])), low2 = __hneg2(__hmin2_nan(__hmin2_nan(e[0], e[1]), __hmin2_nan(e[2], e[3])));
    P both = __hmax2_nan(lows(high2, low2), highs(high2, low2));      // (maximum, -minimum)
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) {
      const uint32_t other = __shfl_xor_sync(0xffffffffu, *reinterpret_cast<const uint32_t*>(&both), o);
      both = __hmax2_nan(both, *reinterpret_cast<const P*>(&other));
    }
    if (at[b] < 0) continue;
    const float high = floats(both).x;
    float low = -floats(both).y;
    const float range = high - low;
    const bool good = range <= kMost && fabsf(low) <= kMost && fabsf(high) <= kMost;     // no NaN, no infinity
    float scale = to_float<T>(from_float<T>(__fdiv_rn(range, 15.0f)));
    if (scale == 0.0f) scale = 1.0f;
    float x[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = floats(e[i]);
      x[2 * i] = f.x - low;
      x[2 * i + 1] = f.y - low;
    }
    const float inverse = __fdiv_rn(1.0f, scale);
    float code[8], near = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float q = x[i] * inverse, r = (q + kMagic) - kMagic;
      code[i] = r;
      near = fmaxf(near, fabsf(q - r));
    }
    // a scale that is a normal number is too low by 2^-8 of itself at most, so no quotient reaches 15.5; the others are divided and clamped
    if (near > kHalf || !(scale >= kNormal)) {
#pragma unroll
      for (int i = 0; i < 8; ++i) code[i] = fminf(rintf(__fdiv_rn(x[i], scale)), 15.0f);
    }
    uint32_t word;
    if (good) {                                      // 16 bits at a time are exact in fp32
      const float even = fmaf(code[3], 4096.0f, fmaf(code[2], 256.0f, fmaf(code[1], 16.0f, code[0])));
      const float odd = fmaf(code[7], 4096.0f, fmaf(code[6], 256.0f, fmaf(code[5], 16.0f, code[4])));
      word = __byte_perm(__float_as_uint(even + 8388608.0f), __float_as_uint(odd + 8388608.0f), 0x5410);
    } else {
      word = 0;
      scale = low = __int_as_float(0x7fffffff);
    }
    reinterpret_cast<uint32_t*>(a.codes + at[b] * (DIM / 2))[lane] = word;
    if (lane == 0) {
      const P pair = rounded(scale, low, T());
      reinterpret_cast<uint32_t*>(a.params)[at[b]] = *reinterpret_cast<const uint32_t*>(&pair);
    }
  }
}

template <typename T, int DIM>
__global__ void __launch_bounds__(256) kv4_gather_kernel(const CacheArgs a) {
  constexpr int LANES = DIM / 8, kBatch = 2, kGroups = 256 / LANES;
  using P = typename Pair<T>::type;
  const int lane = threadIdx.x % LANES;
  const unsigned first = blockIdx.x * (kBatch * kGroups) + threadIdx.x / LANES, count = 2u * a.tokens * a.heads;
  uint32_t word[kBatch], bits[kBatch];
  T* dst[kBatch];
#pragma unroll
  for (int b = 0; b < kBatch; ++b) {
    const unsigned vec = first + b * kGroups;
    word[b] = bits[b] = 0;                           // a slot outside reads 0 * 0 + 0
    dst[b] = nullptr;
    if (vec < count) {
      const unsigned row = vec / (unsigned)a.heads;
      const int head = (int)(vec - row * a.heads), which = row & 1, token = (int)(row >> 1);
      const long long slot = slot_of(a.slots, a.wide_slots, token);
      dst[b] = reinterpret_cast<T*>(which ? a.out[1] : a.out[0]) + ((long long)token * a.heads + head) * DIM;
      if (slot >= 0 && slot < a.capacity) {
        const long long at = (((slot >> a.page_shift) * 2 + which) * a.heads + head) * a.page_size + (slot & (a.page_size - 1));
        word[b] = reinterpret_cast<const uint32_t*>(a.codes + at * (DIM / 2))[lane];
        bits[b] = reinterpret_cast<const uint32_t*>(a.params)[at];
      }
    }
  }
#pragma unroll
  for (int b = 0; b < kBatch; ++b) {
    if (dst[b] == nullptr) continue;
    const float2 p = floats(*reinterpret_cast<const P*>(&bits[b]));
    // a byte under the exponent of 2^23 is 2^23 + code; code * scale is exact
    const uint32_t even = word[b] & 0x0f0f0f0fu, odd = word[b] >> 4 & 0x0f0f0f0fu;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = fmaf(__uint_as_float(__byte_perm(i & 1 ? odd : even, 0x4b000000u, 0x7440 + (i >> 1))) - 8388608.0f, p.x, p.y);
    P r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = rounded(v[2 * i], v[2 * i + 1], T());
    reinterpret_cast<uint4*>(dst[b])[lane] = *reinterpret_cast<const uint4*>(r);
  }
}

template <typename T, int DIM>
int launch(const CacheArgs& a, bool append, cudaStream_t stream) {
  const long long vectors = 2LL * a.tokens * a.heads, of_block = 2 * (256 / (DIM / 8));
  const long long grid = (vectors + of_block - 1) / of_block;
  if (append)
    kv4_append_kernel<T, DIM><<<(unsigned)grid, 256, 0, stream>>>(a);
  else
    kv4_gather_kernel<T, DIM><<<(unsigned)grid, 256, 0, stream>>>(a);
  return launch_status();
}

int dispatch(const CacheArgs& a, int dim, int dtype, bool append, cudaStream_t stream) {
  if (dtype == XQT_B200_BF16) {
    if (dim == 64) return launch<__nv_bfloat16, 64>(a, append, stream);
    if (dim == 128) return launch<__nv_bfloat16, 128>(a, append, stream);
    return launch<__nv_bfloat16, 256>(a, append, stream);
  }
  if (dim == 64) return launch<__half, 64>(a, append, stream);
  if (dim == 128) return launch<__half, 128>(a, append, stream);
  return launch<__half, 256>(a, append, stream);
}

bool served(int tokens, int heads, int dim, long long pages, int page_size, int dtype) {
  return tokens >= 0 && heads >= 1 && heads <= (1 << 16) && (dim == 64 || dim == 128 || dim == 256) && pages >= 0 && page_size >= 16 && page_size <= 4096 &&
         (page_size & (page_size - 1)) == 0 && 2LL * tokens * heads < (1LL << 31) &&
         (dtype == XQT_B200_FP16 || dtype == XQT_B200_BF16);
}

}  // namespace
}  // namespace xqt_b200

extern "C" int xqt_b200_kv4_append(const void* k, const void* v, void* codes, void* params, const void* slots, const long long* strides, int tokens,
                                   int heads, int dim, long long pages, int page_size, int wide_slots, int dtype, cudaStream_t stream) {
  using namespace xqt_b200;
  XQT_REQUIRE(served(tokens, heads, dim, pages, page_size, dtype));
  if (tokens == 0 || pages == 0) return 0;
  XQT_REQUIRE(k && v && codes && params && slots && strides);
  XQT_REQUIRE((((uintptr_t)k | (uintptr_t)v) & 15) == 0 && (((uintptr_t)codes | (uintptr_t)params) & 3) == 0);
  XQT_REQUIRE(((strides[0] | strides[1] | strides[2] | strides[3]) & 7) == 0);
  CacheArgs a = {};
  a.x[0] = k;
  a.x[1] = v;
  a.x_token[0] = strides[0];
  a.x_head[0] = strides[1];
  a.x_token[1] = strides[2];
  a.x_head[1] = strides[3];
  a.codes = (uint8_t*)codes;
  a.params = params;
  a.slots = slots;
  a.capacity = pages * page_size;
  a.wide_slots = wide_slots;
  a.tokens = tokens;
  a.heads = heads;
  a.page_size = page_size;
  a.page_shift = __builtin_ctz((unsigned)page_size);
  return dispatch(a, dim, dtype, true, stream);
}

extern "C" int xqt_b200_kv4_gather(const void* codes, const void* params, const void* slots, void* k_out, void* v_out, int tokens, int heads, int dim,
                                   long long pages, int page_size, int wide_slots, int dtype, cudaStream_t stream) {
  using namespace xqt_b200;
  XQT_REQUIRE(served(tokens, heads, dim, pages, page_size, dtype));
  if (tokens == 0) return 0;
  XQT_REQUIRE(slots && k_out && v_out && (pages == 0 || (codes && params)));
  XQT_REQUIRE((((uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0 && (((uintptr_t)codes | (uintptr_t)params) & 3) == 0);
  CacheArgs a = {};
  a.out[0] = k_out;
  a.out[1] = v_out;
  a.codes = (uint8_t*)codes;
  a.params = (void*)params;
  a.slots = slots;
  a.capacity = pages * page_size;
  a.wide_slots = wide_slots;
  a.tokens = tokens;
  a.heads = heads;
  a.page_size = page_size;
  a.page_shift = __builtin_ctz((unsigned)page_size);
  return dispatch(a, dim, dtype, false, stream);
}
