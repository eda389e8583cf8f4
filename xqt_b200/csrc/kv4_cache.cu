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
// A head's tokens of one page are contiguous in both, so attention fetches them with one bulk copy each.  Both kernels move
// 2 * dim bytes one way and dim / 2 + 4 the other.  A lane takes the same channels of a token's key and value: what it computes
// once (the place in the cache, by multiplication) serves both, and both loads are in flight together.  An append is bound by the issue of
// instructions before HBM (minimum, maximum, rounding, the test for halves, packing), so minimum and maximum run on packed pairs as they
// come, everything else on packed fp32, and nothing divides.  Measured, 16,001 tokens of 8 heads of 128 channels: append fp16 19.5 us, bf16 20.5
// (83 MB: 4.2 TB/s; with divisions 8 channels a lane and keys apart from values 36), gather 15 us (5.6 TB/s, HBM); up to 256 tokens 2.3 to 2.7 us.
#include <type_traits>

#include "pairs.cuh"

namespace xqt_b200 {

namespace {

using sm100::Two;
using sm100::fma2;

struct CacheArgs {
  const void* x[2];                 // keys, values (append)
  void* out[2];                     // keys, values (gather)
  long long x_token[2], x_head[2];  // strides of x, in elements
  uint8_t* codes;
  void* params;
  const void* slots;
  long long capacity;               // pages * page_size
  int wide_slots, tokens, heads, page_size, page_shift;
  unsigned heads_factor, heads_shift;   // n / heads = n * factor >> shift for n < 2^31
};

// Where vector `item` (token * heads + head) stands: its key's place in the cache (-1: nowhere); its value's is heads * page_size further.
__device__ __forceinline__ long long place_of(const CacheArgs& a, unsigned item, int& token, int& head) {
  token = (int)((unsigned long long)item * a.heads_factor >> a.heads_shift);
  head = (int)item - token * a.heads;
  const long long slot = a.wide_slots ? reinterpret_cast<const long long*>(a.slots)[token] : (long long)reinterpret_cast<const int*>(a.slots)[token];
  if ((unsigned long long)slot >= (unsigned long long)a.capacity) return -1;
  const unsigned page = (unsigned)(slot >> a.page_shift), in_page = (unsigned)slot & (unsigned)(a.page_size - 1);
  return (long long)page * (2LL * a.heads * a.page_size) + ((long long)head * a.page_size + in_page);
}

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

// x / 15, rounded as the division is: the product with 1 / 15 and one correction (equal for each of the 2^23 mantissas; where the correction
// would be subnormal, the division).
__device__ __forceinline__ float fifteenth(float x) {
  constexpr float k = 1.0f / 15.0f;
  const float q = x * k;
  return x < 1e-28f ? __fdiv_rn(x, 15.0f) : fmaf(fmaf(-15.0f, q, x), k, q);
}
__device__ __forceinline__ float reciprocal(float x) {         // to 2^-23 of itself
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

// The key and the value of one token and head per group of DIM / 16 lanes (16 channels a lane: what is computed once per lane, the place
// and the scale, is a third of the work at 8).  Minimum and maximum on packed pairs as they come, the minimum negated so that both
// are maxima, NaN kept.  The division is a product with the reciprocal, which is off by less than 2^-18 of a code: the
// quotients that close to half a code are looked at again.
template <typename T, int DIM>
__global__ void __launch_bounds__(256) kv4_append_kernel(const CacheArgs a) {
  constexpr int LANES = DIM / 16, kGroups = 256 / LANES;
  constexpr float kHalf = 0.5f - 1.0f / 65536.0f, kMagic = 12582912.0f, kMost = 3.402823466e38f;     // kMagic: 1.5 * 2^23, rounds to whole numbers
  constexpr float kNormal = std::is_same<T, __half>::value ? 6.103515625e-05f : 1e-30f;
  using P = typename Pair<T>::type;
  const int lane = threadIdx.x % LANES;
  const unsigned item = blockIdx.x * kGroups + threadIdx.x / LANES;
  long long at = -1;
  uint4 raw[2][2] = {};
  sm100::grid_launch_dependents();
  sm100::grid_dependency_wait();
  if (item < (unsigned)a.tokens * a.heads) {
    int token, head;
    at = place_of(a, item, token, head);
    if (at >= 0) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const uint4* const src = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.x[b]) + token * a.x_token[b] + head * a.x_head[b] + 16 * lane);
        raw[b][0] = src[0];
        raw[b][1] = src[1];
      }
    }
  }
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const P* const e = reinterpret_cast<const P*>(raw[b]);
    P high2 = e[0], low2 = e[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) {
      high2 = __hmax2_nan(high2, e[i]);
      low2 = __hmin2_nan(low2, e[i]);
    }
    low2 = __hneg2(low2);
    P both = __hmax2_nan(lows(high2, low2), highs(high2, low2));      // (maximum, -minimum)
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) {
      const uint32_t other = __shfl_xor_sync(0xffffffffu, *reinterpret_cast<const uint32_t*>(&both), o);
      both = __hmax2_nan(both, *reinterpret_cast<const P*>(&other));
    }
    if (at < 0) continue;
    const float high = floats(both).x;
    float low = -floats(both).y;
    const float range = high - low;
    const bool good = range <= kMost && fabsf(low) <= kMost && fabsf(high) <= kMost;     // no NaN, no infinity
    float scale = to_float<T>(from_float<T>(fifteenth(range)));
    if (scale == 0.0f) scale = 1.0f;
    const Two inverse(reciprocal(scale)), minus(-low);
    uint32_t word[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      Two x[4], code[4];
      float near = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = floats(e[4 * h + i]);
        x[i] = Two(f.x, f.y) + minus;
        code[i] = fma2(x[i], inverse, Two(kMagic)) + Two(-kMagic);
        const float2 off = fma2(x[i], inverse, code[i] * Two(-1.0f)).both();
        near = fmaxf(near, fmaxf(fabsf(off.x), fabsf(off.y)));
      }
      // A scale that is a normal number is too low by 2^-8 of itself at most, so no quotient reaches 15.5.  Near a half the quotient is corrected
      // once, which rounds it as the division does: the remainder is exact, the correction good to 2^-20 of a step, and a quotient by the
      // 8 or 11 bits of a scale is at least 2^-12 of a step away from where rounding turns.  Bf16 vectors stand on halves often.
      if (near > kHalf) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const Two q = x[i] * inverse;
          code[i] = fma2(fma2(q, Two(-scale), x[i]), inverse, q) + Two(kMagic) + Two(-kMagic);
        }
      }
      if (!(scale >= kNormal)) {                       // divided and clamped
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = x[i].both();
          code[i] = Two(fminf(rintf(__fdiv_rn(f.x, scale)), 15.0f), fminf(rintf(__fdiv_rn(f.y, scale)), 15.0f));
        }
      }
      // 16 bits at a time are exact in fp32; 2^23 puts them in the low bits
      const float2 lo = fma2(code[1], Two(256.0f), code[0]).both(), hi = fma2(code[3], Two(256.0f), code[2]).both();
      word[h] = __byte_perm(__float_as_uint(fmaf(lo.y, 16.0f, lo.x) + 8388608.0f), __float_as_uint(fmaf(hi.y, 16.0f, hi.x) + 8388608.0f), 0x5410);
    }
    if (!good) {
      word[0] = word[1] = 0;
      scale = low = __int_as_float(0x7fffffff);
    }
    const long long to = at + (b ? (long long)a.heads * a.page_size : 0);
    reinterpret_cast<uint2*>(a.codes + to * (DIM / 2))[lane] = make_uint2(word[0], word[1]);
    if (lane == 0) {
      const P pair = rounded(scale, low, T());
      reinterpret_cast<uint32_t*>(a.params)[to] = *reinterpret_cast<const uint32_t*>(&pair);
    }
  }
}

template <typename T, int DIM>
__global__ void __launch_bounds__(256) kv4_gather_kernel(const CacheArgs a) {
  constexpr int LANES = DIM / 8, kGroups = 256 / LANES;
  using P = typename Pair<T>::type;
  const int lane = threadIdx.x % LANES;
  const unsigned item = blockIdx.x * kGroups + threadIdx.x / LANES;
  sm100::grid_launch_dependents();
  sm100::grid_dependency_wait();
  if (item >= (unsigned)a.tokens * a.heads) return;
  int token, head;
  const long long at = place_of(a, item, token, head);
  uint32_t word[2] = {}, bits[2] = {};               // a slot outside reads 0 * 0 + 0
  if (at >= 0) {
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const long long from = at + (b ? (long long)a.heads * a.page_size : 0);
      word[b] = reinterpret_cast<const uint32_t*>(a.codes + from * (DIM / 2))[lane];
      bits[b] = reinterpret_cast<const uint32_t*>(a.params)[from];
    }
  }
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const float2 p = floats(*reinterpret_cast<const P*>(&bits[b]));
    // a byte under the exponent of 2^23 is 2^23 + code; code * scale is exact
    const uint32_t even = word[b] & 0x0f0f0f0fu, odd = word[b] >> 4 & 0x0f0f0f0fu;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = fmaf(__uint_as_float(__byte_perm(i & 1 ? odd : even, 0x4b000000u, 0x7440 + (i >> 1))) - 8388608.0f, p.x, p.y);
    P r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = rounded(v[2 * i], v[2 * i + 1], T());
    reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.out[b]) + (long long)item * DIM)[lane] = *reinterpret_cast<const uint4*>(r);
  }
}

template <typename T, int DIM>
int launch(const CacheArgs& a, bool append, cudaStream_t stream) {
  const int of_block = 256 / (DIM / (append ? 16 : 8));
  const long long grid = ((long long)a.tokens * a.heads + of_block - 1) / of_block;
  return append ? launch_pdl(kv4_append_kernel<T, DIM>, dim3((unsigned)grid), dim3(256), 0, stream, a)
                : launch_pdl(kv4_gather_kernel<T, DIM>, dim3((unsigned)grid), dim3(256), 0, stream, a);
}

int dispatch(CacheArgs a, int dim, int dtype, bool append, cudaStream_t stream) {
  int bits = 0;
  while ((1 << bits) < a.heads) ++bits;
  a.heads_shift = 31 + bits;
  a.heads_factor = (unsigned)(((1ULL << a.heads_shift) + a.heads - 1) / a.heads);
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
  return tokens >= 0 && heads >= 1 && heads <= (1 << 16) && (dim == 64 || dim == 128 || dim == 256) && pages >= 0 && pages < (1LL << 31) && page_size >= 16 && page_size <= 4096 &&
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
  XQT_REQUIRE((((uintptr_t)k | (uintptr_t)v) & 15) == 0 && ((uintptr_t)codes & 7) == 0 && ((uintptr_t)params & 3) == 0);
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
