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
  int wide_slots, tokens, heads, page_size;
};

// One vector per group of DIM / 8 lanes.
template <typename T, int DIM>
__global__ void __launch_bounds__(256) kv4_append_kernel(const CacheArgs a) {
  constexpr int LANES = DIM / 8;
  const long long vec = ((long long)blockIdx.x * 256 + threadIdx.x) / LANES;
  const int lane = threadIdx.x % LANES;
  const bool in_grid = vec < 2LL * a.tokens * a.heads;
  const int head = in_grid ? (int)(vec % a.heads) : 0;
  const int which = in_grid ? (int)(vec / a.heads & 1) : 0;
  const int token = in_grid ? (int)(vec / a.heads >> 1) : 0;
  const long long slot = in_grid ? slot_of(a.slots, a.wide_slots, token) : -1;
  const bool mine = slot >= 0 && slot < a.capacity;
  float x[8];
  float low = 0.0f, high = 0.0f;
  bool finite = true;
  if (mine) {
    const T* src = which ? reinterpret_cast<const T*>(a.x[1]) + token * a.x_token[1] + head * a.x_head[1]
                         : reinterpret_cast<const T*>(a.x[0]) + token * a.x_token[0] + head * a.x_head[0];
    const uint4 raw = *reinterpret_cast<const uint4*>(src + 8 * lane);
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_float<T>(e[i]);
    low = high = x[0];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      low = fminf(low, x[i]);
      high = fmaxf(high, x[i]);
      finite = finite && fabsf(x[i]) <= 3.402823466e38f;
    }
  }
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) {
    low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
    high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
  }
  const unsigned votes = __ballot_sync(0xffffffffu, finite);
  if (!mine) return;
  const unsigned group = LANES == 32 ? 0xffffffffu : ((1u << (LANES & 31)) - 1) << (threadIdx.x % 32 / LANES * LANES);
  const float range = high - low;
  const bool good = (votes & group) == group && range <= 3.402823466e38f;
  T scale_t = from_float<T>(__fdiv_rn(range, 15.0f));
  float scale = to_float<T>(scale_t);
  if (scale == 0.0f) scale = 1.0f;
  uint32_t word = 0;
  if (good) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float c = fminf(rintf(__fdiv_rn(x[i] - low, scale)), 15.0f);
      word |= (uint32_t)c << (4 * i);
    }
  } else {
    scale = low = __int_as_float(0x7fffffff);
  }
  const long long page = slot / a.page_size;
  const int row = (int)(slot % a.page_size);
  const long long at = ((page * 2 + which) * a.heads + head) * a.page_size + row;
  reinterpret_cast<uint32_t*>(a.codes + at * (DIM / 2))[lane] = word;
  if (lane == 0) {
    T pair[2] = {from_float<T>(scale), from_float<T>(low)};
    reinterpret_cast<uint32_t*>(a.params)[at] = *reinterpret_cast<uint32_t*>(pair);
  }
}

template <typename T, int DIM>
__global__ void __launch_bounds__(256) kv4_gather_kernel(const CacheArgs a) {
  constexpr int LANES = DIM / 8;
  const long long vec = ((long long)blockIdx.x * 256 + threadIdx.x) / LANES;
  const int lane = threadIdx.x % LANES;
  if (vec >= 2LL * a.tokens * a.heads) return;
  const int head = (int)(vec % a.heads), which = (int)(vec / a.heads & 1), token = (int)(vec / a.heads >> 1);
  const long long slot = slot_of(a.slots, a.wide_slots, token);
  uint4 raw = make_uint4(0, 0, 0, 0);
  if (slot >= 0 && slot < a.capacity) {
    const long long at = ((slot / a.page_size * 2 + which) * a.heads + head) * a.page_size + slot % a.page_size;
    const uint32_t word = reinterpret_cast<const uint32_t*>(a.codes + at * (DIM / 2))[lane];
    const uint32_t bits = reinterpret_cast<const uint32_t*>(a.params)[at];
    const T* pair = reinterpret_cast<const T*>(&bits);
    const float scale = to_float<T>(pair[0]), low = to_float<T>(pair[1]);
    T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = from_float<T>((float)(word >> (4 * i) & 15u) * scale + low);
  }
  reinterpret_cast<uint4*>(reinterpret_cast<T*>(which ? a.out[1] : a.out[0]) + ((long long)token * a.heads + head) * DIM)[lane] = raw;
}

template <typename T, int DIM>
int launch(const CacheArgs& a, bool append, cudaStream_t stream) {
  const long long threads = 2LL * a.tokens * a.heads * (DIM / 8);
  const long long grid = (threads + 255) / 256;
  XQT_REQUIRE(grid < (1LL << 31) - 1);
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
  return tokens >= 0 && heads >= 1 && heads <= (1 << 16) && (dim == 64 || dim == 128 || dim == 256) && pages >= 0 && page_size >= 1 &&
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
  return dispatch(a, dim, dtype, false, stream);
}
