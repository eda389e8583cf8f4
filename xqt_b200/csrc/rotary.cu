// RMS norm of query and key heads and the position rotation, in one pass.
//
//   y = x * rsqrt(mean(x^2) + eps) * w          (no weight: y = x)
//   pair j of the first `rotary` channels -- (j, j + rotary/2), or (2j, 2j+1) where they are interleaved -- turns by
//   position[axis_j, token] * frequency_j; the other channels pass.  fp32 arithmetic, one rounding.
//
// The angle is kept as a 64-bit fixed-point fraction of a turn: position * fraction wraps exactly modulo one turn.  What is left is the rounding of
// frequency / (2 pi) to 64-bit floating point, at most 2^-53 * |position| turns (for frequencies up to a turn per position): below the fp32 of sine and cosine for every 32-bit position (fp32
// angles are off by 2^-24 of the angle itself: 0.006 rad at position 100,000).
//
// Bound by HBM: every channel is read and written once.  A block makes the cosines of up to 16 tokens in shared memory, then its lane groups go
// through the heads of those tokens: dim / 16 lanes (padded to a power of two) hold one head, 16 channels a lane, chosen so that both
// channels of a pair are in one lane.  Sums of squares, products and turns are packed fp32 instructions: with single ones the kernel waited on issue.
// Measured, heads of 128 channels: 8191 tokens of 32 + 8 heads 31 us (5.4 TB/s), 32,760 tokens of 20 + 20 heads on three axes 120 us (5.6 TB/s,
// a copy reaches 6.6; 131 us where the inputs change from call to call); a call of one token 3.1 us, which is its launch and one chain load -> sum -> store.
#include "pairs.cuh"

namespace xqt_b200 {

namespace {

using sm100::Two;
using sm100::fma2;

struct RopeArgs {
  const void* x[2];        // queries, keys
  void* out[2];
  const void* weight[2];   // [dim] or null
  long long x_token[2], x_head[2], o_token[2], o_head[2];   // strides, in elements
  int heads[2];
  const void* positions;   // [axes, tokens] of int32 or int64
  long long p_axis, p_token;
  const double* frequencies;   // [rotary / 2], radians per position
  const int* axes;             // [rotary / 2] or null (all 0)
  int axis_count, wide_positions, weight_dtype;
  int tokens, dim, rotary, block_tokens;
  float eps;
};

// eight channels as packed pairs, and back (one conversion per pair)
__device__ __forceinline__ Two unpack2(uint32_t v, __half) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v));
  return Two(f.x, f.y);
}
__device__ __forceinline__ Two unpack2(uint32_t v, __nv_bfloat16) { return Two(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u)); }
__device__ __forceinline__ uint32_t pack2(Two v, __half) {
  const float2 f = v.both();
  const __half2 h = __floats2half2_rn(f.x, f.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(Two v, __nv_bfloat16) {
  const float2 f = v.both();
  const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ void unpack8(const uint4& v, Two (&f)[4]) {
  f[0] = unpack2(v.x, T());
  f[1] = unpack2(v.y, T());
  f[2] = unpack2(v.z, T());
  f[3] = unpack2(v.w, T());
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const Two (&f)[4]) {
  return make_uint4(pack2(f[0], T()), pack2(f[1], T()), pack2(f[2], T()), pack2(f[3], T()));
}

constexpr int kThreads = 256, kPerSm = 4, kMostTokens = 16;      // kPerSm: blocks on an SM

// The two runs of 8 channels of lane l.
template <bool INTERLEAVED>
__device__ __forceinline__ void runs(const RopeArgs& a, int l, int& c0, int& c1) {
  if (INTERLEAVED || a.rotary == 0) {
    c0 = 16 * l;
    c1 = c0 + 8;
  } else if (l < a.rotary / 16) {
    c0 = 8 * l;
    c1 = c0 + a.rotary / 2;
  } else {
    c0 = a.rotary + 8 * (l - a.rotary / 16);
    c1 = c0 + (a.dim - a.rotary) / 2;
  }
}

// LANES: lanes of a head, a power of two; lanes past dim / 16 only take part in the sums.
template <typename T, int LANES, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads, kPerSm) rope_kernel(const RopeArgs a) {
  // four floats of every lane side by side, so that a quarter warp reads 128 contiguous bytes: pair 8 l + 4 h + i at 4 (l + 16 h) + i, and the
  // lane's channel e of run r at 4 (l + 16 (2 r + e / 4)) + e % 4
  __shared__ __align__(16) float s_cos[kMostTokens][128], s_sin[kMostTokens][128], s_weight[2][256];
  sm100::grid_launch_dependents();          // (the next kernel's launch under this one's end: 8191 tokens, calls back to back, 31.5 us, without 33.1)
  sm100::grid_dependency_wait();
  const int pairs = a.rotary / 2, token0 = blockIdx.x * a.block_tokens, block_tokens = min(a.block_tokens, a.tokens - token0);
  for (int i = threadIdx.x; i < block_tokens * pairs; i += kThreads) {
    const int token = i / pairs, pair = i - token * pairs, spot = 4 * ((pair >> 3) + 16 * (pair >> 2 & 1)) + (pair & 3);
    int axis = a.axes ? a.axes[pair] : 0;
    axis = axis < 0 ? 0 : (axis >= a.axis_count ? a.axis_count - 1 : axis);
    const long long at = axis * a.p_axis + (token0 + token) * a.p_token;
    const long long position = a.wide_positions ? reinterpret_cast<const long long*>(a.positions)[at] : (long long)reinterpret_cast<const int*>(a.positions)[at];
    double turn = a.frequencies[pair] * 0.15915494309189533577;   // 1 / (2 pi)
    turn -= floor(turn);
    const unsigned long long fraction = __double2ull_rn(turn * 18446744073709551616.0);
    const unsigned long long angle = fraction * (unsigned long long)position;
    sincospif((float)(int)(angle >> 32) * 4.656612873077393e-10f, &s_sin[token][spot], &s_cos[token][spot]);   // 2^-31: half turns
  }
  const bool normed = a.weight[0] != nullptr || a.weight[1] != nullptr;     // uniform: then every lane of a warp takes part in the sums
  if (normed) {
    for (int i = threadIdx.x; i < 2 * a.dim; i += kThreads) {
      const int which = i >= a.dim, at = which ? i - a.dim : i, owner = at >> 4, run = at >> 3 & 1, e = at & 7;
      const void* weight = which ? a.weight[1] : a.weight[0];
      int c0, c1;
      runs<INTERLEAVED>(a, owner, c0, c1);
      s_weight[which][4 * (owner + 16 * (2 * run + (e >> 2))) + (e & 3)] = weight != nullptr ? load_param(weight, a.weight_dtype, (run ? c1 : c0) + e) : 1.0f;
    }
  }
  __syncthreads();

  constexpr int kGroups = kThreads / LANES, kBatch = 2;      // heads of a group loaded before the first is worked on
  const int lane = threadIdx.x % LANES, all = a.heads[0] + a.heads[1];
  const bool active = lane < a.dim / 16, turns = lane < a.rotary / 16;
  int c0, c1;
  runs<INTERLEAVED>(a, lane, c0, c1);
  const float inv_dim = 1.0f / (float)a.dim;
  int token = 0, head = threadIdx.x / LANES;
  for (int item = 0; item < block_tokens * all; item += kBatch * kGroups) {
    uint4 raw[kBatch][2];
    T* dst[kBatch];
    int of[kBatch], which[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      while (head >= all) {
        head -= all;
        ++token;
      }
      of[b] = token;
      which[b] = head >= a.heads[0];
      raw[b][0] = raw[b][1] = make_uint4(0, 0, 0, 0);
      dst[b] = nullptr;
      if (active && token < block_tokens) {
        const long long row = token0 + token, h = which[b] ? head - a.heads[0] : head;
        const T* src = which[b] ? reinterpret_cast<const T*>(a.x[1]) + row * a.x_token[1] + h * a.x_head[1]
                                : reinterpret_cast<const T*>(a.x[0]) + row * a.x_token[0] + h * a.x_head[0];
        dst[b] = which[b] ? reinterpret_cast<T*>(a.out[1]) + row * a.o_token[1] + h * a.o_head[1]
                          : reinterpret_cast<T*>(a.out[0]) + row * a.o_token[0] + h * a.o_head[0];
        raw[b][0] = *reinterpret_cast<const uint4*>(src + c0);
        raw[b][1] = *reinterpret_cast<const uint4*>(src + c1);
      }
      head += kGroups;
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      Two u[4], v[4];
      unpack8<T>(raw[b][0], u);
      unpack8<T>(raw[b][1], v);
      if (normed) {
        Two squares(0.0f);
#pragma unroll
        for (int i = 0; i < 4; ++i) squares = fma2(u[i], u[i], fma2(v[i], v[i], squares));
        float sum = squares.both().x + squares.both().y;
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (dst[b] != nullptr && (which[b] ? a.weight[1] : a.weight[0]) != nullptr) {
          const Two r(rsqrtf(sum * inv_dim + a.eps));
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float4 w0 = *reinterpret_cast<const float4*>(&s_weight[which[b]][4 * (lane + 16 * h)]), w1 = *reinterpret_cast<const float4*>(&s_weight[which[b]][4 * (lane + 16 * (2 + h))]);
            u[2 * h] = u[2 * h] * (r * Two(w0.x, w0.y));
            u[2 * h + 1] = u[2 * h + 1] * (r * Two(w0.z, w0.w));
            v[2 * h] = v[2 * h] * (r * Two(w1.x, w1.y));
            v[2 * h + 1] = v[2 * h + 1] * (r * Two(w1.z, w1.w));
          }
        }
      }
      if (dst[b] != nullptr) {
        if (turns) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {      // pairs 8 lane + 4 h .. + 3
            const float4 c = *reinterpret_cast<const float4*>(&s_cos[of[b]][4 * (lane + 16 * h)]), s = *reinterpret_cast<const float4*>(&s_sin[of[b]][4 * (lane + 16 * h)]);
            if (INTERLEAVED) {
              auto turn = [](Two x, float cs, float sn) {
                const float2 f = x.both();
                return fma2(Two(f.x), Two(cs, sn), Two(f.y) * Two(-sn, cs));
              };
              Two* const x = h ? v : u;
              x[0] = turn(x[0], c.x, s.x);
              x[1] = turn(x[1], c.y, s.y);
              x[2] = turn(x[2], c.z, s.z);
              x[3] = turn(x[3], c.w, s.w);
            } else {
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const Two cs = i ? Two(c.z, c.w) : Two(c.x, c.y), sn = i ? Two(s.z, s.w) : Two(s.x, s.y), neg = i ? Two(-s.z, -s.w) : Two(-s.x, -s.y);
                const Two x0 = u[2 * h + i], x1 = v[2 * h + i];
                u[2 * h + i] = fma2(x0, cs, x1 * neg);
                v[2 * h + i] = fma2(x0, sn, x1 * cs);
              }
            }
          }
        }
        *reinterpret_cast<uint4*>(dst[b] + c0) = pack8<T>(u);
        *reinterpret_cast<uint4*>(dst[b] + c1) = pack8<T>(v);
      }
    }
  }
}

template <typename T, int LANES>
int launch(const RopeArgs& a, bool interleaved, cudaStream_t stream) {
  const unsigned grid = (unsigned)ceil_div(a.tokens, a.block_tokens);
  return interleaved ? launch_pdl(rope_kernel<T, LANES, true>, dim3(grid), dim3(kThreads), 0, stream, a)
                     : launch_pdl(rope_kernel<T, LANES, false>, dim3(grid), dim3(kThreads), 0, stream, a);
}

template <typename T>
int launch_lanes(const RopeArgs& a, bool interleaved, cudaStream_t stream) {
  if (a.dim <= 64) return launch<T, 4>(a, interleaved, stream);
  if (a.dim <= 128) return launch<T, 8>(a, interleaved, stream);
  return launch<T, 16>(a, interleaved, stream);
}

}  // namespace
}  // namespace xqt_b200

extern "C" int xqt_b200_qk_norm_rope(const void* q, const void* k, void* q_out, void* k_out, const void* q_weight, const void* k_weight,
                                     const void* positions, const double* frequencies, const int* axes, const long long* strides, int tokens,
                                     int q_heads, int k_heads, int dim, int rotary, int axis_count, int wide_positions, int interleaved, int dtype,
                                     int weight_dtype, float eps, cudaStream_t stream) {
  using namespace xqt_b200;
  XQT_REQUIRE(tokens >= 0 && q_heads >= 1 && k_heads >= 0 && q_heads <= (1 << 20) && k_heads <= (1 << 20));
  XQT_REQUIRE(dim >= 16 && dim <= 256 && dim % 16 == 0 && rotary >= 0 && rotary <= dim && rotary % 16 == 0 && axis_count >= 1);
  XQT_REQUIRE(dtype == XQT_B200_FP16 || dtype == XQT_B200_BF16);
  XQT_REQUIRE(weight_dtype == XQT_B200_FP16 || weight_dtype == XQT_B200_BF16 || weight_dtype == XQT_B200_FP32);
  if (tokens == 0) return 0;
  XQT_REQUIRE(q && q_out && strides && (k_heads == 0 || (k && k_out)));
  XQT_REQUIRE(rotary == 0 || (positions && frequencies));
  RopeArgs a = {};
  const void* in[2] = {q, k};
  void* out[2] = {q_out, k_out};
  const void* weight[2] = {q_weight, k_weight};
  const int heads[2] = {q_heads, k_heads};
  for (int i = 0; i < (k_heads ? 2 : 1); ++i) {
    a.x[i] = in[i];
    a.out[i] = out[i];
    a.weight[i] = weight[i];
    a.heads[i] = heads[i];
    a.x_token[i] = strides[4 * i];
    a.x_head[i] = strides[4 * i + 1];
    a.o_token[i] = strides[4 * i + 2];
    a.o_head[i] = strides[4 * i + 3];
    XQT_REQUIRE((((uintptr_t)in[i] | (uintptr_t)out[i]) & 15) == 0);
    XQT_REQUIRE(((a.x_token[i] | a.x_head[i] | a.o_token[i] | a.o_head[i]) & 7) == 0);
  }
  a.positions = positions;
  a.p_axis = strides[8];
  a.p_token = strides[9];
  a.frequencies = frequencies;
  a.axes = axes;
  a.axis_count = axis_count;
  a.wide_positions = wide_positions;
  a.weight_dtype = weight_dtype;
  a.tokens = tokens;
  a.dim = dim;
  a.rotary = rotary;
  a.eps = eps;
  // Tokens of a block: their cosines are made together, so more of them fill its threads; as many as make whole waves of blocks (tokens
  // of 32 + 8 heads, this | powers of two for two blocks an SM: 4096 16.8 | 17.9 us, 6000 24.7 | 28.4, 8191 31.2 | 33.4, 12,000 46.7 | 55).
  const long long wave = (long long)kPerSm * sm_count(), waves = (tokens + wave * kMostTokens - 1) / (wave * kMostTokens);
  a.block_tokens = (int)((tokens + wave * waves - 1) / (wave * waves));
  return dtype == XQT_B200_BF16 ? launch_lanes<__nv_bfloat16>(a, interleaved != 0, stream) : launch_lanes<__half>(a, interleaved != 0, stream);
}
