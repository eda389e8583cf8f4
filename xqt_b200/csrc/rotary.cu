// RMS norm of query and key heads and the position rotation, in one pass.
//
//   y = x * rsqrt(mean(x^2) + eps) * w          (no weight: y = x)
//   pair j of the first `rotary` channels -- (j, j + rotary/2), or (2j, 2j+1) where they are interleaved -- turns by
//   position[axis_j, token] * frequency_j; the other channels pass.  fp32 arithmetic, one rounding.
//
// The angle is kept as a 64-bit fixed-point fraction of a turn: position * fraction wraps exactly modulo one turn, so a far
// position loses nothing (fp32 angles are off by 2^-24 of the angle itself: 0.006 rad at position 100,000).
//
// Bound by HBM: every channel is read and written once.  A lane group of `dim / 16` (padded to a power of two) lanes holds one
// head, 16 channels a lane, chosen so that both channels of a pair are in one lane; it computes the cosines of its 8 pairs
// once and goes through `heads_per_group` heads of its token.
#include "common.cuh"

namespace xqt_b200 {

namespace {

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
  int tokens, dim, rotary, heads_per_group, chunks;
  float eps;
};

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& v, float* f) {
  const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = to_float<T>(e[i]);
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float* f) {
  uint4 v;
  T* e = reinterpret_cast<T*>(&v);
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = from_float<T>(f[i]);
  return v;
}

// LANES: lanes of a head, a power of two; lanes past dim / 16 only take part in the sums.
template <typename T, int LANES, bool INTERLEAVED>
__global__ void __launch_bounds__(256) rope_kernel(const RopeArgs a) {
  const long long group = ((long long)blockIdx.x * 256 + threadIdx.x) / LANES;
  const int lane = threadIdx.x % LANES;
  const bool in_grid = group < (long long)a.tokens * a.chunks;
  const int token = in_grid ? (int)(group / a.chunks) : 0;
  const int head0 = in_grid ? (int)(group % a.chunks) * a.heads_per_group : 0;
  const int all_heads = a.heads[0] + a.heads[1];
  const bool active = in_grid && lane < a.dim / 16;
  const bool turns = active && lane < a.rotary / 16;
  // the lane's two runs of 8 channels
  int c0, c1;
  if (INTERLEAVED || a.rotary == 0) {
    c0 = 16 * lane;
    c1 = c0 + 8;
  } else if (lane < a.rotary / 16) {
    c0 = 8 * lane;
    c1 = c0 + a.rotary / 2;
  } else {
    c0 = a.rotary + 8 * (lane - a.rotary / 16);
    c1 = c0 + (a.dim - a.rotary) / 2;
  }
  float cosine[8], sine[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    cosine[i] = 1.0f;
    sine[i] = 0.0f;
    if (turns) {
      const int pair = 8 * lane + i;
      int axis = a.axes ? a.axes[pair] : 0;
      axis = axis < 0 ? 0 : (axis >= a.axis_count ? a.axis_count - 1 : axis);
      const long long at = axis * a.p_axis + token * a.p_token;
      const long long position = a.wide_positions ? reinterpret_cast<const long long*>(a.positions)[at] : (long long)reinterpret_cast<const int*>(a.positions)[at];
      double turn = a.frequencies[pair] * 0.15915494309189533577;   // 1 / (2 pi)
      turn -= floor(turn);
      const unsigned long long fraction = __double2ull_rn(turn * 18446744073709551616.0);
      const unsigned long long angle = fraction * (unsigned long long)position;
      sincospif((float)(int)(angle >> 32) * 4.656612873077393e-10f, &sine[i], &cosine[i]);   // 2^-31: half turns
    }
  }
  const float inv_dim = 1.0f / (float)a.dim;
  constexpr int kBatch = 2;      // heads loaded before the first is worked on
  for (int first = 0; first < a.heads_per_group; first += kBatch) {
    uint4 raw[kBatch][2];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int head = head0 + first + b;
      raw[b][0] = raw[b][1] = make_uint4(0, 0, 0, 0);
      if (active && first + b < a.heads_per_group && head < all_heads) {
        const int which = head < a.heads[0] ? 0 : 1;
        const T* src = which ? reinterpret_cast<const T*>(a.x[1]) + token * a.x_token[1] + (head - a.heads[0]) * a.x_head[1]
                             : reinterpret_cast<const T*>(a.x[0]) + token * a.x_token[0] + head * a.x_head[0];
        raw[b][0] = *reinterpret_cast<const uint4*>(src + c0);
        raw[b][1] = *reinterpret_cast<const uint4*>(src + c1);
      }
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int head = head0 + first + b;
      const bool mine = first + b < a.heads_per_group && head < all_heads;
      const int which = head < a.heads[0] ? 0 : 1;
      float u[8], v[8];
      unpack8<T>(raw[b][0], u);
      unpack8<T>(raw[b][1], v);
      const void* weight = which ? a.weight[1] : a.weight[0];
      if (a.weight[0] != nullptr || a.weight[1] != nullptr) {   // uniform: every lane of the warp takes part in the sums
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = fmaf(u[i], u[i], fmaf(v[i], v[i], sum));
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (active && mine && weight != nullptr) {
          const float r = rsqrtf(sum * inv_dim + a.eps);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            u[i] = u[i] * r * load_param(weight, a.weight_dtype, c0 + i);
            v[i] = v[i] * r * load_param(weight, a.weight_dtype, c1 + i);
          }
        }
      }
      if (active && mine) {
        if (turns) {
          if (INTERLEAVED) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float x0 = u[2 * i], x1 = u[2 * i + 1], z0 = v[2 * i], z1 = v[2 * i + 1];
              u[2 * i] = fmaf(x0, cosine[i], -(x1 * sine[i]));
              u[2 * i + 1] = fmaf(x0, sine[i], x1 * cosine[i]);
              v[2 * i] = fmaf(z0, cosine[4 + i], -(z1 * sine[4 + i]));
              v[2 * i + 1] = fmaf(z0, sine[4 + i], z1 * cosine[4 + i]);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float x0 = u[i], x1 = v[i];
              u[i] = fmaf(x0, cosine[i], -(x1 * sine[i]));
              v[i] = fmaf(x0, sine[i], x1 * cosine[i]);
            }
          }
        }
        T* dst = which ? reinterpret_cast<T*>(a.out[1]) + token * a.o_token[1] + (head - a.heads[0]) * a.o_head[1]
                       : reinterpret_cast<T*>(a.out[0]) + token * a.o_token[0] + head * a.o_head[0];
        *reinterpret_cast<uint4*>(dst + c0) = pack8<T>(u);
        *reinterpret_cast<uint4*>(dst + c1) = pack8<T>(v);
      }
    }
  }
}

template <typename T, int LANES>
int launch(const RopeArgs& a, bool interleaved, cudaStream_t stream) {
  const long long threads = (long long)a.tokens * a.chunks * LANES;
  const unsigned grid = (unsigned)((threads + 255) / 256);
  if (interleaved)
    rope_kernel<T, LANES, true><<<grid, 256, 0, stream>>>(a);
  else
    rope_kernel<T, LANES, false><<<grid, 256, 0, stream>>>(a);
  return launch_status();
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
  // Heads per lane group: more heads share the cosines, fewer fill the SMs when there are few tokens.  Halved until the
  // groups fill about two blocks of every SM.
  const int all = q_heads + k_heads, lanes = dim <= 64 ? 4 : dim <= 128 ? 8 : 16;
  int per = 8;
  while (per > 1 && (long long)tokens * ceil_div(all, per) * lanes < 2LL * 256 * sm_count()) per >>= 1;
  a.heads_per_group = per;
  a.chunks = ceil_div(all, per);
  XQT_REQUIRE((long long)tokens * a.chunks * lanes / 256 < (1LL << 31) - 1);
  return dtype == XQT_B200_BF16 ? launch_lanes<__nv_bfloat16>(a, interleaved != 0, stream) : launch_lanes<__half>(a, interleaved != 0, stream);
}
