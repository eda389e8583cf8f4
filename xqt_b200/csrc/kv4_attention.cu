// Attention of few queries over a paged cache of keys and values in 4 bits (layout: kv4_cache.cu).
//
//   out = softmax(scale * q K^T + mask) V,   K, V = code * s + m  per (token, head)
//
// The queries of a sequence are its last tokens; query i sees the keys up to its own position, with a window only the last
// `window` of them.  A row that sees nothing is 0.
//
// Neither K nor V is ever formed.  The matrix instructions (mma.sync m16n8k16, fp16 operands, fp32 sums) run on the codes themselves: a
// nibble in the low bits of a half is the subnormal c * 2^-24, so one AND per two codes makes an operand, and
//   q . K_t = s_t * sum(c q) + m_t * sum(q)          P V = sum((p_t s_t) c) + sum(p_t m_t)
// puts scales and minima on the scores and on the probabilities.  Queries are scaled by a power of two per row so that fp16 holds
// them exactly down to 2^-26 of the row's largest (2^-22 in the odd channels, whose operand is 16 times smaller; the sum that goes with m is taken
// before that); p_t s_t is rounded to fp16 against a running power of two above the scales, with
// 2^15 of headroom, so nothing underflows; softmax statistics and all sums are fp32.
//
// The keys are the 16-row operand and the queries the 8-column one (transposed products), so that eight rows -- the query heads of
// one key head -- fill a tile.  Work is cut into units of W chunks of CT keys (a chunk per warp); the units of all (sequence, row tile,
// head) items form one list, of which each CTA takes an equal contiguous share whatever the lengths are; items that
// CTAs share are joined by a second kernel, or (few items of few keys) by a cluster of CTAs per item in its distributed shared memory.
// Each warp fetches its own chunks with bulk copies, S of them ahead.
//
// Its floor is HBM, (dim + 8) bytes per key and head, but it runs at half of that: the loads alone take 52 of 70 us (two documents of 131,071 keys,
// 64 query heads on 8 of 128 channels: 4.1 TB/s), the arithmetic alone 57 (5 instructions per code word for the operands, ex2 and the sums of
// a softmax in 8 columns), and two CTAs of four warps, all that the registers allow, do not hide one behind the other completely.
// 64 sequences of up to 8192 keys, 8 heads: 82 us (3.6 TB/s); one of 777 keys: 7 us, launch and one chain of loads and products.
#include "kv4_attention.cuh"

namespace xqt_b200 {

namespace {

using namespace kv4;

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_16816_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void prefetch_l1(const void* p) { asm volatile("prefetch.global.L1 [%0];\n" ::"l"(p)); }
template <int D_, int NT_, int W_, int CT_, int S_, int PER_SM_>
struct Shape {
  static constexpr int D = D_, NT = NT_, W = W_, CT = CT_, S = S_, PER_SM = PER_SM_;
  static constexpr int ROWS = 8 * NT, KROW = D / 2, KWORDS = D / 32, VWORDS = D / 64, MT = CT / 16;
  static constexpr int UNIT = W * CT;
  static constexpr int OPENING = 1;                      // a unit for an item's beginning and end: its queries read, its warps joined
  static constexpr bool PROMPT = false;
  static constexpr int CODE_BYTES = CT * KROW, PARAM_BYTES = CT * 4, STAGE = 2 * (CODE_BYTES + PARAM_BYTES);
  static constexpr int MERGE_ROW = D + 8;
  static constexpr int MERGES = W / 2;                    // buffers: the warps add to them in rounds
  static constexpr int MERGE_BYTES = MERGES * ROWS * MERGE_ROW * 4, STAT_BYTES = (2 * W + 1) * ROWS * 16;      // the warps' statistics twice: an item's are written while the last one's are read
  static constexpr int SMEM = W * S * STAGE + MERGE_BYTES + STAT_BYTES + W * S * 8;
};

template <typename L>
__device__ __forceinline__ void advance(const AttnArgs& a, Walk& w) {
  if (++w.unit < w.s.units) return;
  w.unit = 0;
  if (++w.head < a.kv_heads) return;
  w.head = 0;
  if (++w.tile < w.s.tiles) return;
  w.tile = 0;
  while (++w.b < a.batch) {
    w.s = sequence<L>(a, w.b);
    if (w.s.tiles > 0) return;
  }
}

__device__ __forceinline__ float2 ld_cluster_f2(uint32_t caddr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];\n" : "=f"(v.x), "=f"(v.y) : "r"(caddr) : "memory");
  return v;
}

// CLUSTER: a cluster of CTAs takes one item, each an equal run of its units, and joins it through distributed shared memory.
template <typename T, typename SH, bool CLUSTER>
__global__ void __launch_bounds__(SH::W * 32, SH::PER_SM) kv4_attention_kernel(const AttnArgs a) {
  constexpr int D = SH::D, NT = SH::NT, W = SH::W, CT = SH::CT, S = SH::S, ROWS = SH::ROWS, MT = SH::MT, KROW = SH::KROW;
  constexpr int KWORDS = SH::KWORDS, VWORDS = SH::VWORDS;
  extern __shared__ __align__(128) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  uint8_t* const ring = smem + warp * (S * SH::STAGE);
  float* const merge = reinterpret_cast<float*>(smem + W * S * SH::STAGE);
  float4* stats = reinterpret_cast<float4*>(smem + W * S * SH::STAGE + SH::MERGE_BYTES);
  float4* const stats0 = stats;
  float4* const cta_ml = stats + 2 * W * ROWS;             // CLUSTER: of the CTA's part
  const uint32_t bars = smem_addr(smem + W * S * SH::STAGE + SH::MERGE_BYTES + SH::STAT_BYTES) + warp * (S * 8);
  if (lane == 0) {
    for (int s = 0; s < S; ++s) mbar_init(bars + 8 * s, 1);
    fence_barrier_init();
  }
  __syncwarp();
  grid_launch_dependents();
  grid_dependency_wait();

  Walk c;
  unsigned u0 = 0, u1;
  if constexpr (CLUSTER) {
    const unsigned rank = cluster_ctarank(), size = cluster_nctarank();
    if (!place_item<SH>(a, lane, blockIdx.x / size, c)) return;        // (all of the cluster)
    const unsigned units = (unsigned)(c.s.units - SH::OPENING), lo = units * rank / size;
    c.unit = SH::OPENING + (int)lo;
    u1 = units * (rank + 1) / size - lo;
  } else {
    Sequence mine = {};
    const Deal d = deal<SH>(a, lane, gridDim.x, mine);
    u0 = d.start(blockIdx.x);
    u1 = d.start(blockIdx.x + 1);
    const bool some = u0 < u1 && place<SH>(a, lane, mine, u0, c);
    if (tid == 0) {                                  // for the second kernel: where this CTA begins
      a.plan[blockIdx.x] = make_int4((int)d.total, some ? c.unit : 0, some ? c.s.units : 0, some ? c.head : 0);
      a.plan[gridDim.x + blockIdx.x] = some ? make_int4(c.b, c.tile, c.s.q0, c.s.nq) : make_int4(0, 0, 0, 0);
    }
    if (!some) return;
  }

  // ---- fetching
  const int psz = min(a.page_size, CT), pieces = CT / psz;
  const int piece = lane >> 2, kind = lane & 3;                      // kind: key codes, value codes, key parameters, value parameters
  const int row_bytes = kind < 2 ? KROW : 4;
  const uint8_t* const source = (kind < 2 ? a.codes : a.params) + (kind & 1) * ((long long)a.kv_heads * a.page_size * row_bytes);
  const long long page_bytes = 2LL * a.kv_heads * a.page_size * row_bytes;
  const uint32_t target = smem_addr(ring) + (kind == 0 ? 0 : kind == 1 ? SH::CODE_BYTES : kind == 2 ? 2 * SH::CODE_BYTES : 2 * SH::CODE_BYTES + SH::PARAM_BYTES) +
                          piece * psz * row_bytes;
  Walk f = c;
  // of the item being fetched: its units not yet asked for, this lane's next key, the keys that some row of the tile sees, the table's row
  int f_units = 0, f_at = 0, f_end = 0, f_begin = 0;
  const int* f_table = nullptr;
  auto open = [&]() {
    const int j0 = f.tile * ROWS / a.each, j1 = min(f.s.nq - 1, (f.tile * ROWS + ROWS - 1) / a.each);
    f_units = f.s.units - f.unit;
    f_at = piece < pieces ? f.s.first + ((f.unit - SH::OPENING) * W + warp) * CT + piece * psz : INT_MAX - (1 << 24);
    f_end = f.b < a.batch ? f.s.len - f.s.nq + j1 + 1 : 0;      // (starts that do not ascend can make the list shorter than it counts)
    f_begin = a.window ? (int)max((long long)f.s.len - f.s.nq + j0 - a.window + 1, 0LL) : 0;
    f_table = a.table + f.b * a.table_stride;
    // its queries, which the warps read when they come to it
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = f.tile * ROWS + nt * 8 + g, j = r / a.each;
      if (j < f.s.nq)
        prefetch_l1(reinterpret_cast<const T*>(a.q) + (long long)(f.s.q0 + j) * a.q_token + (long long)(f.head * a.each + r - j * a.each) * a.q_head + t * (D / 4));
    }
  };
  open();
  int to_fetch = (int)(u1 - u0);
  int next_page = -1, next_row = 0;
  uint32_t masks = 0, phases = 0;
  bool dead = false;
  // the table entry of the next chunk to fetch, asked for one chunk ahead of its use
  auto look_up = [&]() {
    next_page = -1;
    if (to_fetch > 0) {
      if (f_at < f_end && f_at + psz > f_begin) next_page = f_table[f_at >> a.page_shift];
      next_row = f.head * a.page_size + (f_at & (a.page_size - 1));
      --to_fetch;
      if (--f_units > 0) {
        if (piece < pieces) f_at += SH::UNIT;
      } else if (to_fetch > 0) {
        f.unit = f.s.units - 1;
        advance<SH>(a, f);
        open();
      }
    }
  };
  auto issue = [&](int stage) {
    const bool valid = (unsigned)next_page < (unsigned)a.pages && !dead;
    const unsigned votes = __ballot_sync(0xffffffffu, valid);
    unsigned mask = votes & 1u;
    if constexpr (MT > 1) mask |= votes >> 3 & 2u;
    if constexpr (MT > 2) mask |= (votes >> 6 & 4u) | (votes >> 9 & 8u);
    masks = (masks & ~(15u << (4 * stage))) | mask << (4 * stage);
    if (mask) {
      const uint32_t bar = bars + 8 * stage;
      if (lane == 0) mbar_expect_tx(bar, (uint32_t)(__popc(mask) * psz * 2 * (KROW + 4)));
      __syncwarp();
      if (valid) bulk_g2s(target + stage * SH::STAGE, source + next_page * page_bytes + (long long)next_row * row_bytes, (uint32_t)(psz * row_bytes), bar);
    }
  };
#pragma unroll 1
  for (int s = 0; s < S; ++s) {
    look_up();
    issue(s);
  }
  look_up();

  // ---- one item's state
  uint32_t qf[NT][2 * KWORDS][2];
  Two qa[NT], qb[NT];
  int hi[NT][2], lo[NT][2];
  Two o[VWORDS * 4][NT][2];
  float mx[NT][2], sigma = 0.0f, inv_sigma = 0.0f;
  Two l[NT], lm[NT], lw[NT];       // sums of p and of p * m, and what the rounding of the operands p * s took away
  int full_hi = 0, full_lo = 0;
  const unsigned all_pieces = (1u << pieces) - 1;
  constexpr bool KEEP_ROUNDING = sizeof(T) == 2 && !std::is_same<T, __nv_bfloat16>::value;

  auto start_item = [&]() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      // as the operand wants it: row g of this 8-column tile, the channels that go with this lane's key words
      const int r = c.tile * ROWS + nt * 8 + g;
      const int j = r / a.each;
      const bool real = j < c.s.nq;
      const T* src = reinterpret_cast<const T*>(a.q) + (long long)(c.s.q0 + (real ? j : 0)) * a.q_token + (long long)(c.head * a.each + r - j * a.each) * a.q_head;
      uint4 raw[KWORDS];
      float top = 0.0f;
#pragma unroll
      for (int w = 0; w < KWORDS; ++w) {
        const int ch = D <= 128 ? t * (D / 4) + 8 * w : 128 * (w >> 2) + 32 * t + 8 * (w & 3);
        raw[w] = real ? *reinterpret_cast<const uint4*>(src + ch) : make_uint4(0, 0, 0, 0);
        const T* e = reinterpret_cast<const T*>(&raw[w]);
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(to_float<T>(e[i])));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // the power of two that brings the largest to [2^12, 2^13)
      const int e = top > 0.0f && top <= 3.402823466e38f ? min(max((int)(__float_as_uint(top) >> 23) - 127 - 12, -110), 110) : 0;
      const float down = __uint_as_float((uint32_t)(127 - e) << 23), up = __uint_as_float((uint32_t)(127 + e) << 23);
      float sum = 0.0f;
#pragma unroll
      for (int w = 0; w < KWORDS; ++w) {
        const T* x = reinterpret_cast<const T*>(&raw[w]);
        __half h[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          h[i] = __float2half_rn(to_float<T>(x[i]) * down);
          sum += __half2float(h[i]);
        }
        // nibbles 0,4 | 1,5 | 2,6 | 3,7 of a word; the odd ones stand 16 times too high in their operand
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float by = i & 1 ? 0.0625f : 1.0f;
          qf[nt][2 * w + (i >> 1)][i & 1] = pack_half2(__half2float(h[i]) * by, __half2float(h[i + 4]) * by);
        }
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      const float per = up * a.scale;
      float qs[2], qt[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int owner = (2 * t + i) * 4;
        qs[i] = __shfl_sync(0xffffffffu, per, owner);
        qt[i] = __shfl_sync(0xffffffffu, sum, owner) * qs[i];
        qs[i] *= 16777216.0f;
        const int row = c.tile * ROWS + nt * 8 + 2 * t + i, jj = row / a.each;
        hi[nt][i] = jj < c.s.nq ? c.s.len - c.s.nq + jj : -1;
        lo[nt][i] = a.window ? (int)max((long long)c.s.len - c.s.nq + jj - a.window + 1, 0LL) : 0;
        mx[nt][i] = -CUDART_INF_F;
      }
      qa[nt] = Two(qs[0], qs[1]);
      qb[nt] = Two(qt[0], qt[1]);
      l[nt] = lm[nt] = lw[nt] = Two(0.0f);
    }
#pragma unroll
    for (int i = 0; i < VWORDS * 4; ++i)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) o[i][nt][e] = Two(0.0f);
    sigma = inv_sigma = 0.0f;
    // keys that every row of the tile sees
    const int j0 = c.tile * ROWS / a.each, j1 = (c.tile * ROWS + ROWS - 1) / a.each;
    full_hi = c.s.len - c.s.nq + j0;
    full_lo = a.window ? (int)max((long long)c.s.len - c.s.nq + min(j1, c.s.nq - 1) - a.window + 1, 0LL) : 0;
  };

  // full: every row sees every key of the chunk
  auto chunk = [&](const uint8_t* st, int tok0, unsigned mask, bool full) {
    const uint8_t* const kp = st + 2 * SH::CODE_BYTES;
    const uint8_t* const vp = kp + SH::PARAM_BYTES;
    const int pg = g ^ (g >> 1 & 1);                 // the key of operand row g: neighbours alternate, which spreads the value rows over the banks
    float p[MT][NT][4];
    uint32_t vb[MT][2];                              // scale and minimum of the values
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int r0 = mt * 16 + pg;
      uint32_t k0[KWORDS], k1[KWORDS];
      if constexpr (D == 64) {
        const uint2 x = *reinterpret_cast<const uint2*>(st + r0 * KROW + 8 * t), y = *reinterpret_cast<const uint2*>(st + (r0 + 8) * KROW + 8 * t);
        k0[0] = x.x; k0[1] = x.y; k1[0] = y.x; k1[1] = y.y;
      } else {
#pragma unroll
        for (int h = 0; h < KWORDS / 4; ++h) {
          const uint4 x = *reinterpret_cast<const uint4*>(st + r0 * KROW + 64 * h + 16 * t), y = *reinterpret_cast<const uint4*>(st + (r0 + 8) * KROW + 64 * h + 16 * t);
          k0[4 * h] = x.x; k0[4 * h + 1] = x.y; k0[4 * h + 2] = x.z; k0[4 * h + 3] = x.w;
          k1[4 * h] = y.x; k1[4 * h + 1] = y.y; k1[4 * h + 2] = y.z; k1[4 * h + 3] = y.w;
        }
      }
      float acc[NT][4];
#pragma unroll
      for (int w = 0; w < KWORDS; ++w) {
        const uint32_t x = k0[w], y = k1[w], x8 = x >> 8, y8 = y >> 8;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if (w == 0)
            mma_16816_first(acc[nt], x & 0x000f000fu, y & 0x000f000fu, x & 0x00f000f0u, y & 0x00f000f0u, qf[nt][0][0], qf[nt][0][1]);
          else
            mma_16816(acc[nt], x & 0x000f000fu, y & 0x000f000fu, x & 0x00f000f0u, y & 0x00f000f0u, qf[nt][2 * w][0], qf[nt][2 * w][1]);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          mma_16816(acc[nt], x8 & 0x000f000fu, y8 & 0x000f000fu, x8 & 0x00f000f0u, y8 & 0x00f000f0u, qf[nt][2 * w + 1][0], qf[nt][2 * w + 1][1]);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float2 s = pair_of<T>(*reinterpret_cast<const uint32_t*>(kp + (r0 + 8 * e) * 4));
        vb[mt][e] = *reinterpret_cast<const uint32_t*>(vp + (r0 + 8 * e) * 4);
        const Two s2(s.x), m2(s.y);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float2 x = fma2(Two(acc[nt][2 * e], acc[nt][2 * e + 1]), s2 * qa[nt], m2 * qb[nt]).both();
          p[mt][nt][2 * e] = x.x;
          p[mt][nt][2 * e + 1] = x.y;
        }
      }
    }
    if (!full) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int at = mt * 16 + pg + 8 * e, tok = tok0 + at;
          const bool there = mask >> (at / psz) & 1u;
          if (!there || tok >= c.s.len) vb[mt][e] = 0;       // nothing was fetched, or nothing was ever written
          // a value that is not finite spoils the rows that see it by their scores, and counts as 0 for the others
          const float2 v = pair_of<T>(vb[mt][e]);
          const bool bad = !(fabsf(v.x) <= 3.402823466e38f && fabsf(v.y) <= 3.402823466e38f);
          if (bad) vb[mt][e] = 0;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              if (bad) p[mt][nt][2 * e + i] = CUDART_NAN_F;
              if (!there || tok > hi[nt][i] || tok < lo[nt][i]) p[mt][nt][2 * e + i] = -CUDART_INF_F;
            }
        }
    }
    // running maxima; nothing is exchanged while no lane exceeds them
    float top[NT][2], big = 0.0f;
    bool grows = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        top[nt][i] = fmaxf(p[0][nt][i], p[0][nt][i + 2]);
#pragma unroll
        for (int mt = 1; mt < MT; ++mt) top[nt][i] = fmaxf(top[nt][i], fmaxf(p[mt][nt][i], p[mt][nt][i + 2]));
        grows = grows || top[nt][i] > mx[nt][i];
      }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) big = fmaxf(big, fmaxf(fabsf(pair_of<T>(vb[mt][0]).x), fabsf(pair_of<T>(vb[mt][1]).x)));
    grows = grows || big > sigma;
    if (__any_sync(0xffffffffu, grows)) {
      big = 0.0f;                                    // without infinities, which spoil only the rows that see them
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (fabsf(pair_of<T>(vb[mt][e]).x) <= 3.402823466e38f) big = fmaxf(big, fabsf(pair_of<T>(vb[mt][e]).x));
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) {
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, x));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 2; ++i) top[nt][i] = fmaxf(top[nt][i], __shfl_xor_sync(0xffffffffu, top[nt][i], x));
      }
      float by = 1.0f;
      if (big > sigma) {
        // a power of two above every scale so far, in [2^-100, 2^127]
        const int e = min(max((int)(__float_as_uint(big) >> 23) + 1, 27), 254);
        const float next = __uint_as_float((uint32_t)e << 23);
        by = sigma == 0.0f ? 0.0f : sigma * (1.0f / next);
        sigma = next;
        inv_sigma = 32768.0f / next;
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float alpha[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float m = fmaxf(mx[nt][i], top[nt][i]);
          alpha[i] = mx[nt][i] == m ? 1.0f : exp2_fast(mx[nt][i] - m);
          mx[nt][i] = m;
        }
        const Two al(alpha[0], alpha[1]), both = al * Two(by);
        l[nt] = l[nt] * al;
        lm[nt] = lm[nt] * al;
        lw[nt] = lw[nt] * both;
#pragma unroll
        for (int i = 0; i < VWORDS * 4; ++i) {
          o[i][nt][0] = o[i][nt][0] * both;
          o[i][nt][1] = o[i][nt][1] * both;
        }
      }
    }
    // probabilities, their sums, and the second operand of P V
    uint32_t pf[MT][NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      Two of_chunk(0.0f), of_minima(0.0f);           // (keys one by one would be lost beside a strong one in a sum of a million; same time)
      const Two minus(mx[nt][0] == -CUDART_INF_F ? 0.0f : -mx[nt][0], mx[nt][1] == -CUDART_INF_F ? 0.0f : -mx[nt][1]);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float2 x = (Two(p[mt][nt][2 * e], p[mt][nt][2 * e + 1]) + minus).both();
          const Two pr(exp2_fast(x.x), exp2_fast(x.y));
          of_chunk = of_chunk + pr;
          const float2 sv = pair_of<T>(vb[mt][e]);
          const Two w2 = pr * Two(sv.x * inv_sigma);
          of_minima = fma2(pr, Two(sv.y), of_minima);
          const float2 w = w2.both();
          const uint32_t h = pack_half2(w.x, w.y);
          if constexpr (KEEP_ROUNDING) {
            const float2 r = __half22float2(*reinterpret_cast<const __half2*>(&h));
            lw[nt] = lw[nt] + (w2 + Two(-r.x, -r.y));
          }
          pf[mt][nt][e] = transpose8x8(h);
        }
      l[nt] = l[nt] + of_chunk;
      lm[nt] = lm[nt] + of_minima;
    }
    const uint8_t* const vs = st + SH::CODE_BYTES + g * (4 * VWORDS);
    const int x0 = 2 * t ^ (t & 1), y0 = x0 ^ 1;
#pragma unroll
    for (int j = 0; j < VWORDS; ++j) {
      float part[4][NT][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const uint8_t* const at = vs + mt * 16 * KROW + 4 * j;
        const uint32_t x = *reinterpret_cast<const uint32_t*>(at + x0 * KROW), y = *reinterpret_cast<const uint32_t*>(at + y0 * KROW);
        const uint32_t z = *reinterpret_cast<const uint32_t*>(at + (x0 + 8) * KROW), w = *reinterpret_cast<const uint32_t*>(at + (y0 + 8) * KROW);
        const uint32_t a01 = __byte_perm(x, y, 0x5410), a23 = __byte_perm(x, y, 0x7632), b01 = __byte_perm(z, w, 0x5410), b23 = __byte_perm(z, w, 0x7632);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t u = (i < 2 ? a01 : a23) >> (8 * (i & 1)), v = (i < 2 ? b01 : b23) >> (8 * (i & 1));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            if (mt == 0)
              mma_16816_first(part[i][nt], u & 0x000f000fu, u & 0x00f000f0u, v & 0x000f000fu, v & 0x00f000f0u, pf[mt][nt][0], pf[mt][nt][1]);
            else
              mma_16816(part[i][nt], u & 0x000f000fu, u & 0x00f000f0u, v & 0x000f000fu, v & 0x00f000f0u, pf[mt][nt][0], pf[mt][nt][1]);
          }
        }
      }
      // added here, rounded to nearest: the matrix unit cuts off what it adds to a running sum
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) o[4 * j + i][nt][e] = o[4 * j + i][nt][e] + Two(part[i][nt][2 * e], part[i][nt][2 * e + 1]);
    }
  };

  // the warps' parts of an item joined, and written as the result or as this CTA's part of it
  auto finish_item = [&](bool whole, int slot) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float2 l2 = l[nt].both(), m2 = lm[nt].both(), w2 = lw[nt].both();
      float ls[2] = {l2.x, l2.y}, ms[2] = {m2.x, m2.y};
      if constexpr (KEEP_ROUNDING) {                 // 7.5, the middle of the codes, times what was lost
        ms[0] = fmaf(w2.x, 7.5f / 32768.0f * sigma, ms[0]);
        ms[1] = fmaf(w2.y, 7.5f / 32768.0f * sigma, ms[1]);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
          ls[i] += __shfl_xor_sync(0xffffffffu, ls[i], x);
          ms[i] += __shfl_xor_sync(0xffffffffu, ms[i], x);
        }
        if (g == 0) stats[warp * ROWS + nt * 8 + 2 * t + i] = make_float4(mx[nt][i], ls[i], ms[i], 0.0f);
      }
    }
    __syncthreads();
#pragma unroll 1
    for (int round = 0; round < W / SH::MERGES; ++round) {
      if (warp / SH::MERGES == round) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int row = nt * 8 + 2 * t + i;
            float m = -CUDART_INF_F;
#pragma unroll
            for (int w = 0; w < W; ++w) m = fmaxf(m, stats[w * ROWS + row].x);
            const float by = m == -CUDART_INF_F ? 0.0f : 512.0f * sigma * exp2_fast(mx[nt][i] - m), by16 = by * 0.0625f;
            float* const dst = merge + (warp % SH::MERGES * ROWS + row) * SH::MERGE_ROW + 2 * g;       // pair j of lane g's channels at 16 j + 2 g
            float2 old[VWORDS * 4];
#pragma unroll
            for (int j = 0; j < VWORDS * 4; ++j) old[j] = round ? *reinterpret_cast<const float2*>(dst + 16 * j) : make_float2(0.0f, 0.0f);
#pragma unroll
            for (int j = 0; j < VWORDS * 4; ++j) {
              const float2 even = o[j][nt][0].both(), odd = o[j][nt][1].both();
              *reinterpret_cast<float2*>(dst + 16 * j) = make_float2(fmaf(i ? even.y : even.x, by, old[j].x), fmaf(i ? odd.y : odd.x, by16, old[j].y));
            }
          }
      }
      __syncthreads();
    }
    constexpr int QUADS = D / 4;
#pragma unroll 2
    for (int i = tid; i < ROWS * QUADS; i += W * 32) {
      const int row = i / QUADS, quad = i % QUADS;   // channels 4 quad .. 4 quad + 3
      const int r = c.tile * ROWS + row, j = r / a.each;
      if (j >= c.s.nq) continue;
      const int at = quad % (D / 32) * 32 + quad / (D / 32) * 2;
      float m = -CUDART_INF_F, weight = 0.0f, add = 0.0f;
#pragma unroll
      for (int w = 0; w < W; ++w) m = fmaxf(m, stats[w * ROWS + row].x);
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float4 st = stats[w * ROWS + row];
        const float by = m == -CUDART_INF_F ? 0.0f : exp2_fast(st.x - m);
        weight = fmaf(st.y, by, weight);
        add = fmaf(st.z, by, add);
      }
      float4 sum = make_float4(add, add, add, add);
#pragma unroll
      for (int w = 0; w < SH::MERGES; ++w) {
        const float* const src = merge + (w * ROWS + row) * SH::MERGE_ROW + at;
        const float2 u = *reinterpret_cast<const float2*>(src), v = *reinterpret_cast<const float2*>(src + 16);
        sum.x += u.x;
        sum.y += u.y;
        sum.z += v.x;
        sum.w += v.y;
      }
      if constexpr (CLUSTER) {                       // the CTA's part, at the places that only this thread reads
        float* const to = merge + row * SH::MERGE_ROW + at;
        *reinterpret_cast<float2*>(to) = make_float2(sum.x, sum.y);
        *reinterpret_cast<float2*>(to + 16) = make_float2(sum.z, sum.w);
        if (quad == 0) cta_ml[row] = make_float4(m, weight, 0.0f, 0.0f);
      } else if (whole) {
        const float inv = weight == 0.0f ? 0.0f : 1.0f / weight;
        T* const dst = reinterpret_cast<T*>(a.out) + ((long long)(c.s.q0 + j) * a.q_heads + c.head * a.each + r - j * a.each) * D + 4 * quad;
        T v[4] = {from_float<T>(sum.x * inv), from_float<T>(sum.y * inv), from_float<T>(sum.z * inv), from_float<T>(sum.w * inv)};
        *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<uint2*>(v);
      } else {
        *reinterpret_cast<float4*>(a.part_o + ((long long)slot * ROWS + row) * D + 4 * quad) = sum;
        if (quad == 0) a.part_ml[(long long)slot * ROWS + row] = make_float2(m, weight);
      }
    }
    if constexpr (CLUSTER) {
      cluster_arrive_release();
      cluster_wait_acquire();
      const unsigned rank = cluster_ctarank(), size = cluster_nctarank();
      for (int i = tid + rank * (W * 32); i < ROWS * (D / 2); i += size * (W * 32)) {
        const int row = i / (D / 2), pair = i % (D / 2);               // channels 2 pair, 2 pair + 1: pair j of lane g's channels at 16 j + 2 g
        const int r = c.tile * ROWS + row, j = r / a.each;
        if (j >= c.s.nq) continue;
        const uint32_t value_at = smem_addr(merge + row * SH::MERGE_ROW + pair % (D / 16) * 16 + pair / (D / 16) * 2), ml_at = smem_addr(cta_ml + row);
        float m = -CUDART_INF_F, weight = 0.0f;
        for (unsigned x = 0; x < size; ++x) m = fmaxf(m, ld_cluster_f2(cluster_map(ml_at, x)).x);
        float2 sum = make_float2(0.0f, 0.0f);
        for (unsigned x = 0; x < size; ++x) {
          const float2 st = ld_cluster_f2(cluster_map(ml_at, x)), v = ld_cluster_f2(cluster_map(value_at, x));
          const float by = st.x == m ? 1.0f : exp2_fast(st.x - m);
          weight = fmaf(st.y, by, weight);
          sum.x = fmaf(v.x, by, sum.x);
          sum.y = fmaf(v.y, by, sum.y);
        }
        const float inv = weight == 0.0f ? 0.0f : 1.0f / weight;
        T v[2] = {from_float<T>(sum.x * inv), from_float<T>(sum.y * inv)};
        *reinterpret_cast<uint32_t*>(reinterpret_cast<T*>(a.out) + ((long long)(c.s.q0 + j) * a.q_heads + c.head * a.each + r - j * a.each) * D + 2 * pair) = *reinterpret_cast<const uint32_t*>(v);
      }
      cluster_arrive_relaxed();                      // nobody leaves while its shared memory is read
      cluster_wait_acquire();
    }
    stats = stats == stats0 ? stats0 + W * ROWS : stats0;
  };

  int stage = 0;
  bool opens = true;
  int from_unit = 0;
  if constexpr (CLUSTER) start_item();
#pragma unroll 1
  for (unsigned u = u0; u < u1; ++u) {
    if (!CLUSTER && opens) {
      start_item();
      from_unit = c.unit;
      opens = false;
    }
    const unsigned mask = masks >> (4 * stage) & 15u;
    if (mask) {
      if (!mbar_wait(bars + 8 * stage, phases >> stage & 1u)) {
        dead = true;
        if (lane == 0 && a.status) *a.status = 1u;
      }
      phases ^= 1u << stage;
      const int tok0 = c.s.first + ((c.unit - SH::OPENING) * W + warp) * CT;
      if (!dead) chunk(ring + stage * SH::STAGE, tok0, mask, mask == all_pieces && tok0 + CT - 1 <= full_hi && tok0 >= full_lo);
      __syncwarp();
    }
    issue(stage);
    look_up();
    stage = stage + 1 == S ? 0 : stage + 1;
    if constexpr (CLUSTER) {
      ++c.unit;
    } else {
      const bool ends = c.unit + 1 == c.s.units;
      if (ends || u + 1 == u1) {
        finish_item(ends && from_unit == 0, 2 * blockIdx.x + (from_unit == 0 ? 1 : 0));
        opens = true;
      }
      advance<SH>(a, c);
    }
  }
  if constexpr (CLUSTER) finish_item(false, 0);
}

// Joins the items that a boundary between two CTAs of the kernel above runs through: block (x, y) for boundary x + 1 and two rows, if it is the first in
// its item.
constexpr int kJoinWarps = 4, kJoinRows = 2;      // warps of a row, rows of a block
template <typename T, typename SH>
__global__ void __launch_bounds__(kJoinRows * kJoinWarps * 32) kv4_attention_join_kernel(const AttnArgs a, unsigned ctas) {
  constexpr int D = SH::D, ROWS = SH::ROWS, PER = D / 32;
  __shared__ float all_sums[kJoinRows][kJoinWarps][D];
  __shared__ float2 all_ml[kJoinRows][kJoinWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32 % kJoinWarps, half = threadIdx.x / (32 * kJoinWarps), row = blockIdx.y * kJoinRows + half;
  float(*const sums)[D] = all_sums[half];
  float2* const ml = all_ml[half];
  grid_launch_dependents();
  grid_dependency_wait();
  const int4 p = a.plan[blockIdx.x + 1], w = a.plan[ctas + blockIdx.x + 1];       // total, unit, units, head | sequence, tile, first query, queries
  if (p.y == 0) return;
  const int r = w.y * ROWS + row, j = r / a.each;
  Deal d;
  d.total = (unsigned)p.x;
  d.each = d.total / ctas;
  d.more = d.total - d.each * ctas;
  const unsigned u0 = d.start(blockIdx.x + 1) - (unsigned)p.y;                    // the item's first unit
  const int i0 = (int)d.owner(u0), i1 = (int)d.owner(u0 + (unsigned)p.z - 1);
  if (i0 != (int)blockIdx.x) return;
  float m = -CUDART_INF_F, weight = 0.0f;
  float sum[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) sum[e] = 0.0f;
  join_parts<D>(a, ROWS, row, j < w.w ? i0 + warp : i1 + 1, i1, kJoinWarps, d, u0, m, weight, sum);
#pragma unroll
  for (int e = 0; e < PER; ++e) sums[warp][lane * PER + e] = sum[e];
  if (lane == 0) ml[warp] = make_float2(m, weight);
  __syncthreads();
  if (j >= w.w) return;
  for (int at = threadIdx.x % (kJoinWarps * 32); at < D; at += kJoinWarps * 32) {
    float top = -CUDART_INF_F, all = 0.0f, value = 0.0f;
#pragma unroll
    for (int i = 0; i < kJoinWarps; ++i) top = fmaxf(top, ml[i].x);
#pragma unroll
    for (int i = 0; i < kJoinWarps; ++i) {
      const float by = ml[i].x == top ? 1.0f : exp2_fast(ml[i].x - top);
      all = fmaf(ml[i].y, by, all);
      value = fmaf(sums[i][at], by, value);
    }
    reinterpret_cast<T*>(a.out)[((long long)(w.z + j) * a.q_heads + p.w * a.each + r - j * a.each) * D + at] = from_float<T>(all == 0.0f ? 0.0f : value / all);
  }
}

constexpr int kFewRows = 32;      // rows for a key head up to which a sequence stays with this file's kernel
constexpr int kMostPerSm = 2;      // CTAs of any shape on an SM

// Two CTAs of four warps on an SM, with all the registers that leaves.  Keys per chunk: 64 for one 8-row tile of up to 128 channels (two
// documents of 131,071 keys, 64 query heads on 8: 70 us; three CTAs of 168 registers with chunks of 64 keys: 72, of 32 keys: 83; with 64 keys, two CTAs
// of two warps: 78), fewer where the sums of a chunk take more registers.
template <int D, int NT>
using Few = Shape<D, NT, 4, D == 256 ? 16 : NT == 1 ? 64 : 32, D * NT == 128 ? 3 : 4, 2>;

// Clusters of `size` CTAs (2, 4 or 8) that are resident together, asked for once per kernel and device.
template <auto Kern>
int resident_clusters(int size, int threads, size_t smem) {
  static int cached[64][3] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return sm_count() / size;
  int& known = cached[dev][size == 8 ? 2 : size == 4 ? 1 : 0];
  if (known == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(sm_count() / size * size));
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)size;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int v = 0;
    if (cudaOccupancyMaxActiveClusters(&v, Kern, &cfg) != cudaSuccess || v <= 0) v = sm_count() / size;
    known = v;
  }
  return known;
}

template <typename T, int D, int NT>
int run(AttnArgs a, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  using SH = Few<D, NT>;
  static_assert((SH::SMEM + 1024) * SH::PER_SM <= 228 * 1024 && SH::PER_SM <= kMostPerSm, "resident together");
  // as many items as there can be: full tiles, and one that is not full per sequence
  const long long most_rows = a.query_starts ? a.few_rows : a.each;
  const long long tiles = min((long long)a.tokens * a.each / SH::ROWS + a.batch, a.batch * ((most_rows + SH::ROWS - 1) / SH::ROWS));
  const long long items = tiles * a.kv_heads, units = items * (((long long)a.table_width << a.page_shift) / SH::UNIT + 1 + SH::OPENING);
  XQT_REQUIRE(items < (1LL << 31) - 1 && units < (1LL << 31));
  // Few items with few keys: a cluster for each, which needs neither the list nor the second kernel (cluster | list: one sequence of 777 keys 6.6 |
  // 9.0 us, 64 of 500 18 | 21).  Where items of many keys do not fill the SMs, or there are many items, the list's even shares win (two of 131,071
  // keys, eight heads: 125 | 70; 64 up to 8192: 95 | 82).  Keys are what the table has room for: one sequence of 777 keys behind a table of 131,072 takes
  // the list and 9.2 us.
  const long long keys = (long long)a.table_width << a.page_shift, seen = a.window ? min(keys, (long long)a.window + min(most_rows / a.each, (long long)a.tokens) + SH::CT) : keys;
  const long long of_item = (seen + SH::UNIT - 1) / SH::UNIT;
  // A cluster's size goes by the items of queries dealt out evenly and by what is resident together.  What the grid has over those items finds
  // nothing and ends, for which an eighth of the places is left (16 x 5 queries in a window of 1024: 14.9 us, by all that there can
  // be 19.4; 9 x 7 queries in a window of 694: with all places taken 15.2 us, like this
  // 9.5; nine sequences of 900 keys: sizes that fill the SMs but are not resident together 13.5, like this 9.6).
  XQT_SMEM_OPT_IN((kv4_attention_kernel<T, SH, true>), SH::SMEM);
  const long long even = min(tiles, a.batch * (((long long)a.tokens * a.each + (long long)a.batch * SH::ROWS - 1) / ((long long)a.batch * SH::ROWS))) * a.kv_heads;
  int size = 8;
  while (size > 1) {
    const long long places = resident_clusters<kv4_attention_kernel<T, SH, true>>(size, SH::W * 32, SH::SMEM);
    if (even + min(items - even, places / 8) <= places && size < 2 * of_item) break;
    size >>= 1;
  }
  if (items * size <= 4LL * SH::PER_SM * sm_count() && of_item <= 8 * size)
    return launch_pdl_cluster(kv4_attention_kernel<T, SH, true>, dim3((unsigned)(items * size)), dim3(SH::W * 32), size, SH::SMEM, stream, a);
  const int ctas = (int)min((long long)SH::PER_SM * sm_count(), units);
  const size_t o_bytes = (size_t)2 * ctas * SH::ROWS * D * 4;
  XQT_REQUIRE(workspace && workspace_bytes >= o_bytes + (size_t)2 * ctas * (SH::ROWS * 8 + 16) && ((uintptr_t)workspace & 15) == 0);
  a.part_o = reinterpret_cast<float*>(workspace);
  a.part_ml = reinterpret_cast<float2*>((uint8_t*)workspace + o_bytes);
  a.plan = reinterpret_cast<int4*>(a.part_ml + (size_t)2 * ctas * SH::ROWS);
  XQT_SMEM_OPT_IN((kv4_attention_kernel<T, SH, false>), SH::SMEM);
  int rc = launch_pdl(kv4_attention_kernel<T, SH, false>, dim3((unsigned)ctas), dim3(SH::W * 32), SH::SMEM, stream, a);
  if (rc || ctas == 1) return rc;
  return launch_pdl(kv4_attention_join_kernel<T, SH>, dim3((unsigned)ctas - 1, SH::ROWS / kJoinRows), dim3(kJoinRows * kJoinWarps * 32), 0, stream, a, (unsigned)ctas);
}

template <typename T>
int run_dim(const AttnArgs& a, int dim, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  // two 8-row tiles where eight rows do not hold a key head's queries (128 and 256 channels: the registers of one of 256)
  const bool wide = a.each > 8 || a.query_starts;
  if (dim == 64) return wide ? run<T, 64, 2>(a, workspace, workspace_bytes, stream) : run<T, 64, 1>(a, workspace, workspace_bytes, stream);
  if (dim == 128) return wide ? run<T, 128, 2>(a, workspace, workspace_bytes, stream) : run<T, 128, 1>(a, workspace, workspace_bytes, stream);
  return run<T, 256, 1>(a, workspace, workspace_bytes, stream);
}

}  // namespace
}  // namespace xqt_b200

extern "C" size_t xqt_b200_kv4_attention_workspace_bytes(int tokens, int batch, int q_heads, int kv_heads, int dim, int has_query_starts) {
  using namespace xqt_b200;
  (void)batch;
  const size_t few = (size_t)2 * kMostPerSm * sm_count() * (16 * (dim + 2) * 4 + 16);
  // the two kernels run one after the other and share it
  if (!has_query_starts || kv_heads < 1 || (long long)tokens * (q_heads / kv_heads) <= kFewRows) return few;
  const size_t prompt = kv4_prompt_workspace_bytes(dim);
  return few > prompt ? few : prompt;
}

extern "C" int xqt_b200_kv4_attention(const void* q, const void* codes, const void* params, const int* table, const int* seq_lens, const int* query_starts,
                                      void* out, const long long* strides, int tokens, int batch, int q_heads, int kv_heads, int dim, long long pages,
                                      int page_size, int table_width, int window, int dtype, float scale, void* workspace, size_t workspace_bytes,
                                      unsigned* status, cudaStream_t stream) {
  using namespace xqt_b200;
  XQT_REQUIRE(tokens >= 0 && batch >= 0 && kv_heads >= 1 && kv_heads <= (1 << 16) && q_heads >= kv_heads && q_heads <= (1 << 16) && q_heads % kv_heads == 0);
  XQT_REQUIRE(dim == 64 || dim == 128 || dim == 256);
  XQT_REQUIRE(dtype == XQT_B200_FP16 || dtype == XQT_B200_BF16);
  XQT_REQUIRE(page_size >= 16 && page_size <= 4096 && (page_size & (page_size - 1)) == 0);
  XQT_REQUIRE(pages >= 0 && pages < (1LL << 31) && table_width >= 0 && (long long)table_width * page_size <= (1LL << 30));
  XQT_REQUIRE(window >= 0 && fabsf(scale) < 0x1p127f && (long long)tokens * (q_heads / kv_heads) < (1LL << 31) - 4096);
  if (tokens == 0 || batch == 0) return 0;
  XQT_REQUIRE(q && out && seq_lens && strides && (table_width == 0 || table) && (pages == 0 || (codes && params)));
  XQT_REQUIRE((query_starts != nullptr) || tokens == batch);
  XQT_REQUIRE((((uintptr_t)q | (uintptr_t)out | (uintptr_t)codes | (uintptr_t)params) & 15) == 0 && ((strides[0] | strides[1]) & 7) == 0);
  AttnArgs a = {};
  a.q = q;
  a.codes = (const uint8_t*)codes;
  a.params = (const uint8_t*)params;
  a.table = table;
  a.seq_lens = seq_lens;
  a.query_starts = query_starts;
  a.out = out;
  a.status = status;
  a.q_token = strides[0];
  a.q_head = strides[1];
  a.table_stride = strides[2];
  a.pages = pages;
  a.tokens = tokens;
  a.batch = batch;
  a.q_heads = q_heads;
  a.kv_heads = kv_heads;
  a.each = q_heads / kv_heads;
  a.page_size = page_size;
  a.page_shift = __builtin_ctz((unsigned)page_size);
  a.table_width = table_width;
  a.window = window;
  a.scale = scale * 1.4426950408889634f;
  // Sequences with more than kFewRows rows go to the prompt kernel, whose tiles of 128 or 256 rows run at half of the tensor core's rate where they are full, unless the whole call is so little work that its two launches more are not worth it (keys: as
  // many as the table holds).  Both sides measured, this kernel for all | prompt kernel above 32 rows: one sequence, 40 queries of 32 heads on 2000
  // keys 25 | 33 us, 64 queries 31 | 36, 16 queries on 30,000 keys 62 | 66; 64 sequences of 16 queries on 2000 keys 332 | 275, of 9 queries 249 | 273.
  // All with tables that fit; behind one of 131,072 keys the rule takes the second side (40 queries on 2000 keys: 31 us instead of 24).
  a.few_rows = INT_MAX;
  if (query_starts != nullptr && (long long)tokens * a.each > kFewRows &&
      (double)tokens * q_heads * table_width * page_size * dim > 768e6) {
    a.few_rows = kFewRows;
    const int rc = kv4_prompt_launch(a, dim, dtype, workspace, workspace_bytes, stream);
    if (rc) return rc;
  }
  return dtype == XQT_B200_BF16 ? run_dim<__nv_bfloat16>(a, dim, workspace, workspace_bytes, stream)
                                : run_dim<__half>(a, dim, workspace, workspace_bytes, stream);
}
