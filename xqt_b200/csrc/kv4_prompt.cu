// Attention of many queries (prompts, chunks of prompts) over the paged 4-bit cache (layout: kv4_cache.cu; the mathematics and the rules
// for what a query sees: kv4_attention.cu), on the tensor cores.
//
// An item is TILES row tiles of 128 (row = query * heads of the key head + head) of one sequence and key head, and the keys they see, BN at
// a time; the chunks of all items form one list, dealt out evenly to one CTA per SM, and items that CTAs share are joined by a second kernel.
// Codes come in by bulk copies; four warps turn them into fp16 keys and values in shared memory (128-byte swizzle), once for all rows; one
// thread per row tile issues S = Q K^T and O += P V (tcgen05, sums in tensor memory); four warps per row tile, a thread per row, do the
// softmax: P goes back to tensor memory over the scores that it came from.  Scores are double-buffered: those of the next chunk are made
// while the softmax works on this one's.
//
//   warp 0       table look-ups and bulk copies
//   warp 2       allocates tensor memory, prefetches queries
//   warps 1, 3   tcgen05.mma, one issuer per row tile: an answer of a barrier takes about 200 clocks, and one thread waiting for both tiles in
//                turn set the pace (8192-token prompt: 476 us of 605 with all other work left out)
//   warps 4-7    codes -> fp16
//   warps 8-15   softmax, rescaling of O, result
//
// Scales.  fp16 has the mantissa that keeps the result as exact as the inputs (bf16 operands lose 8 times more), but not the range, so all
// three operands go in with a power of two: a query row with its own (largest element in [1, 2)), the keys of a chunk with one
// for the chunk (largest in [2^13, 2^14)), values with one that only grows along the sequence (O is rescaled then).  The powers come back
// in the fp32 factor of the scores and at the end.  P is formed against a running maximum that moves only when a row exceeds
// it by 2^8, so O is rescaled rarely, and times 2^7 (in its sum and in O alike): P <= 2^15 fits fp16, and an element below 2^-14, whose
// rounding is not relative to it any more, stands for at most 2^-21 of the row's largest; what rounds to 0 for 2^-32.
//
// Rounding keys, values and P to fp16 adds about as much error each as rounding the result does: nothing beside a bf16 result's own rounding, but twice
// an fp16 result's.  So for fp16 the converting warps keep what their rounding leaves of keys and values as a second operand, and both products are made
// twice (PARTS = 2): the error is 1.3 to 1.4 roundings of the result instead of 2.  It costs shared memory (two stages instead of four; 32 keys at
// a time for 256 channels) and time: the 8192-token prompt 697 | 558 us (64 channels, fp16 | bf16), 1115 | 629 (128), 4005 | 1766 (256).
//
// The tensor core cuts off the bits of a product that stand below its running sum's, so a sum that grew over a whole long context would be too small, by
// 1.6 half steps of an fp16 result after 131,072 keys of equal weight, by up to 4 where one key is far more probable than the others.  O therefore
// starts afresh after a RUN of keys (4096 for fp16, 16,384 for bf16, whose result holds 8 times less): what it held is added, rounded to
// nearest, to the row's part in the workspace (2048 queries on 65,536 keys, without | with: fp16 3914 | 3992 us, bf16 2120 | 2159).
//
// A vector that is not finite counts as NaN: its key becomes NaN, its value 0, so the rows that see it are NaN and the others never
// meet it.  Keys that are not there (no page, past the end) become 0 and are masked.
//
// The order of a word's codes: pairs (0,4) (1,5) (2,6) (3,7) come out of one AND each, so channels stand in shared memory as 0 4 1 5 2 6 3 7 in
// every group of eight; queries are stored in the same order, and the result is put back when it is written.
//
// Bound by shared memory (operands 42 % of the clocks for 128 channels in bf16, the warps' own accesses 23 %), the tensor core and ex2 (16 a clock and SM),
// 41 % each; what is left between that and the measured time is the chain scores -> softmax -> P -> product, of which two tiles overlap, and what an item costs before and after its chunks.
// Measured: 629 us for the prompt of 8192 tokens (32 heads on 8 of 128 channels: 874 TFLOP/s, half of a library GEMM's rate), 474 us for chunks of
// four prompts, 8188 queries of 40 heads on 8 in all (760 TFLOP/s).
#include <type_traits>

#include "kv4_attention.cuh"

namespace xqt_b200 {

namespace {

using namespace kv4;

template <int D_, int TILES_, int STAGES_, int PARTS_, int BN_>
struct PromptShape {
  static constexpr int D = D_, TILES = TILES_, STAGES = STAGES_, BN = BN_;    // STAGES: of codes, keys and values
  static constexpr int PARTS = PARTS_;                         // 2: what rounding a key or value to fp16 leaves is a second operand
  static constexpr int GROUP_WARPS = 4 / STAGES;               // that convert one chunk
  static constexpr int ROWS = 128 * TILES, UNIT = BN, CT = BN;
  static constexpr int OPENING = 7 * 64 / BN;                  // what an item costs besides its chunks, in chunks
  static constexpr int RUN = (PARTS == 2 ? 4096 : 16384) / BN;   // chunks that O is summed over in tensor memory
  static constexpr bool PROMPT = true;
  static constexpr int THREADS = 256 + 128 * TILES;
  static constexpr int BLOCKS = D / 64;                        // 128-byte wide column blocks of an operand
  static constexpr int Q_BYTES = ROWS * D * 2, PART_BYTES = BN * D * 2, KV_BYTES = PARTS * PART_BYTES;
  static constexpr int CODE_BYTES = BN * D / 2, PARAM_BYTES = BN * 4, RAW_BYTES = 2 * (CODE_BYTES + PARAM_BYTES);
  static constexpr int OFF_K = Q_BYTES, OFF_V = OFF_K + STAGES * KV_BYTES, OFF_RAW = OFF_V + STAGES * KV_BYTES, OFF_MISC = OFF_RAW + STAGES * RAW_BYTES;
  static constexpr int SMEM = OFF_MISC + 768;
  // tensor memory: two buffers of scores per tile from column 0, P over the first half of its scores; O from 256
  static constexpr uint32_t O_COL = 256;
  static_assert(2 * TILES * BN <= 256 && TILES * D <= 256 && SMEM <= 227 * 1024 && (STAGES == 2 || STAGES == 4) && (BN == 64 || (BN == 32 && STAGES == 2)), "tensor and shared memory");
};

// Barriers, in 8-byte words behind the tiles.  Those of scores, P and O are per tile and chunk parity: a softmax warp may be a chunk ahead of its
// neighbours, and a wait may come two products late.
enum : int { kRawFull = 0, kRawEmpty = 4, kKReady = 8, kVReady = 12, kKEmpty = 16, kVEmpty = 20, kSFull = 24, kPReady = 28, kODone = 32, kGrown = 36, kQReady = 40 };
constexpr float kLift = 7.0f;      // log2 of P where a score equals the running maximum
constexpr int kRing = 16;          // chunks that loader, conversion and softmax may lie apart: more than 2 + 2 * STAGES

template <int N>
struct Ring {
  int slot = 0, phase = 0;
  __device__ __forceinline__ void next() {
    if (++slot == N) {
      slot = 0;
      phase ^= 1;
    }
  }
};

__device__ __forceinline__ void wait_ld_dep32(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;\n"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
                 "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]),
                 "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]),
                 "+r"(r[31])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};\n" ::"r"(taddr),
               "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
               "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
               : "memory");
}
// Shared-memory operand whose long side is the contiguous one (values as the second operand of P V), 128-byte swizzle: 64 channels of eight
// keys are 1024 bytes, the next eight keys follow, the next 64 channels are `block_bytes` away.
__device__ __forceinline__ uint64_t umma_desc_mn_sw128(uint32_t saddr, uint32_t block_bytes) {
  return (uint64_t)((saddr & 0x3FFFF) >> 4) | (uint64_t)(block_bytes >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
__device__ __forceinline__ uint32_t half2_bits(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }
__device__ __forceinline__ __half2 bits_half2(uint32_t v) { return *reinterpret_cast<const __half2*>(&v); }
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }     // -126 <= e <= 127
// e with |v| < 2^e, in [-100, 127]
__device__ __forceinline__ int above(float v) { return min(max((int)(__float_as_uint(v) >> 23) - 126, -100), 127); }

// eight codes -> c * s + m in fp16, rounded once (the codes themselves are exact: 1024 + c and 64 + c less that)
__device__ __forceinline__ uint4 eight(uint32_t x, __half2 s, __half2 m) {
  const __half2 k1024 = bits_half2(0x64006400u), k64 = bits_half2(0x54005400u);
  const uint32_t y = x >> 8;
  uint4 r;
  r.x = half2_bits(__hfma2(__hsub2(bits_half2((x & 0x000f000fu) | 0x64006400u), k1024), s, m));
  r.y = half2_bits(__hfma2(__hsub2(bits_half2((x & 0x00f000f0u) | 0x54005400u), k64), s, m));
  r.z = half2_bits(__hfma2(__hsub2(bits_half2((y & 0x000f000fu) | 0x64006400u), k1024), s, m));
  r.w = half2_bits(__hfma2(__hsub2(bits_half2((y & 0x00f000f0u) | 0x54005400u), k64), s, m));
  return r;
}

// the same, and what the rounding left (sums of two halves and products of two are exact with their errors)
__device__ __forceinline__ void both_parts(__half2 c, __half2 s, __half2 m, uint32_t& high, uint32_t& low) {
  const __half2 p = __hmul2_rn(c, s), of_p = __hfma2(c, s, __hneg2(p)), h = __hadd2_rn(p, m), b = __hsub2_rn(h, p);
  high = half2_bits(h);
  low = half2_bits(__hadd2_rn(__hadd2_rn(__hsub2_rn(p, __hsub2_rn(h, b)), __hsub2_rn(m, b)), of_p));
}
__device__ __forceinline__ uint4 eight(uint32_t x, __half2 s, __half2 m, uint4& low) {
  const __half2 k1024 = bits_half2(0x64006400u), k64 = bits_half2(0x54005400u);
  const uint32_t y = x >> 8;
  uint4 r;
  both_parts(__hsub2_rn(bits_half2((x & 0x000f000fu) | 0x64006400u), k1024), s, m, r.x, low.x);
  both_parts(__hsub2_rn(bits_half2((x & 0x00f000f0u) | 0x54005400u), k64), s, m, r.y, low.y);
  both_parts(__hsub2_rn(bits_half2((y & 0x000f000fu) | 0x64006400u), k1024), s, m, r.z, low.z);
  both_parts(__hsub2_rn(bits_half2((y & 0x00f000f0u) | 0x54005400u), k64), s, m, r.w, low.w);
  return r;
}

// Both functions below are not inlined: their registers would crowd those of the softmax loop, and they run once per item.
//
// The 32 query rows of a warp, each lane its own (or null), to shared memory: scaled by a power of two per row, fp16, channels in the order of
// the codes, 128-byte swizzle.  Returns what the lane's scores have to be multiplied by.
template <typename T, int D>
__device__ __noinline__ float load_queries(const T* src, uint8_t* dst, float scale) {
  const int lane = threadIdx.x & 31;
  float factor = 0.0f;
  // D / 8 lanes read a row together (a row per lane would touch 32 lines with every load): its largest, then scaled and stored
  constexpr int LPR = D / 8, RPR = 32 / LPR, BATCH = LPR < 8 ? LPR : 8;
  const float sign = scale == 0.0f ? 0.0f : copysignf(1.0f, scale), size = scale == 0.0f ? 1.0f : fabsf(scale);
  const int c = lane % LPR;
#pragma unroll 1
  for (int first = 0; first < LPR; first += BATCH) {
    uint4 x[BATCH];
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      const T* const from_row = reinterpret_cast<const T*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(src), (first + k) * RPR + lane / LPR));
      x[k] = from_row != nullptr ? *reinterpret_cast<const uint4*>(from_row + 8 * c) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      const T* const v = reinterpret_cast<const T*>(&x[k]);
      // magnitudes order as their bits
      uint32_t most = __vmaxu2(__vmaxu2(x[k].x & 0x7fff7fffu, x[k].y & 0x7fff7fffu), __vmaxu2(x[k].z & 0x7fff7fffu, x[k].w & 0x7fff7fffu));
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) most = __vmaxu2(most, __shfl_xor_sync(0xffffffffu, most, o));
      const float2 most2 = pair_of<T>(most);
      const float top = fmaxf(most2.x, most2.y);
      const int e = top > 0.0f && top <= 3.402823466e38f ? min(max(above(top) - 1, -100), 100) : 0;
      const float down = pow2(-e) * sign, of_owner = __shfl_sync(0xffffffffu, pow2(e) * size, lane % RPR * LPR);
      if (lane / RPR == first + k) factor = of_owner;
      uint4 y;
      y.x = half2_bits(__floats2half2_rn(to_float<T>(v[0]) * down, to_float<T>(v[4]) * down));
      y.y = half2_bits(__floats2half2_rn(to_float<T>(v[1]) * down, to_float<T>(v[5]) * down));
      y.z = half2_bits(__floats2half2_rn(to_float<T>(v[2]) * down, to_float<T>(v[6]) * down));
      y.w = half2_bits(__floats2half2_rn(to_float<T>(v[3]) * down, to_float<T>(v[7]) * down));
      const int at = (first + k) * RPR + lane / LPR;
      *reinterpret_cast<uint4*>(dst + (c >> 3) * (128 * 128) + at * 128 + (((c & 7) ^ (at & 7)) << 4)) = y;
    }
  }
  return factor;
}

// The 32 rows of a warp from tensor memory, times `by`: kResult, to the rows of the result; kPart, to the rows' parts (fp32); kAdded, added to those; kScaled,
// added to what they hold times `keep`; kSum, the same, but to the rows of the result.  Each lane gives its own row's addresses (0: no row) and factors.
enum : int { kResult, kPart, kAdded, kScaled, kSum };
template <typename T, int D>
__device__ __noinline__ void store_rows(uint32_t o_at, unsigned long long part, unsigned long long out, float by, float keep, int how) {
  const int lane = threadIdx.x & 31;
  // Four lanes write 64 bytes of a row together (a lane alone would touch a line of its own with every store): they exchange 16-byte pieces,
  // piece i of row k for piece k of row i.  A part's piece is the same lane's every time, so nothing depends on an order among lanes.
  unsigned long long parts_at[4], outs_at[4];
  float keeps[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    parts_at[k] = __shfl_sync(0xffffffffu, part, (lane & 28) + k);
    outs_at[k] = __shfl_sync(0xffffffffu, out, (lane & 28) + k);
    keeps[k] = __shfl_sync(0xffffffffu, keep, (lane & 28) + k);
  }
  auto exchange = [&](uint4 (&x)[4]) {
    auto swap = [](uint4& keep_low, uint4& keep_high, bool upper, int o) {
      uint4 give = upper ? keep_low : keep_high;
      give.x = __shfl_xor_sync(0xffffffffu, give.x, o);
      give.y = __shfl_xor_sync(0xffffffffu, give.y, o);
      give.z = __shfl_xor_sync(0xffffffffu, give.z, o);
      give.w = __shfl_xor_sync(0xffffffffu, give.w, o);
      if (upper) keep_low = give;
      else keep_high = give;
    };
    swap(x[0], x[1], lane & 1, 1);
    swap(x[2], x[3], lane & 1, 1);
    swap(x[0], x[2], lane & 2, 2);
    swap(x[1], x[3], lane & 2, 2);
  };
#pragma unroll 1
  for (int c = 0; c < D / 32; ++c) {
    uint32_t r[32];
    tmem_ld_32x32(o_at + 32 * c, r);
    wait_ld_dep32(r);
    auto value = [&](int e) { return __uint_as_float(r[(e & ~7) + ((e & 7) < 4 ? 2 * (e & 7) : 2 * (e & 7) - 7)]) * by; };      // channel e of these 32
    uint4 x[4];
    if (how == kResult) {
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        T* const t = reinterpret_cast<T*>(&x[b]);
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = from_float<T>(value(8 * b + e));
      }
      exchange(x);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (outs_at[k] != 0) *reinterpret_cast<uint4*>(outs_at[k] + 64 * c + 16 * (lane & 3)) = x[k];
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int b = 0; b < 4; ++b)
          x[b] = make_uint4(__float_as_uint(value(16 * h + 4 * b)), __float_as_uint(value(16 * h + 4 * b + 1)), __float_as_uint(value(16 * h + 4 * b + 2)),
                            __float_as_uint(value(16 * h + 4 * b + 3)));
        exchange(x);
        const int offset = 128 * c + 64 * h + 16 * (lane & 3);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (parts_at[k] == 0) continue;
          float4 v = make_float4(__uint_as_float(x[k].x), __uint_as_float(x[k].y), __uint_as_float(x[k].z), __uint_as_float(x[k].w));
          float4* const at = reinterpret_cast<float4*>(parts_at[k] + offset);
          if (how == kAdded) {                       // no answer to wait for (with kScaled always the fp16 figure above is 4239)
            atomicAdd(at, v);
            continue;
          }
          if (how >= kScaled) {
            const float4 old = __ldcg(at);
            v = make_float4(fmaf(old.x, keeps[k], v.x), fmaf(old.y, keeps[k], v.y), fmaf(old.z, keeps[k], v.z), fmaf(old.w, keeps[k], v.w));
          }
          if (how == kSum) {
            T t[4] = {from_float<T>(v.x), from_float<T>(v.y), from_float<T>(v.z), from_float<T>(v.w)};
            *reinterpret_cast<uint2*>(outs_at[k] + offset / 2) = *reinterpret_cast<uint2*>(t);
          } else {
            *at = v;
          }
        }
      }
    }
  }
}

// An item of the list and a unit of it: SH::OPENING units stand for its queries and its result, the others are its chunks.
struct PromptItem {
  int b, tile, head, unit, begin, chunks;
  Sequence s;
};

// Chunks [lo, hi) of an item, SH::RUN at most: whether they are the first and the last of those that are this CTA's, whether those are the whole item
// and whether they are its beginning; and how many chunks the CTA has had before.
struct Run {
  int lo, hi, before;
  bool first, last, whole, opens;
};

// the keys that some row of a tile sees start in chunk begin / BN; how many chunks
template <typename SH>
__device__ __forceinline__ int prompt_chunks(const AttnArgs& a, const Sequence& s, int tile, int& begin) {
  const int pos0 = s.len - s.nq;                                       // the position of the sequence's first query
  const int j0 = tile * SH::ROWS / a.each, j1 = min(s.nq - 1, (tile * SH::ROWS + SH::ROWS - 1) / a.each);
  const int end = pos0 + j1 + 1;
  begin = a.window ? (int)max((long long)pos0 + j0 - a.window + 1, 0LL) / SH::BN * SH::BN : 0;
  return end > begin ? (end - begin + SH::BN - 1) / SH::BN : 0;
}

// Goes through the tiles of all sequences, 32 at a time, and calls visit(b, sequence, first tile, this lane's units) until it says to stop;
// one warp.
template <typename SH, typename V>
__device__ __forceinline__ void prompt_tiles(const AttnArgs& a, int lane, V visit) {
  for (int b0 = 0; b0 < a.batch; b0 += 32) {
    Sequence mine = {};
    if (b0 + lane < a.batch) mine = sequence<SH>(a, b0 + lane);
    for (unsigned some = __ballot_sync(0xffffffffu, mine.tiles > 0); some; some &= some - 1) {
      const int at = __ffs(some) - 1;
      const Sequence s = sequence_of(mine, at);
      for (int t0 = 0; t0 < s.tiles; t0 += 32) {
        int begin;
        const unsigned units = t0 + lane < s.tiles ? (unsigned)a.kv_heads * (prompt_chunks<SH>(a, s, t0 + lane, begin) + SH::OPENING) : 0u;
        if (!visit(b0 + at, s, t0, units)) return;
      }
    }
  }
}

template <typename SH>
__device__ __forceinline__ Deal prompt_deal(const AttnArgs& a, int lane, unsigned ctas) {
  Deal d = {};
  unsigned sum = 0;
  prompt_tiles<SH>(a, lane, [&](int, const Sequence&, int, unsigned units) {
    sum += units;
    return true;
  });
  d.total = __reduce_add_sync(0xffffffffu, sum);
  d.each = d.total / ctas;
  d.more = d.total - d.each * ctas;
  return d;
}

template <typename SH>
__device__ __forceinline__ void prompt_place(const AttnArgs& a, int lane, unsigned u, PromptItem& w) {
  unsigned base = 0;
  prompt_tiles<SH>(a, lane, [&](int b, const Sequence& s, int t0, unsigned units) {
    const unsigned cum = scan32(units, lane), over = __ballot_sync(0xffffffffu, base + cum > u);
    if (over) {
      const int at = __ffs(over) - 1;
      const unsigned rest = u - base - __shfl_sync(0xffffffffu, cum - units, at);
      w.b = b;
      w.s = s;
      w.tile = t0 + at;
      w.chunks = prompt_chunks<SH>(a, s, w.tile, w.begin);
      w.head = (int)(rest / (unsigned)(w.chunks + SH::OPENING));
      w.unit = (int)(rest - (unsigned)w.head * (w.chunks + SH::OPENING));
      return false;
    }
    base += __shfl_sync(0xffffffffu, cum, 31);
    return true;
  });
}

// the item behind w
template <typename SH>
__device__ __forceinline__ void prompt_next(const AttnArgs& a, PromptItem& w) {
  w.unit = 0;
  if (++w.head < a.kv_heads) return;
  w.head = 0;
  if (++w.tile >= w.s.tiles) {
    w.tile = 0;
    while (++w.b < a.batch) {
      w.s = sequence<SH>(a, w.b);
      if (w.s.tiles > 0) break;
    }
  }
  w.chunks = w.b < a.batch ? prompt_chunks<SH>(a, w.s, w.tile, w.begin) : 0;      // (starts that do not ascend can make the list shorter than it counts)
}

template <typename T, typename SH>
__global__ void __launch_bounds__(SH::THREADS, 1) kv4_prompt_kernel(const AttnArgs a) {
  constexpr int D = SH::D, TILES = SH::TILES, BN = SH::BN, BLOCKS = SH::BLOCKS;
  const float kLowest = -CUDART_INF_F;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint8_t* const misc = smem + SH::OFF_MISC;
  const uint32_t bar0 = smem_addr(misc);
  auto bar = [&](int slot) { return bar0 + 8u * (uint32_t)slot; };
  volatile uint32_t* const s_mask = reinterpret_cast<volatile uint32_t*>(misc + 336);       // [kRing] which 16-key groups of a chunk are there
  volatile float* const s_key = reinterpret_cast<volatile float*>(misc + 400);               // [kRing] what a chunk's keys were divided by
  volatile float* const s_value = reinterpret_cast<volatile float*>(misc + 464);             // [kRing] what O has to be multiplied by before it
  volatile float* const s_scale = reinterpret_cast<volatile float*>(misc + 528);             // [kRing] what its values were divided by
  volatile int* const s_grown = reinterpret_cast<volatile int*>(misc + 592);                 // [4] values so far are below 2^this
  volatile uint32_t* const s_abort = reinterpret_cast<volatile uint32_t*>(misc + 608);
  uint32_t* const s_tmem = reinterpret_cast<uint32_t*>(misc + 612);
  PromptItem* const s_start = reinterpret_cast<PromptItem*>(misc + 616);
  unsigned* const s_range = reinterpret_cast<unsigned*>(misc + 616 + sizeof(PromptItem));    // [2]

  grid_launch_dependents();
  grid_dependency_wait();
  if (warp == 0) {
    const Deal d = prompt_deal<SH>(a, lane, gridDim.x);
    const unsigned u0 = d.start(blockIdx.x), u1 = d.start(blockIdx.x + 1);
    PromptItem first = {};
    if (u0 < u1) prompt_place<SH>(a, lane, u0, first);
    if (lane == 0) {
      *s_start = first;
      s_range[0] = u0;
      s_range[1] = u1;
      a.plan[blockIdx.x] = make_int4((int)d.total, first.unit, first.chunks + SH::OPENING, first.head);
      a.plan[gridDim.x + blockIdx.x] = make_int4(first.b, first.tile, first.s.q0, first.s.nq);
    }
  }
  if (tid == 0) {
    *s_abort = 0;
    for (int i = 0; i < 4; ++i) {
      mbar_init(bar(kRawFull + i), 1);
      mbar_init(bar(kRawEmpty + i), SH::GROUP_WARPS);
      mbar_init(bar(kKReady + i), SH::GROUP_WARPS);
      mbar_init(bar(kVReady + i), SH::GROUP_WARPS);
      mbar_init(bar(kGrown + i), 1);
      mbar_init(bar(kKEmpty + i), TILES);
      mbar_init(bar(kVEmpty + i), TILES);
      mbar_init(bar(kSFull + i), 1);
      mbar_init(bar(kPReady + i), 4);
      mbar_init(bar(kODone + i), 1);
    }
    for (int i = 0; i < 2; ++i) mbar_init(bar(kQReady + i), 4);
    fence_barrier_init();
  }
  if (warp == 2) {
    tmem_alloc(smem_addr(s_tmem), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  // The CTA's part of the list: `body` gets an item and a run of its chunks.  Every role goes through it for itself.  Returns how many chunks there were.
  auto runs = [&](auto body) {
    PromptItem w = *s_start;
    unsigned left = s_range[1] - s_range[0];
    int before = 0;
    while (left > 0) {
      const unsigned units = (unsigned)(w.chunks + SH::OPENING), take = min(units - w.unit, left);
      const int lo = max(w.unit - SH::OPENING, 0), hi = max((int)(w.unit + take) - SH::OPENING, 0);
      const bool opens = w.unit == 0, whole = opens && take == units;
      int at = lo;
      do {
        const int to = min(at + SH::RUN, hi);
        body(w, Run{at, to, before, at == lo, to == hi, whole, opens});
        before += to - at;
        at = to;
      } while (at < hi);
      left -= take;
      if (left > 0) prompt_next<SH>(a, w);
    }
    return before;
  };
  // Every wait is bounded: when one runs out, no role waits for another any more, and the host is told.  Who has copies or products in flight then waits for
  // those, with a limit again, before the CTA gives its memory back.
  auto guarded = [&](uint32_t b, uint32_t parity) {
    if (*s_abort == 0u && !mbar_wait(b, parity)) {
      *s_abort = 1u;
      if (a.status) *a.status = 1u;
    }
  };

  // the same by polling, where the wake-up of a suspended thread would set the pace
  auto polled = [&](uint32_t b, uint32_t parity) {
    if (*s_abort == 0u && !mbar_spin(b, parity)) {
      *s_abort = 1u;
      if (a.status) *a.status = 1u;
    }
  };

  auto polled2 = [&](uint32_t b0, uint32_t parity0, uint32_t b1, uint32_t parity1) {
    if (*s_abort != 0u) return;
    for (uint32_t i = 0; i < (kSpinLimit << 3); ++i) {
      const bool x = mbar_test_wait(b0, parity0), y = mbar_test_wait(b1, parity1);
      if (x && y) return;
    }
    *s_abort = 1u;
    if (a.status) *a.status = 1u;
  };

  int mine = 0;                                      // warp 0: where its ring stands; issuers: their products
  if (warp == 0) {
    // ------------------------------------------------------------ codes and parameters into the raw ring
    const int psz = min(a.page_size, BN), pieces = BN / psz, groups = psz / 16;
    const int piece = lane >> 2, kind = lane & 3;                    // kind: key codes, value codes, key parameters, value parameters
    const int row_bytes = kind < 2 ? D / 2 : 4;
    const long long page_bytes = 2LL * a.kv_heads * a.page_size * row_bytes;
    const uint32_t target = smem_addr(smem + SH::OFF_RAW) +
                            (kind == 0 ? 0 : kind == 1 ? SH::CODE_BYTES : kind == 2 ? 2 * SH::CODE_BYTES : 2 * SH::CODE_BYTES + SH::PARAM_BYTES) + piece * psz * row_bytes;
    Ring<SH::STAGES> ring;
    runs([&](const PromptItem& w, const Run& run) {
      const int lo = run.lo, hi = run.hi, before = run.before;
      const uint8_t* const source = (kind < 2 ? a.codes : a.params) + ((long long)(kind & 1) * a.kv_heads + w.head) * a.page_size * row_bytes;
      const int* const table = a.table + w.b * a.table_stride;
      auto look_up = [&](int i) {
        const int at = w.begin + i * BN + piece * psz;
        return i < hi && piece < pieces && at < w.s.len ? table[at >> a.page_shift] : -1;
      };
      int page = look_up(lo);
      for (int i = lo; i < hi; ++i, ring.next()) {
        const int stage = ring.slot, following = look_up(i + 1);
        const bool valid = (unsigned)page < (unsigned)a.pages;
        const unsigned votes = __ballot_sync(0xffffffffu, valid);
        unsigned mask = 0;
#pragma unroll
        for (int p = 0; p < BN / 16; ++p) mask |= (votes >> (4 * (p / groups)) & 1u) << p;
        guarded(bar(kRawEmpty + stage), ring.phase ^ 1);
        if (!__all_sync(0xffffffffu, *s_abort == 0u)) break;      // one answer for the warp: what is announced is copied, and the ring stands still
        if (lane == 0) {
          s_mask[(before + i - lo) % kRing] = mask;
          mbar_expect_tx(bar(kRawFull + stage), (uint32_t)(__popc(mask) * 16 * 2 * (D / 2 + 4)));
        }
        __syncwarp();
        const int at = w.begin + i * BN + piece * psz;
        if (valid)
          bulk_g2s(target + stage * SH::RAW_BYTES, source + page * page_bytes + (long long)(at & (a.page_size - 1)) * row_bytes, (uint32_t)(psz * row_bytes), bar(kRawFull + stage));
        page = following;
      }
    });
    mine = 2 * ring.slot + ring.phase;
  } else if (warp == 1 || (TILES == 2 && warp == 3)) {
    // ------------------------------------------------------------ the tensor core, for one row tile
    if (elect_one()) {
      constexpr uint32_t kScores = umma_idesc(kAccF32, kFmtF16, kFmtF16, 128, BN);
      constexpr uint32_t kOut = umma_idesc(kAccF32, kFmtF16, kFmtF16, 128, D) | 1u << 16;      // second operand: long side contiguous
      const int tile = warp >> 1;
      const uint32_t base = smem_addr(smem), s_tile = tmem + 2 * tile * BN, o_tile = tmem + SH::O_COL + tile * D;
      const uint64_t q_desc = umma_desc_sw128(base + tile * (BLOCKS * 128 * 128)), k_desc = umma_desc_sw128(base + SH::OFF_K);
      const uint64_t v_desc = umma_desc_mn_sw128(base + SH::OFF_V, BN * 128);
      // scores run one chunk ahead; a buffer of theirs is free again behind the product that read P from it (the tensor core works in order)
      Ring<SH::STAGES> kr, vr;
      uint32_t q_phase = 0;
      mine = runs([&](const PromptItem&, const Run& run) {
        const int lo = run.lo, hi = run.hi, before = run.before;
        if (hi == lo) return;
        if (run.first) {
          polled(bar(kQReady + tile), q_phase);
          q_phase ^= 1;
        }
        bool k_ready = false;
        const int n_end = before + hi - lo;
        for (int n = before; n <= n_end; ++n) {
          if (n < n_end) {
            if (!k_ready) polled(bar(kKReady + kr.slot), kr.phase);
            tc_fence_after();
            const uint64_t kd = k_desc + kr.slot * (SH::KV_BYTES >> 4);
#pragma unroll
            for (int part = 0; part < SH::PARTS; ++part)
#pragma unroll
              for (int s = 0; s < D / 16; ++s)
                umma_ss(s_tile + (n & 1) * BN, q_desc + (s >> 2) * (128 * 128 >> 4) + 2 * (s & 3), kd + part * (SH::PART_BYTES >> 4) + (s >> 2) * (BN * 128 >> 4) + 2 * (s & 3), kScores,
                        part || s ? 1u : 0u);
            umma_commit(bar(kSFull + 2 * tile + (n & 1)));
            umma_commit(bar(kKEmpty + kr.slot));
            kr.next();
          }
          k_ready = n + 1 < n_end && mbar_test_wait(bar(kKReady + kr.slot), kr.phase);      // answered while the wait below goes on
          if (n > before) {
            const int last = n - 1;
            polled2(bar(kVReady + vr.slot), vr.phase, bar(kPReady + 2 * tile + (last & 1)), last >> 1 & 1);
            tc_fence_after();
            const uint64_t vd = v_desc + vr.slot * (SH::KV_BYTES >> 4);
#pragma unroll
            for (int part = 0; part < SH::PARTS; ++part)
#pragma unroll
              for (int s = 0; s < BN / 16; ++s)
                umma_ts_f16(o_tile, s_tile + (last & 1) * BN + 8 * s, vd + part * (SH::PART_BYTES >> 4) + s * (2048 >> 4), kOut, last > before || part || s ? 1u : 0u);
            umma_commit(bar(kVEmpty + vr.slot));
            umma_commit(bar(kODone + 2 * tile + (last & 1)));      // the last of what is in flight: the softmax waits for it
            vr.next();
          }
        }
      });
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------ the queries of all the CTA's items into L2, ahead of their use
    runs([&](const PromptItem& w, const Run& run) {
      if (run.hi == run.lo || !run.first) return;
      for (int r = lane; r < SH::ROWS; r += 32) {
        const int row = w.tile * SH::ROWS + r, j = row / a.each;
        if (j >= w.s.nq) return;
        const T* const src = reinterpret_cast<const T*>(a.q) + (long long)(w.s.q0 + j) * a.q_token + (long long)(w.head * a.each + row - j * a.each) * a.q_head;
#pragma unroll
        for (int c = 0; c < D; c += 64) asm volatile("prefetch.global.L2 [%0];\n" ::"l"(src + c));
      }
    });
  } else if (warp >= 4 && warp < 8) {
    // ------------------------------------------------------------ codes -> fp16, chunk i by the warps of group i % STAGES
    // (converting a chunk is a chain of waits and shuffles that a warp cannot overlap with itself; a group has a slot of each ring to itself,
    // so the phase that it waits for is never two away)
    constexpr int PIECES = D / 32;                                   // 16-byte pieces of a key's codes
    constexpr int GROUP = SH::GROUP_WARPS;
    const int slot = (warp & 3) / GROUP;
    const uint8_t* const raw = smem + SH::OFF_RAW + slot * SH::RAW_BYTES;
    runs([&](const PromptItem& w, const Run& run) {
      const int lo = run.lo, hi = run.hi, before = run.before;
      for (int n = before + (slot - before % SH::STAGES + SH::STAGES) % SH::STAGES; n < before + hi - lo; n += SH::STAGES) {
        const int i = lo + n - before;
        const uint32_t phase = n / SH::STAGES & 1;
        guarded(bar(kRawFull + slot), phase);
        const uint32_t* const kp = reinterpret_cast<const uint32_t*>(raw + 2 * SH::CODE_BYTES);
        const uint32_t* const vp = kp + BN;
        const uint32_t mask = s_mask[n % kRing];
        const int t0 = w.begin + i * BN;
        // the chunk's largest key and value element; what is not there or not finite does not count
        constexpr int HALVES = BN / 32;
        float2 k[HALVES], v[HALVES];
        bool there[HALVES], k_good[HALVES], v_good[HALVES];
        float top_k = 0.0f, top_v = 0.0f;
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
          const int row = lane + 32 * h;
          there[h] = (mask >> (row >> 4) & 1u) && t0 + row < w.s.len;
          k[h] = pair_of<T>(kp[row]);
          v[h] = pair_of<T>(vp[row]);
          v_good[h] = fabsf(v[h].x) <= 3.402823466e38f && fabsf(v[h].y) <= 3.402823466e38f;
          k_good[h] = fabsf(k[h].x) <= 3.402823466e38f && fabsf(k[h].y) <= 3.402823466e38f;
          const float tk = fmaxf(fabsf(k[h].y), fabsf(fmaf(15.0f, k[h].x, k[h].y))), tv = fmaxf(fabsf(v[h].y), fabsf(fmaf(15.0f, v[h].x, v[h].y)));
          if (there[h] && k_good[h]) top_k = fmaxf(top_k, fminf(tk, 3.402823466e38f));
          if (there[h] && v_good[h]) top_v = fmaxf(top_v, fminf(tv, 3.402823466e38f));
        }
        const int ek = above(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top_k))));      // (positive floats order as their bits)
        const int own = above(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top_v))));
        // values are divided by a power that only grows along an item: the chunk before says how far it has
        if (n > 0) guarded(bar(kGrown + (n - 1 & 3)), (n - 1) >> 2 & 1);
        // (an item's first chunk leaves a factor of four for later ones, so that O is hardly ever rescaled for them)
        const int grown = i > lo ? s_grown[n - 1 & 3] : min(own + 2, 127), ev = max(grown, own);
        __syncwarp();
        if (lane == 0 && (warp & 3) % GROUP == 0) {
          s_grown[n & 3] = ev;
          s_key[n % kRing] = pow2(max(ek - 14, -126));
          s_value[n % kRing] = pow2(max(grown - ev, -126));
          s_scale[n % kRing] = pow2(max(ev - 14, -126));
          mbar_arrive(bar(kGrown + (n & 3)));
        }
        const float fk = pow2(14 - ek), fv = pow2(14 - ev), nan = __int_as_float(0x7fffffff);
        // K, then V: a row (or two) of this lane's in each.  One small loop body: unrolled, the four groups' places in the code evict one another
        // from the instruction cache (8192-token prompt: 1098 us)
#pragma unroll 1
        for (int which = 0; which < 2; ++which) {
          guarded(bar((which ? kVEmpty : kKEmpty) + slot), phase ^ 1);
          const uint8_t* const codes = raw + which * SH::CODE_BYTES;
          uint8_t* const dst = smem + (which ? SH::OFF_V : SH::OFF_K) + slot * SH::KV_BYTES;
          // two warps share a chunk: 32 of its 64 rows each, or half of the channels of its 32
          constexpr bool BY_ROWS = GROUP == 2 && HALVES == 2, BY_PIECES = GROUP == 2 && HALVES == 1;
#pragma unroll 1
          for (int h = BY_ROWS ? warp & 1 : 0; h < (BY_ROWS ? (warp & 1) + 1 : HALVES); ++h) {
            const int row = lane + 32 * h, L = HALVES - 1;
            const bool here = h ? there[L] : there[0], good = (h ? v_good[L] : v_good[0]) && (which || (h ? k_good[L] : k_good[0]));
            const float2 par = which ? (h ? v[L] : v[0]) : (h ? k[L] : k[0]);
            const float by = which ? fv : fk, bad = which ? 0.0f : nan;
            const __half2 s = __float2half2_rn(!here ? 0.0f : good ? par.x * by : bad), m = __float2half2_rn(!here ? 0.0f : good ? par.y * by : bad);
            const int turn = D == 64 ? row >> 2 : D == 128 ? row >> 1 : row;       // which piece first: spreads the rows over the banks
            const uint8_t* const src = codes + row * (D / 2);
            uint8_t* const lines = dst + row * 128;
            constexpr int MINE = BY_PIECES ? PIECES / 2 : PIECES;
            const int from = BY_PIECES ? (warp & 1) * MINE : 0;
            uint4 x = *reinterpret_cast<const uint4*>(src + (from + turn % MINE) * 16);
#pragma unroll 1
            for (int e = 0; e < MINE; ++e) {
              const int piece = from + (turn + e) % MINE;
              const uint4 following = *reinterpret_cast<const uint4*>(src + (from + (turn + e + 1) % MINE) * 16);
              uint8_t* const line = lines + (piece >> 1) * (BN * 128);
              const int first = (piece & 1) * 4, swizzle = row & 7;
              auto put = [&](int at, uint32_t codes8) {
                uint8_t* const to = line + ((at ^ swizzle) << 4);
                if constexpr (SH::PARTS == 2) {
                  uint4 low;
                  *reinterpret_cast<uint4*>(to) = eight(codes8, s, m, low);
                  *reinterpret_cast<uint4*>(to + SH::PART_BYTES) = low;
                } else {
                  *reinterpret_cast<uint4*>(to) = eight(codes8, s, m);
                }
              };
              put(first + 0, x.x);
              put(first + 1, x.y);
              put(first + 2, x.z);
              put(first + 3, x.w);
              x = following;
            }
          }
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar((which ? kVReady : kKReady) + slot));
        }
        if (lane == 0) mbar_arrive(bar(kRawEmpty + slot));
      }
    });
  } else if (warp >= 8) {
    // ------------------------------------------------------------ softmax: a thread per row
    const int tile = (warp - 8) >> 2, quarter = warp & 3, line = quarter * 32 + lane;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const uint32_t s_tile = tmem + lanes + 2 * tile * BN, o_at = tmem + lanes + SH::O_COL + tile * D;
    // a finished run whose O is still in tensor memory: it is written when the queries of the next one are on their way
    T* out = nullptr;
    float* part = nullptr;
    float out_by = 0.0f, out_keep = 0.0f;
    int out_n = -1, out_how = kResult;
    auto flush = [&]() {
      if (out_n < 0) return;
      guarded(bar(kODone + 2 * tile + (out_n & 1)), out_n >> 1 & 1);
      tc_fence_after();
      store_rows<T, D>(o_at, reinterpret_cast<unsigned long long>(part), reinterpret_cast<unsigned long long>(out), out_by, out_keep, out_how);
    };
    float factor = 0.0f;                             // what the row's scores are multiplied by
    runs([&](const PromptItem& w, const Run& run) {
      const int lo = run.lo, hi = run.hi, before = run.before;
      const int row = w.tile * SH::ROWS + tile * 128 + line;
      const bool real = row < w.s.nq * a.each;
      const int j = real ? row / a.each : 0, head = w.head * a.each + (real ? row - j * a.each : 0);
      const int hi_key = real ? w.s.len - w.s.nq + j : -1, from = a.window ? (int)max((long long)w.s.len - w.s.nq + j - a.window + 1, 0LL) : 0;
      const int n_end = before + hi - lo;
      float m = kLowest;
      Two l(0.0f);
      if (hi > lo && run.first) {
        const T* const src = real ? reinterpret_cast<const T*>(a.q) + (long long)(w.s.q0 + j) * a.q_token + (long long)head * a.q_head : nullptr;
        factor = load_queries<T, D>(src, smem + tile * (BLOCKS * 128 * 128) + quarter * 32 * 128, a.scale);
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kQReady + tile));
      }
      flush();
      out = nullptr;                                 // none of it is held while the chunks need the registers
      part = nullptr;
      out_by = out_keep = 0.0f;
      out_n = -1;
      out_how = kResult;
      bool s_ready = false;
      for (int n = before; n < n_end; ++n) {
        if (!s_ready) guarded(bar(kSFull + 2 * tile + (n & 1)), n >> 1 & 1);
        tc_fence_after();
        const uint32_t s_at = s_tile + (n & 1) * BN;
        const int t0 = w.begin + (lo + n - before) * BN;
        const float f = fminf(fmaxf(factor * s_key[n % kRing], 7.5e-37f), 1.3e30f), ratio = s_value[n % kRing];
        const uint32_t there = s_mask[n % kRing];
        const bool all = there == (1u << BN / 16) - 1 && t0 + BN - 1 <= hi_key && t0 >= from;
        const bool masked = __any_sync(0xffffffffu, !all);
        // which of the 32 keys from t on this row sees
        auto visible = [&](int h) {
          const int t = t0 + 32 * h;
          uint32_t bits = 0xffffffffu;
          if (hi_key < t + 31) bits = hi_key < t ? 0u : 0xffffffffu >> (t + 31 - hi_key);
          if (from > t) bits = from > t + 31 ? 0u : bits & 0xffffffffu << (from - t);
          const uint32_t two = there >> (2 * h);
          return bits & ((two & 1u ? 0xffffu : 0u) | (two & 2u ? 0xffff0000u : 0u));
        };
        auto hide = [&](uint32_t (&r)[32], int h) {
          const uint32_t bits = visible(h);
#pragma unroll
          for (int e = 0; e < 32; ++e) r[e] = bits >> e & 1u ? r[e] : 0xff800000u;
        };
        auto largest = [](const uint32_t (&r)[32]) {
          float x = __uint_as_float(r[0]), y = __uint_as_float(r[1]);
#pragma unroll
          for (int e = 2; e < 32; e += 2) {
            x = fmaxf(x, __uint_as_float(r[e]));
            y = fmaxf(y, __uint_as_float(r[e + 1]));
          }
          return fmaxf(x, y);
        };
        uint32_t ra[32], rb[32];
        tmem_ld_32x32(s_at, ra);
        if constexpr (BN == 64) tmem_ld_32x32(s_at + 32, rb);
        wait_ld_dep32(ra);
        if constexpr (BN == 64) wait_ld_dep32(rb);
        if (masked) {
          hide(ra, 0);
          if constexpr (BN == 64) hide(rb, 1);
        }
        float top = largest(ra);
        if constexpr (BN == 64) top = fmaxf(top, largest(rb));
        top *= f;
        const bool moves = top > m + 8.0f || (m == kLowest && top > kLowest);
        if (__any_sync(0xffffffffu, moves) || ratio != 1.0f) {
          const float next = fmaxf(m, top);
          const float alpha = m == next ? 1.0f : exp2_fast(m - next);
          m = next;
          l = l * Two(alpha);
          if (n > before) {
            guarded(bar(kODone + 2 * tile + (n - 1 & 1)), n - 1 >> 1 & 1);       // the product before has to be in O
            tc_fence_after();
            const Two by(alpha * ratio);
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              uint32_t r[32];
              tmem_ld_32x32(o_at + 32 * c, r);
              wait_ld_dep32(r);
#pragma unroll
              for (int e = 0; e < 32; e += 2) {
                const float2 v = (Two(__uint_as_float(r[e]), __uint_as_float(r[e + 1])) * by).both();
                r[e] = __float_as_uint(v.x);
                r[e + 1] = __float_as_uint(v.y);
              }
              tmem_st_32x32(o_at + 32 * c, r);
            }
          }
        }
        const Two f2(f), minus(m == kLowest ? 0.0f : kLift - m);
        auto weigh = [&](const uint32_t (&r)[32], int at) {
          uint32_t h[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float2 x = fma2(Two(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1])), f2, minus).both();
            const float2 p = make_float2(exp2_fast(x.x), exp2_fast(x.y));
            l = l + Two(p.x, p.y);
            h[e] = half2_bits(__floats2half2_rn(p.x, p.y));
          }
          tmem_st_32x16(s_at + 16 * at, h);             // over the scores, which are all in registers
        };
        weigh(ra, 0);
        s_ready = n + 1 < n_end && mbar_test_wait(bar(kSFull + 2 * tile + (n + 1 & 1)), n + 1 >> 1 & 1);
        if constexpr (BN == 64) weigh(rb, 1);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kPReady + 2 * tile + (n & 1)));
      }
      const float2 sums = l.both();
      // Parts stand relative to the first run's maximum, or to a later one's that is above it by 2^8; less 2^15, so that they are no larger than sums of
      // values.  A whole item of several runs is summed where the part of an item that ends in another CTA will stand.
      const long long slot_row = (long long)(2 * blockIdx.x + (run.opens ? 1 : 0)) * SH::ROWS + tile * 128 + line;
      const float2 past = run.first || !real ? make_float2(kLowest, 0.0f) : a.part_ml[slot_row];
      const bool moves = past.x == kLowest || m > past.x + 8.0f;
      const float top = moves ? fmaxf(past.x, m) : past.x, keep = past.x == top ? 1.0f : exp2_fast(past.x - top);
      const float by = (m == top ? 1.0f : exp2_fast(m - top)) * 0x1p-15f, weight = fmaf(past.y, keep, (sums.x + sums.y) * by);
      T* const row_out = real ? reinterpret_cast<T*>(a.out) + ((long long)(w.s.q0 + j) * a.q_heads + head) * D : nullptr;
      if (!(run.whole && run.last) && real) a.part_ml[slot_row] = make_float2(top, weight);
      if (hi > lo) {
        const float scale = s_scale[(n_end - 1) % kRing] * by;
        out_n = n_end - 1;
        out = row_out;
        part = real ? a.part_o + slot_row * D : nullptr;
        const bool result = run.whole && run.last, scaled = __any_sync(0xffffffffu, keep != 1.0f);
        out_how = run.first ? (result ? kResult : kPart) : result ? kSum : scaled ? kScaled : kAdded;
        out_by = !result ? scale : weight == 0.0f ? 0.0f : scale / weight;
        out_keep = !result ? keep : weight == 0.0f ? 0.0f : keep / weight;
      } else if (run.whole && real) {                // no keys at all
        for (int c = 0; c < D / 8; ++c) reinterpret_cast<uint4*>(row_out)[c] = make_uint4(0, 0, 0, 0);
      }
    });
    flush();
  }
  tc_fence_before();
  __syncthreads();
  if (*s_abort != 0u) {                              // (here, behind all roles: inside them it moves their code, and the 8192-token prompt takes 676 us)
    if (warp == 0) {                                 // (a stage that was never filled counts as done)
      for (int s = 0; s < SH::STAGES; ++s) mbar_wait(bar(kRawFull + s), s < mine >> 1 ? mine & 1 : ~mine & 1);
    } else if (mine > 0) {                           // the last product, and so those before it
      mbar_spin(bar(kODone + 2 * (warp >> 1) + (mine - 1 & 1)), mine - 1 >> 1 & 1);
    }
    tc_fence_before();
    __syncthreads();
  }
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the items that a boundary between two CTAs runs through: block x for boundary x + 1, if it is the first in its item; a row per warp.
template <typename T, typename SH>
__global__ void __launch_bounds__(256) kv4_prompt_join_kernel(const AttnArgs a, unsigned ctas) {
  constexpr int D = SH::D, PER = D / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  grid_launch_dependents();
  grid_dependency_wait();
  const int4 p = a.plan[blockIdx.x + 1], w = a.plan[ctas + blockIdx.x + 1];       // total, unit, units, head | sequence, tile, first query, queries
  if (p.y == 0) return;
  Deal d;
  d.total = (unsigned)p.x;
  d.each = d.total / ctas;
  d.more = d.total - d.each * ctas;
  const unsigned u0 = d.start(blockIdx.x + 1) - (unsigned)p.y;                    // the item's first unit
  const unsigned i0 = d.owner(u0), i1 = d.owner(u0 + (unsigned)p.z - 1);
  if (i0 != blockIdx.x) return;
  {
    const int line = blockIdx.y * 8 + warp, row = w.y * SH::ROWS + line, j = row / a.each;
    if (j >= w.w) return;
    float m = -CUDART_INF_F, weight = 0.0f, sum[PER];
#pragma unroll
    for (int e = 0; e < PER; ++e) sum[e] = 0.0f;
    join_parts<D>(a, SH::ROWS, line, (int)i0, (int)i1, 1, d, u0, m, weight, sum);
    const float inv = weight == 0.0f ? 0.0f : 1.0f / weight;
    T* const out = reinterpret_cast<T*>(a.out) + ((long long)(w.z + j) * a.q_heads + p.w * a.each + row - j * a.each) * D + lane * PER;
#pragma unroll
    for (int e = 0; e < PER; ++e) out[e] = from_float<T>(sum[e] * inv);
  }
}

// CTAs, and the bytes behind each other in the workspace: sums, their maxima and weights, the CTAs' beginnings
template <typename SH>
long long prompt_units(const AttnArgs& a) {
  const long long items = ((long long)a.tokens * a.each / SH::ROWS + a.batch) * a.kv_heads;
  return items * (((long long)a.table_width << a.page_shift) / SH::BN + 1 + SH::OPENING);
}
size_t prompt_bytes(int ctas, int rows, int dim) { return (size_t)2 * ctas * rows * (dim * 4 + 8) + (size_t)2 * ctas * 16; }

template <typename T, int D, int TILES, int STAGES, int PARTS, int BN = 64>
int run(AttnArgs a, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  using SH = PromptShape<D, TILES, STAGES, PARTS, BN>;
  const long long units = prompt_units<SH>(a);
  XQT_REQUIRE(units < (1LL << 31));
  const int ctas = (int)min((long long)sm_count(), units);
  XQT_REQUIRE(workspace && workspace_bytes >= prompt_bytes(ctas, SH::ROWS, D) && ((uintptr_t)workspace & 15) == 0);
  a.part_o = reinterpret_cast<float*>(workspace);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + (size_t)2 * ctas * SH::ROWS * D);
  a.plan = reinterpret_cast<int4*>(a.part_ml + (size_t)2 * ctas * SH::ROWS);
  XQT_SMEM_OPT_IN((kv4_prompt_kernel<T, SH>), SH::SMEM);
  const int rc = launch_pdl(kv4_prompt_kernel<T, SH>, dim3((unsigned)ctas), dim3(SH::THREADS), SH::SMEM, stream, a);
  if (rc || ctas == 1) return rc;
  return launch_pdl(kv4_prompt_join_kernel<T, SH>, dim3((unsigned)ctas - 1, SH::ROWS / 8), dim3(256), 0, stream, a, (unsigned)ctas);
}

template <typename T>
int run_dim(const AttnArgs& a, int dim, void* workspace, size_t bytes, cudaStream_t stream) {
  // (see above: fp16 results are held to more than one fp16 rounding each of keys, values and P would leave)
  constexpr int PARTS = std::is_same<T, __half>::value ? 2 : 1;
  if (dim == 64) return run<T, 64, 2, 4, PARTS>(a, workspace, bytes, stream);
  if (dim == 128) return run<T, 128, 2, PARTS == 2 ? 2 : 4, PARTS>(a, workspace, bytes, stream);
  return run<T, 256, 1, 2, PARTS, PARTS == 2 ? 32 : 64>(a, workspace, bytes, stream);
}

}  // namespace

int kv4_prompt_launch(const kv4::AttnArgs& a, int dim, int dtype, void* workspace, size_t bytes, cudaStream_t stream) {
  return dtype == XQT_B200_BF16 ? run_dim<__nv_bfloat16>(a, dim, workspace, bytes, stream) : run_dim<__half>(a, dim, workspace, bytes, stream);
}

size_t kv4_prompt_workspace_bytes(int dim) { return prompt_bytes(sm_count(), dim == 256 ? 128 : 256, dim); }

}  // namespace xqt_b200
