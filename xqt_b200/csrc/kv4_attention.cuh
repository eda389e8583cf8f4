// What the two attention kernels over the 4-bit cache share: their arguments, and the list of the work in a batch whose lengths only the
// device knows.
#pragma once

#include <limits.h>
#include <math_constants.h>

#include <type_traits>

#include "pairs.cuh"

namespace xqt_b200 {
namespace kv4 {

using namespace sm100;

struct AttnArgs {
  const void* q;
  const uint8_t* codes;
  const uint8_t* params;
  const int* table;
  const int* seq_lens;
  const int* query_starts;   // null: one query per sequence
  void* out;
  float* part_o;             // [2 * CTAs][ROWS][D]
  float2* part_ml;           // [2 * CTAs][ROWS]
  int4* plan;                // [2 * CTAs] where each CTA begins
  unsigned* status;
  long long q_token, q_head, pages, table_stride;
  int tokens, batch, q_heads, kv_heads, each, page_size, page_shift, table_width, window, few_rows;     // few_rows: sequences with more rows for a key head go to the prompt kernel
  float scale;               // times log2(e)
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ float2 pair_of(uint32_t bits) {
  const T* e = reinterpret_cast<const T*>(&bits);
  return make_float2(to_float<T>(e[0]), to_float<T>(e[1]));
}

// A list's shape L: ROWS of a row tile, UNIT keys of a unit (OPENING units in front of every item have no keys), CT to which an item's first
// key is rounded down; PROMPT: the sequences with more than few_rows rows, else those with no more.

// A sequence as the work list sees it.
struct Sequence {
  int q0, nq, len, first, tiles, units;   // `first`: where its units start; units per (tile, head) item
};

template <typename L>
__device__ __forceinline__ Sequence sequence(const AttnArgs& a, int b) {
  Sequence s;
  if (a.query_starts) {
    const int lo = min(max(a.query_starts[b], 0), a.tokens);
    s.q0 = lo;
    s.nq = min(max(a.query_starts[b + 1], lo), a.tokens) - lo;
  } else {
    s.q0 = b;
    s.nq = 1;
  }
  const long long most = (long long)a.table_width << a.page_shift;
  s.len = (int)min((long long)max(a.seq_lens[b], 0), most);
  const long long from = a.window ? (long long)s.len - s.nq + 1 - a.window : 0;
  s.first = from > 0 ? (int)(from / L::CT * L::CT) : 0;
  const long long rows = (long long)s.nq * a.each;
  s.tiles = (L::PROMPT ? rows <= a.few_rows : rows > a.few_rows) ? 0 : (int)((rows + L::ROWS - 1) / L::ROWS);
  s.units = max((s.len - s.first + L::UNIT - 1) / L::UNIT, 0) + L::OPENING;   // an empty sequence still has its rows written
  return s;
}

// A place in the work list.
struct Walk {
  int b, tile, head, unit;
  Sequence s;
};

// The list: its units are dealt out in equal contiguous runs, the first `more` CTAs one unit longer.  32 bits: the host refuses more.
struct Deal {
  unsigned total, each, more;
  __device__ __forceinline__ unsigned start(unsigned i) const { return each * i + min(i, more); }
  __device__ __forceinline__ unsigned owner(unsigned u) const {
    const unsigned long_run = more * (each + 1);
    return u < long_run ? u / (each + 1) : more + (u - long_run) / max(each, 1u);
  }
};

__device__ __forceinline__ unsigned scan32(unsigned v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += x;
  }
  return v;
}

template <typename L>
__device__ __forceinline__ Deal deal(const AttnArgs& a, int lane, unsigned ctas, Sequence& mine) {
  Deal d = {};
  for (int b0 = (a.batch - 1) & ~31; b0 >= 0; b0 -= 32) {      // backwards: `mine` ends as sequence `lane`
    unsigned units = 0;
    if (b0 + lane < a.batch) {
      mine = sequence<L>(a, b0 + lane);
      units = (unsigned)mine.tiles * a.kv_heads * mine.units;
    }
    d.total += __reduce_add_sync(0xffffffffu, units);
  }
  d.each = d.total / ctas;
  d.more = d.total - d.each * ctas;
  return d;
}

// the sequence that lane `lane` has
__device__ __forceinline__ Sequence sequence_of(const Sequence& s, int lane) {
  Sequence r;
  r.q0 = __shfl_sync(0xffffffffu, s.q0, lane);
  r.nq = __shfl_sync(0xffffffffu, s.nq, lane);
  r.len = __shfl_sync(0xffffffffu, s.len, lane);
  r.first = __shfl_sync(0xffffffffu, s.first, lane);
  r.tiles = __shfl_sync(0xffffffffu, s.tiles, lane);
  r.units = __shfl_sync(0xffffffffu, s.units, lane);
  return r;
}

// The place of unit `u`.
template <typename L>
__device__ __forceinline__ bool place(const AttnArgs& a, int lane, const Sequence& mine, unsigned u, Walk& w) {
  unsigned base = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 32) {
    Sequence s = mine;
    unsigned units = 0;
    if (b0 + lane < a.batch) {
      if (b0 > 0) s = sequence<L>(a, b0 + lane);
      units = (unsigned)s.tiles * a.kv_heads * s.units;
    }
    const unsigned cum = scan32(units, lane);
    const unsigned over = __ballot_sync(0xffffffffu, base + cum > u);
    if (over) {
      const int at = __ffs(over) - 1;
      const unsigned rest = u - base - __shfl_sync(0xffffffffu, cum - units, at);
      w.b = b0 + at;
      w.s = sequence_of(s, at);
      const unsigned item = rest / (unsigned)w.s.units;
      w.unit = (int)(rest - item * w.s.units);
      w.tile = (int)(item / (unsigned)a.kv_heads);
      w.head = (int)(item - (unsigned)w.tile * a.kv_heads);
      return true;
    }
    base += __shfl_sync(0xffffffffu, cum, 31);
  }
  return false;
}

// Item (tile, head) number `item` of the list.
template <typename L>
__device__ __forceinline__ bool place_item(const AttnArgs& a, int lane, unsigned item, Walk& w) {
  if (!a.query_starts) {                             // the same number of items in each sequence
    const unsigned tiles = (unsigned)(a.each + L::ROWS - 1) / L::ROWS, of_sequence = item / (unsigned)a.kv_heads;
    w.head = (int)(item - of_sequence * a.kv_heads);
    w.b = (int)(of_sequence / tiles);
    w.tile = (int)(of_sequence - w.b * tiles);
    w.s = sequence<L>(a, w.b);
    return true;
  }
  unsigned base = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 32) {
    Sequence s = {};
    if (b0 + lane < a.batch) s = sequence<L>(a, b0 + lane);
    const unsigned items = (unsigned)s.tiles * a.kv_heads, cum = scan32(items, lane);
    const unsigned over = __ballot_sync(0xffffffffu, base + cum > item);
    if (over) {
      const int at = __ffs(over) - 1;
      const unsigned rest = item - base - __shfl_sync(0xffffffffu, cum - items, at);
      w.b = b0 + at;
      w.s = sequence_of(s, at);
      w.tile = (int)(rest / (unsigned)a.kv_heads);
      w.head = (int)(rest - (unsigned)w.tile * a.kv_heads);
      return true;
    }
    base += __shfl_sync(0xffffffffu, cum, 31);
  }
  return false;
}

// Adds up row `row` of the parts of an item (first unit u0) that CTAs first, first + step, .. last hold, for the lane's D / 32 channels, four parts
// in flight.  A part that saw nothing has weight 0, and its sums were never written.
template <int D>
__device__ __forceinline__ void join_parts(const AttnArgs& a, int rows, int row, int first, int last, int step, const Deal& d, unsigned u0, float& m, float& weight,
                                           float (&sum)[D / 32]) {
  constexpr int PER = D / 32;
  const int lane = threadIdx.x & 31;
  for (int i = first; i <= last; i += 4 * step) {
    float2 s[4];
    float v[4][PER];
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const int cta = i + b * step;
      s[b] = make_float2(-CUDART_INF_F, 0.0f);
      if (cta <= last) {
        const long long at = (2LL * cta + (d.start(cta) > u0 ? 0 : 1)) * rows + row;
        s[b] = a.part_ml[at];
#pragma unroll
        for (int e = 0; e < PER; e += 2) *reinterpret_cast<float2*>(&v[b][e]) = *reinterpret_cast<const float2*>(a.part_o + at * D + lane * PER + e);
      }
    }
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      if (s[b].y == 0.0f) continue;                  // (a NaN has no maximum, but a weight)
      const float top = fmaxf(m, s[b].x), keep = m == top ? 1.0f : exp2_fast(m - top), by = exp2_fast(s[b].x - top);
      m = top;
      weight = fmaf(s[b].y, by, weight * keep);
#pragma unroll
      for (int e = 0; e < PER; ++e) sum[e] = fmaf(v[b][e], by, sum[e] * keep);
    }
  }
}

}  // namespace kv4

int kv4_prompt_launch(const kv4::AttnArgs& a, int dim, int dtype, void* workspace, size_t bytes, cudaStream_t stream);
size_t kv4_prompt_workspace_bytes(int dim);

}  // namespace xqt_b200
