// bq.cuh — block-quantised rows: the arithmetic of the codes and scales, and the walk over the
// output tiles of a dense or grouped product.
//
// A block of 128 components with largest finite magnitude t has the scale 2^s, s the smallest
// exponent >= -126 with t <= 448 * 2^s, kept as the byte s + 127 (E8M0). 448 = 1.75 * 2^8 is the
// largest e4m3 value, so for t = 1.f * 2^(E - 127) the byte is E - 8, one more when 1.f > 1.75:
// an integer rule on t's bits. Scaling by a power of two is exact, so a code carries one
// rounding, that to e4m3.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "bq_reports.cuh"
#include "common.cuh"

namespace pxc {
namespace bq {

constexpr uint32_t BLOCK = 128;  // components per scale

// A failure that only the device sees, into the caller's record.
__device__ __forceinline__ void leave_fault(const Record& r, Fault which) {
  *reinterpret_cast<volatile uint32_t*>(r.words + which) = r.id;
  __threadfence_system();
}

// ---- one block's scale ----
// `top` holds the bits of the largest finite magnitude. Bytes are 1..247 (127 for top == 0), so
// both 2^s and 2^-s are normal floats.
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
  if (top == 0) return 127u;
  const int32_t e = static_cast<int32_t>(top >> 23) - 8 + ((top & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return static_cast<uint32_t>(max(e, 1));
}
__device__ __forceinline__ float inverse_scale(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }
// 2^(byte - 127) for any E8M0 byte: 0 is the subnormal 2^-127, 255 is NaN.
__device__ __forceinline__ float scale_value(uint32_t byte) {
  if (byte == 0) return __uint_as_float(0x00400000u);
  return byte == 255u ? __uint_as_float(0x7FC00000u) : __uint_as_float(byte << 23);
}
// Magnitude bits of a finite value, 0 for an infinity or NaN.
__device__ __forceinline__ uint32_t finite_bits(float x) {
  const uint32_t b = __float_as_uint(x) & 0x7FFFFFFFu;
  return b < 0x7F800000u ? b : 0u;
}

// Four values to four e4m3 codes, the first in the lowest byte: nearest, ties to even,
// magnitudes above 448 (only infinities, after scaling) to 448, NaN to NaN.
__device__ __forceinline__ uint32_t to_codes(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
// Two codes to f32: every e4m3 value is a half.
__device__ __forceinline__ float2 from_codes(uint32_t two) {
  return __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two), __NV_E4M3)));
}

template <class T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// ---- the tiles of a product ----
// A dense product is one group over all rows. Query offsets and base offsets are read where given
// (`groups` + 1 each); without base offsets every group has n_each rows and the output is
// indexed by query, else the groups' matrices follow one another.
struct Groups {
  const int64_t* q_offsets;  // NULL: dense, one group
  const int64_t* b_offsets;  // NULL: even (or dense)
  uint32_t groups;
  uint64_t nq, nb;      // rows on either side
  uint64_t n_each;      // even (and dense): base rows per group, and the output's row pitch is `stride`
  uint64_t stride;
  uint64_t size;        // room in the output, in values (ragged)
  Record record;        // for failures
};

// One output tile: `queries` x `rows` values from (q0, b0), the first at out[at].
struct Tile {
  uint32_t q0, queries, b0, rows;
  uint64_t at, stride;
};

// Walks the tiles in order, a warp at a time: a chunk of 128 groups, four to a lane. Tiles are numbered
// through the groups; find() is called with rising numbers, so that each chunk is read once, and the next
// one's offsets are on their way meanwhile. Short groups come at one a tile and more, so what a chunk and a
// group cost counts: 32-bit scans and shuffles wherever the numbers allow, and no division for a
// group of one tile of queries.
//
// Inside a group the base rows come in panels of PANEL tiles, all queries against one panel before the
// next: neighbouring CTAs write neighbouring columns of the same output rows, and a panel's rows stay in
// L2 while the queries pass.
//
// Every group is checked before it counts: its offsets rise and lie within the rows, and its
// matrix ends within the output. One that fails leaves a fault, and it and all groups behind it count as
// empty. So no offsets lead to an access out of range, the groups that count are disjoint in rows and outputs, and
// the number of tiles is at most that of output values.
struct Walk {
  static constexpr uint32_t PANEL = 64, PER = 4, CHUNK = 32 * PER;
  const Groups& g;
  const uint32_t lane;
  const uint32_t TQ, tb_log2;  // the most queries of a tile; its base rows are a power of two
  uint32_t chunk = 0;
  uint64_t tiles_before = 0, values_before = 0;  // of earlier chunks
  uint64_t tiles_upto = 0, values_upto = 0;      // of this one, up to and with this lane's groups
  bool stopped = false;                          // at a group whose offsets are no good
  // this lane's groups: first rows, sizes, tiles and output values
  uint32_t q0[PER], b0[PER], m[PER], n[PER];
  uint64_t tiles[PER], values[PER];
  // the group found last, in every lane: its tiles are [first, last)
  uint64_t first = 0, last = 0, first_value = 0;
  uint32_t gq = 0, gb = 0, gm = 0, gn = 0;
  uint32_t qt = 0, bt = 0, width = 0;

  __device__ __forceinline__ Walk(const Groups& groups, uint32_t lane_id, uint32_t queries, uint32_t rows_log2)
      : g(groups), lane(lane_id), TQ(queries), tb_log2(rows_log2) {}

  // Reads the first chunk; before find().
  __device__ __forceinline__ void start() {
    if (g.q_offsets) {
      fetch(0);
      load();
    } else {  // dense: one group of everything
      chunk = g.groups;
      gm = static_cast<uint32_t>(g.nq), gn = static_cast<uint32_t>(g.nb);
      split();
    }
  }

  // The group's tiles from `first` on: an even split of its queries in steps of 16 (at most TQ, so that no tile is
  // empty).
  __device__ __forceinline__ void split() {
    qt = query_tiles(gm), bt = base_tiles(gn);
    width = ((qt == 1 ? gm : (gm + qt - 1) / qt) + 15) / 16 * 16;
    last = first + static_cast<uint64_t>(qt) * bt;
  }

  // The offsets around this lane's groups of the chunk from group `from` on; behind the last group, its end.
  int64_t q_next[PER + 1], b_next[PER + 1];
  __device__ __forceinline__ void fetch(uint64_t from) {
#pragma unroll
    for (uint32_t j = 0; j <= PER; ++j) {
      const uint64_t i = min(from + lane * PER + j, static_cast<uint64_t>(g.groups));
      q_next[j] = __ldg(g.q_offsets + i);
      b_next[j] = g.b_offsets ? __ldg(g.b_offsets + i) : 0;
    }
  }

  template <class U>
  __device__ __forceinline__ static U scan_as(U v, uint32_t lane) {
#pragma unroll
    for (uint32_t d = 1; d < 32; d <<= 1) {
      const U u = __shfl_up_sync(0xFFFFFFFFu, v, d);
      if (lane >= d) v += u;
    }
    return v;
  }
  __device__ __forceinline__ uint64_t scan(uint64_t v) const {
    if (__any_sync(0xFFFFFFFFu, v >> 26 != 0)) return scan_as<uint64_t>(v, lane);
    return scan_as<uint32_t>(static_cast<uint32_t>(v), lane);
  }
  __device__ __forceinline__ uint32_t query_tiles(uint32_t queries) const {
    return queries <= TQ ? (queries != 0) : (queries + TQ - 1) / TQ;
  }
  __device__ __forceinline__ uint32_t base_tiles(uint32_t rows) const {
    return (rows + (1u << tb_log2) - 1) >> tb_log2;
  }
  __device__ __forceinline__ static bool within(int64_t lo, int64_t hi, uint64_t rows) {
    return lo >= 0 && hi >= lo && hi <= static_cast<int64_t>(rows);
  }

  __device__ __forceinline__ void load() {
    bool bad = false;  // a group of this lane, or one before
    uint64_t value_sum = 0, tile_sum = 0;
#pragma unroll
    for (uint32_t j = 0; j < PER; ++j) {
      const uint64_t i = static_cast<uint64_t>(chunk) + lane * PER + j;
      const bool there = i < g.groups;
      q0[j] = static_cast<uint32_t>(q_next[j]);
      m[j] = static_cast<uint32_t>(q_next[j + 1]) - q0[j];
      b0[j] = g.b_offsets ? static_cast<uint32_t>(b_next[j]) : static_cast<uint32_t>(i * g.n_each);
      n[j] = g.b_offsets ? static_cast<uint32_t>(b_next[j + 1]) - b0[j] : there ? static_cast<uint32_t>(g.n_each) : 0u;
      const bool good =
          within(q_next[j], q_next[j + 1], g.nq) && (!g.b_offsets || within(b_next[j], b_next[j + 1], g.nb));
      bad = bad || (there && !good);
      if (bad || !good) m[j] = n[j] = 0;
    }
    const uint32_t bad_lanes = __ballot_sync(0xFFFFFFFFu, bad);
    if (bad_lanes != 0) leave_fault(g.record, FAULT_OFFSETS);
    const bool behind = stopped || (bad_lanes & ((1u << lane) - 1)) != 0;
    stopped = stopped || bad_lanes != 0;
#pragma unroll
    for (uint32_t j = 0; j < PER; ++j) {
      if (behind) m[j] = n[j] = 0;
      // m, n < 2^31 and size <= 2^48: with each term held to size + 1 no sum overflows, and one that is past the
      // room stays past it for all groups behind
      values[j] = g.b_offsets ? min(static_cast<uint64_t>(m[j]) * n[j], g.size + 1) : 0;
      value_sum += values[j];
    }
    if (g.b_offsets) {
      values_upto = scan(value_sum);
      uint64_t upto = values_before + values_upto - value_sum;
      bool past = false;
#pragma unroll
      for (uint32_t j = 0; j < PER; ++j) {
        upto += values[j];
        if (values[j] != 0 && upto > g.size) past = true, m[j] = 0;
      }
      if (past) leave_fault(g.record, FAULT_OFFSETS);
    }
#pragma unroll
    for (uint32_t j = 0; j < PER; ++j) {
      tiles[j] = static_cast<uint64_t>(query_tiles(m[j])) * base_tiles(n[j]);
      tile_sum += tiles[j];
    }
    tiles_upto = scan(tile_sum);
    if (g.groups - chunk > CHUNK) fetch(static_cast<uint64_t>(chunk) + CHUNK);
  }

  // Tile number t, or false when there are fewer. All lanes call and get the same answer.
  __device__ __forceinline__ bool find(uint64_t t, Tile& out) {
    if (t >= last && !enter(t)) return false;
    const uint64_t r = t - first;
    uint32_t qi, bi;
    if (qt == 1) {
      qi = 0, bi = static_cast<uint32_t>(r);
    } else if (last - first <= 0xFFFFFFFFu) {
      const uint32_t r32 = static_cast<uint32_t>(r);
      // at most 2^32 / bt tiles of queries, so a panel's PANEL * qt tiles fit 32 bits whenever bt >= PANEL
      const uint32_t panel = bt <= PANEL ? 0 : r32 / (PANEL * qt);
      const uint32_t in_panel = r32 - panel * PANEL * qt;
      const uint32_t across = min(PANEL, bt - panel * PANEL);
      qi = in_panel / across;
      bi = panel * PANEL + in_panel - qi * across;
    } else {
      const uint32_t panel = static_cast<uint32_t>(r / (static_cast<uint64_t>(PANEL) * qt));
      const uint64_t in_panel = r - static_cast<uint64_t>(panel) * PANEL * qt;
      const uint32_t across = min(PANEL, bt - panel * PANEL);
      qi = static_cast<uint32_t>(in_panel / across);
      bi = panel * PANEL + static_cast<uint32_t>(in_panel - static_cast<uint64_t>(qi) * across);
    }
    const uint32_t qa = qi * width, ba = bi << tb_log2;  // below gm and gn
    out.q0 = gq + qa;
    out.queries = min(width, gm - qa);
    out.b0 = gb + ba;
    out.rows = min(1u << tb_log2, gn - ba);
    if (g.b_offsets) {
      out.stride = gn;
      out.at = first_value + static_cast<uint64_t>(qa) * gn + ba;
    } else {
      out.stride = g.stride;
      out.at = static_cast<uint64_t>(gq + qa) * g.stride + ba;
    }
    return true;
  }

  // Goes on to the group that holds tile t.
  __device__ __forceinline__ bool enter(uint64_t t) {
    for (;;) {
      const uint64_t total = __shfl_sync(0xFFFFFFFFu, tiles_upto, 31);
      if (t < tiles_before + total) break;
      tiles_before += total;
      values_before = min(values_before + __shfl_sync(0xFFFFFFFFu, values_upto, 31), uint64_t(1) << 60);
      if (stopped || g.groups - chunk <= CHUNK) {
        chunk = g.groups;  // nothing behind: later calls find nothing either
        tiles_upto = values_upto = 0;
        return false;
      }
      chunk += CHUNK;
      load();
    }
    // the first lane whose groups reach beyond t has it; which of its groups, every lane works out for its own
    const uint32_t who = __ffs(__ballot_sync(0xFFFFFFFFu, t < tiles_before + tiles_upto)) - 1;
    uint64_t start = tiles_before + tiles_upto, value = values_before + values_upto;
#pragma unroll
    for (uint32_t j = 0; j < PER; ++j) start -= tiles[j], value -= values[j];
    uint32_t sq = q0[0], sb = b0[0], sm = m[0], sn = n[0];
#pragma unroll
    for (uint32_t j = 1; j < PER; ++j) {
      if (t >= start + tiles[j - 1]) {
        sq = q0[j], sb = b0[j], sm = m[j], sn = n[j];
        start += tiles[j - 1], value += values[j - 1];
      } else {
        break;
      }
    }
    gm = __shfl_sync(0xFFFFFFFFu, sm, who), gn = __shfl_sync(0xFFFFFFFFu, sn, who);
    gq = __shfl_sync(0xFFFFFFFFu, sq, who), gb = __shfl_sync(0xFFFFFFFFu, sb, who);
    first_value = __shfl_sync(0xFFFFFFFFu, value, who);
    first = __shfl_sync(0xFFFFFFFFu, start, who);
    split();
    return true;
  }
};

}  // namespace bq
}  // namespace pxc
