// bq.cu — the block quantiser (pxc_bq_*): encode, decode, the product of two sets of
// encoded rows, and the product grouped by ragged lists.
#include <algorithm>
#include <type_traits>

#include "bq.cuh"
#include "bq_tc.cuh"
#include "tmap.cuh"

namespace pxc {
namespace bq {

constexpr uint64_t MAX_ROWS = (uint64_t(1) << 31) - 1024;  // row numbers and tile ends fit an int32
constexpr uint32_t MAX_DIM = 1u << 20;
constexpr uint64_t MAX_SIZE = uint64_t(1) << 48;  // values in an output: offsets of them cannot overflow

static uint64_t up(uint64_t x, uint64_t to) { return (x + to - 1) / to * to; }
static uint32_t blocks_of(uint32_t dim) { return (dim + BLOCK - 1) / BLOCK; }

// ---- encode and decode ----
// Both should be bound by the bytes they read and write: a block of 16-bit components moves 388, which an SM's share of
// 6.5 TB/s brings in 17 cycles, and its four schedulers issue 66 instructions of a warp meanwhile at the very
// best. So eight lanes share a block and a warp works on four rows at once: a lane
// moves 16 bytes of vector at a time, and what is done once per block (the reduction, the scale, the
// addresses) is done for four. Items go by a fixed step: no division stands in the loop.
//
// Where rows do not start on 16 bytes (an odd pitch or base), the encoder gathers the same 16 bytes from
// narrower loads, none of which leaves them. The decoder takes short rows without gaps as one array then, and
// else gives a whole warp to a block, its lanes 32 apart, so that each store covers neighbouring bytes: partial
// sectors would each be written several times over.

// The items of one warp: a block of the R rows from `row` on.
template <uint32_t R>
struct Items {
  uint64_t row;
  uint32_t block;
  __device__ __forceinline__ Items(uint32_t blocks) {
    const uint32_t number = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    row = static_cast<uint64_t>(number / blocks) * R;
    block = number % blocks;
  }
  __device__ __forceinline__ void next(uint64_t step_rows, uint32_t step_blocks, uint32_t blocks) {
    row += step_rows;
    if (step_blocks == 0) {
      // a step of whole rows would leave a warp at one block of them, the short last one always to the
      // same warps: all of a step's items move on by one block together
      block = block + 1 == blocks ? 0 : block + 1;
    } else {
      block += step_blocks;
      if (block >= blocks) block -= blocks, row += R;
    }
  }
};

template <class T>
constexpr uint32_t CHUNK = 16 / sizeof(T);  // components in 16 bytes
// Chunks of 16 bytes per lane in a block, and rows per item: 2 KB of vectors per warp in flight either way.
// Short vectors have one chunk a lane at most, and 16 rows an item.
template <class T>
constexpr uint32_t FULL = 16 / CHUNK<T>;
template <class T>
constexpr uint32_t SHORT_DIM = 8 * CHUNK<T>;
template <class T, uint32_t C>
constexpr uint32_t WIDE_ROWS = C == 1 ? 16 : 16 / C;
constexpr uint32_t NARROW_ROWS = 4;

// 16 bytes of components as f32, and back.
template <class T>
__device__ __forceinline__ void unpack(const uint4& q, float (&v)[CHUNK<T>]) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same_v<T, float>) {
      v[i] = __uint_as_float(w[i]);
    } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
      v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
  }
}
template <class T>
__device__ __forceinline__ uint4 pack(const float (&v)[CHUNK<T>]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same_v<T, float>) {
      w[i] = __float_as_uint(v[i]);
    } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// One row's scale byte, and the padding behind the last.
__device__ __forceinline__ void store_scale(uint8_t* row, uint32_t block, uint32_t blocks, uint32_t byte) {
  if (blocks == 1) {
    *reinterpret_cast<uint32_t*>(row) = byte;
  } else {
    row[block] = static_cast<uint8_t>(byte);
    if (block + 1 == blocks)
      for (uint32_t k = blocks; k & 3; ++k) row[k] = 0;
  }
}

// 16 bytes of components from any address that is aligned to one: 16-bit types by the three words that lie
// on word boundaries and the two components around or behind them.
template <class T>
__device__ __forceinline__ uint4 gather(const T* p) {
  if constexpr (sizeof(T) == 4) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(p);
    return make_uint4(__ldcs(w), __ldcs(w + 1), __ldcs(w + 2), __ldcs(w + 3));
  } else {
    const uint32_t odd = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p) >> 1) & 1u, shift = 16 * odd;
    const uint32_t* w = reinterpret_cast<const uint32_t*>(p + odd);
    const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
    const uint32_t w0 = w[0], w1 = w[1], w2 = w[2], h0 = h[odd ? 0 : 6], h7 = h[7];
    return make_uint4(__funnelshift_l(h0 << 16, w0, shift), __funnelshift_l(w0, w1, shift),
                      __funnelshift_l(w1, w2, shift), __funnelshift_l(w2, odd ? h7 : h0 | h7 << 16, shift));
  }
}

template <class T, bool WIDE, uint32_t C>
__global__ void __launch_bounds__(256)
    encode_kernel(const T* __restrict__ x, uint64_t stride, uint64_t rows, uint32_t dim, uint32_t blocks,
                       uint8_t* __restrict__ codes, uint64_t ld, uint8_t* __restrict__ scales, uint64_t sld,
                       uint64_t step_rows, uint32_t step_blocks) {
  constexpr uint32_t V = CHUNK<T>, R = WIDE_ROWS<T, C>, U = R / 4;
  const uint32_t lane = threadIdx.x & 31, l = lane & 7, group = lane >> 3;
  const uint32_t code_end = (dim + 15) / 16 * 16;
  for (Items<R> it(blocks); it.row < rows; it.next(step_rows, step_blocks, blocks)) {
    const uint32_t c0 = it.block * BLOCK + l * V;  // chunk k: 8 * V further each
    float v[U][C][V];
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      const uint64_t r = it.row + u * 4 + group;
      const T* p = x + r * stride + c0;
#pragma unroll
      for (uint32_t k = 0; k < C; ++k) {
        uint4 q = make_uint4(0, 0, 0, 0);
        if (r < rows && c0 + k * 8 * V + V <= dim) {
          if constexpr (WIDE)
            q = __ldcs(reinterpret_cast<const uint4*>(p + k * 8 * V));
          else
            q = gather<T>(p + k * 8 * V);
        }
        unpack<T>(q, v[u][k]);
      }
    }
    if (dim % V != 0 && it.block + 1 == blocks) {  // the components behind the last whole chunk
#pragma unroll
      for (uint32_t u = 0; u < U; ++u) {
        const uint64_t r = it.row + u * 4 + group;
#pragma unroll
        for (uint32_t k = 0; k < C; ++k) {
          const uint32_t c = c0 + k * 8 * V;
          if (r < rows && c < dim && c + V > dim)
#pragma unroll
            for (uint32_t i = 0; i < V - 1; ++i)
              if (c + i < dim) v[u][k][i] = to_f32<T>(x[r * stride + c + i]);
        }
      }
    }
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      // fmax passes over NaN; an infinity is left out when it shows
      float top = 0.0f;
#pragma unroll
      for (uint32_t k = 0; k < C; ++k)
#pragma unroll
        for (uint32_t i = 0; i < V; ++i) top = fmaxf(top, fabsf(v[u][k][i]));
#pragma unroll
      for (uint32_t d = 4; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
      if (__any_sync(0xFFFFFFFFu, __float_as_uint(top) == 0x7F800000u)) {
        uint32_t finite = 0;
#pragma unroll
        for (uint32_t k = 0; k < C; ++k)
#pragma unroll
          for (uint32_t i = 0; i < V; ++i) finite = max(finite, finite_bits(v[u][k][i]));
#pragma unroll
        for (uint32_t d = 4; d; d >>= 1) finite = max(finite, __shfl_xor_sync(0xFFFFFFFFu, finite, d));
        top = __uint_as_float(finite);
      }
      const uint32_t byte = scale_byte(__float_as_uint(top));
      const float f = inverse_scale(byte);
      const uint64_t r = it.row + u * 4 + group;
      if (r < rows) {
        uint8_t* to = codes + r * ld + c0;
#pragma unroll
        for (uint32_t k = 0; k < C; ++k) {
          uint32_t four[V / 4];
#pragma unroll
          for (uint32_t i = 0; i < V; i += 4)
            four[i / 4] = to_codes(v[u][k][i] * f, v[u][k][i + 1] * f, v[u][k][i + 2] * f, v[u][k][i + 3] * f);
          if (c0 + k * 8 * V < code_end) {
            if constexpr (V == 4)
              *reinterpret_cast<uint32_t*>(to + k * 32) = four[0];
            else
              *reinterpret_cast<uint2*>(to + k * 64) = make_uint2(four[0], four[1]);
          }
        }
        if (l == 0) store_scale(scales + r * sld, it.block, blocks, byte);
      }
    }
  }
}

template <class T, uint32_t C>
__global__ void __launch_bounds__(256)
    decode_wide_kernel(const uint8_t* __restrict__ codes, uint64_t ld, const uint8_t* __restrict__ scales, uint64_t sld,
                       uint64_t rows, uint32_t dim, uint32_t blocks, T* __restrict__ out, uint64_t stride,
                       uint64_t step_rows, uint32_t step_blocks) {
  constexpr uint32_t V = CHUNK<T>, R = WIDE_ROWS<T, C>, U = R / 4;
  const uint32_t lane = threadIdx.x & 31, l = lane & 7, group = lane >> 3;
  for (Items<R> it(blocks); it.row < rows; it.next(step_rows, step_blocks, blocks)) {
    const uint32_t c0 = it.block * BLOCK + l * V;
    uint32_t q[U][C][V / 4], byte[U];
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      const uint64_t r = it.row + u * 4 + group;
      const uint8_t* p = codes + r * ld + c0;
      byte[u] = r < rows ? scales[r * sld + it.block] : 0u;
#pragma unroll
      for (uint32_t k = 0; k < C; ++k) {
        const bool any = r < rows && c0 + k * 8 * V < dim;  // a chunk is 4 or 8 bytes of the pitch's 16
        if constexpr (V == 4) {
          q[u][k][0] = any ? __ldcs(reinterpret_cast<const uint32_t*>(p + k * 32)) : 0u;
        } else {
          const uint2 w = any ? __ldcs(reinterpret_cast<const uint2*>(p + k * 64)) : make_uint2(0, 0);
          q[u][k][0] = w.x, q[u][k][1] = w.y;
        }
      }
    }
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      const uint64_t r = it.row + u * 4 + group;
      const float f = scale_value(byte[u]);
      T* p = out + r * stride + c0;
#pragma unroll
      for (uint32_t k = 0; k < C; ++k) {
        float v[V];
#pragma unroll
        for (uint32_t i = 0; i < V; i += 2) {
          const float2 two = from_codes((q[u][k][i / 4] >> (8 * (i & 2))) & 0xFFFFu);
          v[i] = two.x * f, v[i + 1] = two.y * f;
        }
        const uint32_t c = c0 + k * 8 * V;
        if (r < rows && c + V <= dim) {
          __stcs(reinterpret_cast<uint4*>(p + k * 8 * V), pack<T>(v));
        } else if (r < rows && c < dim) {
#pragma unroll
          for (uint32_t i = 0; i < V - 1; ++i)
            if (c + i < dim) p[k * 8 * V + i] = from_f32<T>(v[i]);
        }
      }
    }
  }
}

template <class T, bool WHOLE>
__device__ __forceinline__ void decode_narrow(const uint8_t* __restrict__ p, uint64_t ld, const uint8_t* __restrict__ s,
                                              uint64_t sld, uint32_t n, uint32_t left, T* __restrict__ to,
                                              uint64_t stride) {
  constexpr uint32_t R = NARROW_ROWS;
  uint32_t code[R][4], byte[R];
#pragma unroll
  for (uint32_t u = 0; u < R; ++u, p += ld, s += sld) {
    byte[u] = WHOLE || u < n ? *s : 0u;
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) code[u][k] = WHOLE || (u < n && 32 * k < left) ? p[32 * k] : 0u;
  }
#pragma unroll
  for (uint32_t u = 0; u < R; ++u, to += stride) {
    const float f = scale_value(byte[u]);
#pragma unroll
    for (uint32_t k = 0; k < 4; k += 2) {
      const float2 two = from_codes(code[u][k] | code[u][k + 1] << 8);
      if (WHOLE || (u < n && 32 * k < left)) to[32 * k] = from_f32<T>(two.x * f);
      if (WHOLE || (u < n && 32 * (k + 1) < left)) to[32 * (k + 1)] = from_f32<T>(two.y * f);
    }
  }
}

template <class T>
__global__ void __launch_bounds__(256)
    decode_narrow_kernel(const uint8_t* __restrict__ codes, uint64_t ld, const uint8_t* __restrict__ scales,
                         uint64_t sld, uint64_t rows, uint32_t dim, uint32_t blocks, T* __restrict__ out,
                         uint64_t stride, uint64_t step_rows, uint32_t step_blocks) {
  constexpr uint32_t R = NARROW_ROWS;
  const uint32_t lane = threadIdx.x & 31;
  for (Items<R> it(blocks); it.row < rows; it.next(step_rows, step_blocks, blocks)) {
    const uint32_t b0 = it.block * BLOCK, c0 = b0 + lane;
    const uint32_t n = static_cast<uint32_t>(min(static_cast<uint64_t>(R), rows - it.row));
    const uint8_t* p = codes + it.row * ld + c0;
    const uint8_t* s = scales + it.row * sld + it.block;
    T* to = out + it.row * stride + c0;
    if (n < R || b0 + BLOCK > dim)
      decode_narrow<T, false>(p, ld, s, sld, n, c0 < dim ? dim - c0 : 0, to, stride);
    else
      decode_narrow<T, true>(p, ld, s, sld, R, 0, to, stride);
  }
}

// Rows without gaps whose pitch is not a multiple of 16 bytes are one array all the same: a thread has 16
// aligned bytes of it, which lie in one row or, dim >= V, in two. A chunk's codes are a funnel of the
// words around them; it meets up to three scales.
template <class T>
__global__ void __launch_bounds__(256)
    decode_flat_kernel(const uint8_t* __restrict__ codes, uint64_t ld, const uint8_t* __restrict__ scales, uint64_t sld,
                       uint64_t rows, uint32_t dim, T* __restrict__ out, uint64_t step_rows, uint32_t step_rest) {
  constexpr uint32_t V = CHUNK<T>, W = V / 4;
  const uint64_t total = rows * dim, step = static_cast<uint64_t>(gridDim.x) * blockDim.x * V;
  uint64_t at = (static_cast<uint64_t>(blockIdx.x) * blockDim.x + threadIdx.x) * V;
  uint64_t row = at / dim;
  uint32_t col = static_cast<uint32_t>(at - row * dim);
  const uint32_t last_word = (dim - 1) / 4;
  for (; at < total; at += step) {
    const uint8_t* s = scales + row * sld;
    const uint32_t* c = reinterpret_cast<const uint32_t*>(codes + row * ld);
    const bool next = row + 1 < rows;  // where not, what lies behind is not stored
    const uint32_t* c2 = next ? reinterpret_cast<const uint32_t*>(codes + (row + 1) * ld) : c;
    const uint32_t split = min(V, dim - col), cut = min(split, BLOCK - (col & (BLOCK - 1)));
    uint32_t w[W + 1], w2[W];
#pragma unroll
    for (uint32_t i = 0; i <= W; ++i) w[i] = __ldg(c + min(col / 4 + i, last_word));
    if (split < V) {
#pragma unroll
      for (uint32_t i = 0; i < W; ++i) w2[i] = __ldg(c2 + i);
    }
    const float f0 = scale_value(s[col / BLOCK]);
    const float f1 = cut < split ? scale_value(s[col / BLOCK + 1]) : f0;
    const float f2 = split < V ? scale_value(next ? s[sld] : s[0]) : f1;
    uint64_t q = 0;
#pragma unroll
    for (uint32_t i = 0; i < W; ++i)
      q |= static_cast<uint64_t>(__funnelshift_r(w[i], w[i + 1], 8 * (col & 3))) << (32 * i);
    if (split < V) {
      uint64_t behind = w2[0];
      if constexpr (W == 2) behind |= static_cast<uint64_t>(w2[1]) << 32;
      q = (q & ((uint64_t(1) << (8 * split)) - 1)) | behind << (8 * split);
    }
    float v[V];
#pragma unroll
    for (uint32_t i = 0; i < V; i += 2) {
      const float2 two = from_codes(static_cast<uint32_t>(q >> (8 * i)) & 0xFFFFu);
      v[i] = two.x * (i < cut ? f0 : i < split ? f1 : f2);
      v[i + 1] = two.y * (i + 1 < cut ? f0 : i + 1 < split ? f1 : f2);
    }
    if (at + V <= total) {
      __stcs(reinterpret_cast<uint4*>(out + at), pack<T>(v));
    } else {
#pragma unroll
      for (uint32_t i = 0; i < V - 1; ++i)
        if (at + i < total) out[at + i] = from_f32<T>(v[i]);
    }
    row += step_rows;
    col += step_rest;
    if (col >= dim) col -= dim, ++row;
  }
}

// A grouped product of no queries, no rows or no room: its offsets are looked over all the same.
__global__ void __launch_bounds__(256) check_empty_kernel(Groups g) {
  bool bad = false;
  for (uint64_t i = blockIdx.x * blockDim.x + threadIdx.x; i < g.groups; i += gridDim.x * blockDim.x) {
    const int64_t q0 = g.q_offsets[i], q1 = g.q_offsets[i + 1];
    bad = bad || !Walk::within(q0, q1, g.nq);
    if (g.b_offsets) {
      const int64_t b0 = g.b_offsets[i], b1 = g.b_offsets[i + 1];
      bad = bad || !Walk::within(b0, b1, g.nb) || (q1 != q0 && b1 != b0);  // a matrix, and no room
    }
  }
  if (bad) leave_fault(g.record, FAULT_OFFSETS);
}

// ---- host ----
// Who makes a call of the device forms, on which stream, and whose failures it reports.
struct Caller {
  pxc_ctx* ctx;
  cudaStream_t stream;
  Record record;    // what this call's kernels write
  Record told[2];   // earlier failures that the call reports

  // `number` 0: told apart by stream. `fails`: this call may leave a failure.
  Caller(pxc_ctx* c, uint64_t number, void* s, bool fails) : ctx(c) {
    PXC_CONFIG(ctx != nullptr, "ctx", 0, "null context");
    stream = s ? static_cast<cudaStream_t>(s) : ctx->stream;
    Reports& reports = *ctx->bq_reports;
    if (number != 0) {
      told[0] = record = reports.of_caller(number, fails);
      if (fails && capturing()) reports.keep(number);
      return;
    }
    told[0] = record = reports.of_stream(stream);
    told[1] = reports.captured();
    if (fails && capturing()) record = reports.captured();
  }
  bool capturing() const {
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(stream, &status) != cudaSuccess) cudaGetLastError();  // the launch will say what is wrong
    return status != cudaStreamCaptureStatusNone;
  }
  void report() const {
    for (const Record& r : told)
      if (r.words) r.take();
  }
};

static void check_common(uint32_t dim, int32_t dtype) {
  PXC_CONFIG(dim >= 1 && dim <= MAX_DIM, "dim", dim, "must be between 1 and 1048576");
  PXC_CONFIG(dtype == PXC_DTYPE_F32 || dtype == PXC_DTYPE_F16 || dtype == PXC_DTYPE_BF16, "dtype", dtype,
             "must be f32, f16 or bf16");
}

// Device rows are read by wide loads and tensor maps; host rows are copied, at any alignment.
static void check_rows(const pxc_bq_rows* r, uint32_t dim, const char* name, bool device) {
  PXC_CONFIG(r != nullptr, name, 0, "null rows");
  PXC_CONFIG(r->rows <= MAX_ROWS, name, r->rows, "at most 2^31 - 1024 rows");
  if (r->rows == 0) return;
  PXC_CONFIG(r->codes != nullptr && r->scales != nullptr, name, 0, "null codes or scales");
  PXC_CONFIG(!device || (reinterpret_cast<uintptr_t>(r->codes) & 15) == 0, name, reinterpret_cast<uintptr_t>(r->codes),
             "codes must be 16-byte aligned");
  PXC_CONFIG(!device || (reinterpret_cast<uintptr_t>(r->scales) & 3) == 0, name, reinterpret_cast<uintptr_t>(r->scales),
             "scales must be 4-byte aligned");
  PXC_CONFIG(r->ld >= dim && (r->ld & 15) == 0 && r->ld < (uint64_t(1) << 32), "ld", r->ld,
             "the code pitch must be a multiple of 16, at least dim and below 2^32");
  PXC_CONFIG(r->sld >= blocks_of(dim) && (r->sld & 3) == 0 && r->sld < (uint64_t(1) << 32), "sld", r->sld,
             "the scale pitch must be a multiple of 4, at least ceil(dim / 128) and below 2^32");
}

static void count_launch(pxc_ctx* ctx) { __atomic_fetch_add(&ctx->launches, 1ull, __ATOMIC_RELAXED); }

static size_t size_of(int32_t dtype) { return dtype == PXC_DTYPE_F32 ? 4 : 2; }

template <class F>
static void with_type(int32_t dtype, F&& f) {
  if (dtype == PXC_DTYPE_F32)
    f(static_cast<float*>(nullptr));
  else if (dtype == PXC_DTYPE_F16)
    f(static_cast<__half*>(nullptr));
  else
    f(static_cast<__nv_bfloat16*>(nullptr));
}

// Grid and step of the kernels above: items are a block of R rows, 8 a CTA at a time. Many short CTAs even out
// the SMs' shares where a warp moves few bytes at a time (decode 1M x 128 to f32: 8 an SM 110 us, 64
// 97 us); 16-bit vectors are encoded by long ones (8192 x 4096 bf16: 21 us, with 64 23 us).
struct Sweep {
  unsigned grid;
  uint64_t step_rows;
  uint32_t step_blocks;
  Sweep(const pxc_ctx* ctx, uint64_t rows, uint32_t blocks, uint32_t R, uint32_t per_sm) {
    const uint64_t items = (rows + R - 1) / R * blocks;
    grid = static_cast<unsigned>(std::min<uint64_t>((items + 7) / 8, static_cast<uint64_t>(ctx->sm_count) * per_sm));
    step_rows = static_cast<uint64_t>(grid) * 8 / blocks * R;
    step_blocks = grid * 8 % blocks;
  }
};

// Whether every row starts on 16 bytes.
static bool rows_wide(const void* p, uint64_t stride, int32_t dtype) {
  return (reinterpret_cast<uintptr_t>(p) | stride * size_of(dtype)) % 16 == 0;
}

static void encode(pxc_ctx* ctx, const void* x, int32_t dtype, uint64_t stride, uint32_t dim, const pxc_bq_rows& out,
                   cudaStream_t s) {
  const uint32_t blocks = blocks_of(dim);
  with_type(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr uint32_t F = FULL<T>;
    const bool wide = rows_wide(x, stride, dtype), few = dim <= SHORT_DIM<T>;
    const Sweep w(ctx, out.rows, blocks, few ? WIDE_ROWS<T, 1> : WIDE_ROWS<T, F>, sizeof(T) == 4 ? 64 : 8);
    auto kernel = few ? (wide ? encode_kernel<T, true, 1> : encode_kernel<T, false, 1>)
                      : (wide ? encode_kernel<T, true, F> : encode_kernel<T, false, F>);
    kernel<<<w.grid, 256, 0, s>>>(static_cast<const T*>(x), stride, out.rows, dim, blocks, out.codes, out.ld,
                                  out.scales, out.sld, w.step_rows, w.step_blocks);
  });
  PXC_CUDA(cudaGetLastError());
  count_launch(ctx);
}

static void decode(pxc_ctx* ctx, const pxc_bq_rows& in, uint32_t dim, void* out, int32_t dtype, uint64_t stride,
                   cudaStream_t s) {
  const uint32_t blocks = blocks_of(dim);
  with_type(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr uint32_t F = FULL<T>;
    const bool wide = rows_wide(out, stride, dtype), few = dim <= SHORT_DIM<T>;
    // Short rows leave the narrow kernel's warps part empty; long ones suit it, 32-bit rows of two blocks already.
    // Narrow and as one array, 2M rows of 31: f32 175 and 79 us, f16 178 and 54. 128M values of f32: dim 97 176 and 153,
    // 127 157 and 151, 129 147 and 155, 193 140 and 149, 385 138 and 147, 1001 139 and 145; of f16: 129 143 and 108,
    // 193 112 and 106, 257 111 and 106, 385 101 and 103, 1001 100 and 100.
    constexpr uint32_t SHORT_BLOCKS = sizeof(T) == 4 ? 1 : 2;
    const bool flat = !wide && stride == dim && reinterpret_cast<uintptr_t>(out) % 16 == 0;
    if (flat && dim >= CHUNK<T> && blocks <= SHORT_BLOCKS) {
      const uint64_t threads = (in.rows * dim + CHUNK<T> - 1) / CHUNK<T>;
      const unsigned grid =
          static_cast<unsigned>(std::min<uint64_t>((threads + 255) / 256, static_cast<uint64_t>(ctx->sm_count) * 32));
      const uint64_t step = static_cast<uint64_t>(grid) * 256 * CHUNK<T>;
      decode_flat_kernel<T><<<grid, 256, 0, s>>>(in.codes, in.ld, in.scales, in.sld, in.rows, dim, static_cast<T*>(out),
                                                 step / dim, static_cast<uint32_t>(step % dim));
      return;
    }
    const Sweep w(ctx, in.rows, blocks, !wide ? NARROW_ROWS : few ? WIDE_ROWS<T, 1> : WIDE_ROWS<T, F>, 64);
    auto kernel = !wide ? decode_narrow_kernel<T> : few ? decode_wide_kernel<T, 1> : decode_wide_kernel<T, F>;
    kernel<<<w.grid, 256, 0, s>>>(in.codes, in.ld, in.scales, in.sld, in.rows, dim, blocks, static_cast<T*>(out),
                                  stride, w.step_rows, w.step_blocks);
  });
  PXC_CUDA(cudaGetLastError());
  count_launch(ctx);
}

// Several times 128 rows per tile where few queries leave a tile little work, as long as the rounds of
// tiles over the SMs stay about as even. By 128, 256 and 512 rows, queries' encoding not counted: 1 x 1M x 128 44.2, 31.4
// and 31.2 us; 16 x 500k x 768 76.0, 72.4 and 71.2; 16 x 75,776 x 768 (4, 2 and 1 rounds) 14.8, 12.7 and 12.6; 1 x 20k x
// 768 (2, 1 and 1) 10.6, 10.1 and 10.7; 48 x 100k x 768 20.6, 16.8 and 18.9. By 128 and 256: 64 x 100k x 768 20.9 and
// 16.8, 64 x 1M x 128 77.2 and 78.0, 100 x 100k x 768 22.9 and 22.1.
static uint32_t narrow_subs(uint32_t q_rows, uint64_t rows, uint64_t sms) {
  const auto rounds = [&](uint64_t subs) { return up(up(rows, subs * bq_tc::BM) / (subs * bq_tc::BM), sms) / sms * subs; };
  for (uint32_t subs = q_rows <= 48 ? 4 : q_rows <= 64 ? 2 : 1; subs > 1; subs /= 2)
    if (rounds(subs) * 10 <= rounds(1) * 11) return subs;
  return 1;
}

// The tile of a dense product: `width` queries, by 128 rows or as a pair by 256.
struct Shape {
  uint32_t width;
  bool pair;
};
// The one whose rounds over the SMs take least (200 x 2000 x 128: 8.6 us with the widest tiles, 6.4 so; 1024 x 1024 x
// 1024: 11.5, 9.7). The widest even split is always among those looked at. A block of a tile takes 340 cycles and 1.4 a
// query (measured from 128 to 224 queries a tile), a tile itself some 1,400, and a CTA on its own a twelfth longer than
// as one of a pair.
static Shape dense_shape(uint64_t nq, uint64_t rows, uint32_t kblocks, uint64_t sms) {
  Shape best{};
  uint64_t least = ~uint64_t(0);
  for (uint32_t width = bq_tc::MAX_Q; width >= 16; width -= 16) {
    const uint64_t qt = (nq + width - 1) / width;
    if (up((nq + qt - 1) / qt, 16) != width) continue;  // the even split is another width
    if (qt > 1 && width < 64) break;  // the rows would pass too often (100 x 2000 x 2048: 11.5 us, by 16 at a time 13)
    for (int pair = 0; pair < 2; ++pair) {
      if (pair && (width <= 112 || rows <= bq_tc::BM)) continue;
      const uint64_t tall = bq_tc::BM << pair, slots = sms >> pair;
      const uint64_t rounds = (qt * ((rows + tall - 1) / tall) + slots - 1) / slots;
      const uint64_t cost = rounds * (static_cast<uint64_t>(kblocks) * (240 + width) + 1000) * (pair ? 12 : 13);
      if (cost < least) least = cost, best = Shape{width, pair != 0};
    }
  }
  return best;
}

static void product(pxc_ctx* ctx, const pxc_bq_rows& q, const pxc_bq_rows& b, uint32_t dim, const Groups& g, void* out,
                    int32_t dtype, cudaStream_t s, const Record& record) {
  using namespace bq_tc;
  Params p{};
  p.groups = g;
  p.groups.nq = q.rows;
  p.groups.nb = b.rows;
  p.groups.record = record;
  p.q_scales = q.scales;
  p.b_scales = b.scales;
  p.q_sld = q.sld;
  p.b_sld = b.sld;
  p.out = out;
  p.dim = dim;
  p.kblocks = blocks_of(dim);
  const bool dense = !g.q_offsets;
  bool pair;
  if (dense) {
    const Shape shape = dense_shape(q.rows, b.rows, p.kblocks, ctx->sm_count);
    p.tile_q = p.q_rows = shape.width;
    pair = shape.pair;
    p.subs = q.rows <= shape.width && !pair ? narrow_subs(p.q_rows, b.rows, ctx->sm_count) : 1;
  } else {
    // room for twice the mean, so that most groups are one tile and the rings stay deep
    const uint64_t mean = q.rows / g.groups;
    p.tile_q = p.q_rows = static_cast<uint32_t>(std::min<uint64_t>(MAX_Q, std::max<uint64_t>(32, up(2 * mean, 32))));
    // Pairs where groups average many queries and many rows: else their fewer, taller tiles leave the groups' and the
    // SMs' last rounds emptier than cheaper loads make up for. Without and with pairs, to bf16, groups x 2048 x 2048:
    // mean 128 59.8 and 66.0 us, 256 49.5 and 52.1, 512 81.1 and 78.5, 1024 73.3 and 68.7; 8 x 4096 x 2048, mean 2048
    // 136.7 and 128.2; 500 x 1000 x 128, mean 200 64 and 74; 32 x 300 x 512, mean 1024 19.1 and 23.3; 32 x 256 x 2048,
    // mean 512 21.2 and 21.3; 64 x 700 x 300, mean 625 35.4 and 33.5.
    pair = mean >= 512 && b.rows / g.groups > 512;
    p.subs = 1;
  }
  const uint32_t tile_rows = pair ? 2 * BM : p.subs * BM;
  p.tile_log2 = tile_rows == BM ? 7 : tile_rows == 2 * BM ? 8 : 9;
  p.q_load = pair ? p.q_rows / 2 : p.q_rows;
  if (dense) {
    p.q_box = p.q_load;  // every tile but the last is this wide: one box brings it
  } else {
    p.q_box = 32;  // as many boxes as a tile needs
    p.q_load = static_cast<uint32_t>(up(p.q_load, 32));
  }
  p.wait_cycles = static_cast<uint64_t>(ctx->wait_ms) * 2000000ull;  // the SM clock is below 2 GHz
  const uint32_t smem = plan(p);
  CUtensorMap map_b, map_q;
  make_tmap_u8_pitched(&map_b, b.codes, dim, b.ld, b.rows, BM);
  make_tmap_u8_pitched(&map_q, q.codes, dim, q.ld, q.rows, p.q_box);
  // no more CTAs than tiles, where the host can tell
  uint64_t tiles = ctx->sm_count;
  if (dense)
    tiles = (q.rows + p.tile_q - 1) / p.tile_q * ((b.rows + tile_rows - 1) / tile_rows);
  else if (!g.b_offsets)
    tiles = (std::min<uint64_t>(g.groups, q.rows) + q.rows / p.tile_q) * ((g.n_each + tile_rows - 1) / tile_rows);
  const uint32_t ctas = pair ? 2 : 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(std::min<uint64_t>(ctx->sm_count / ctas, std::max<uint64_t>(tiles, 1))) * ctas);
  config.blockDim = dim3(THREADS);
  config.dynamicSmemBytes = smem;
  config.stream = s;
  cudaLaunchAttribute cluster{};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = 2;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  config.attrs = &cluster;
  config.numAttrs = pair ? 1 : 0;
  with_type(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    auto kernel = pair          ? product_kernel<T, true, 1>
                  : p.subs == 4 ? product_kernel<T, false, 4>
                  : p.subs == 2 ? product_kernel<T, false, 2>
                                : product_kernel<T, false, 1>;
    const uint32_t bit = 1u << (4 * dtype + (pair ? 3 : p.subs / 2));
    if (!(__atomic_load_n(&ctx->bq_ready, __ATOMIC_ACQUIRE) & bit)) {  // once per context and kernel
      PXC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_LIMIT));
      __atomic_fetch_or(&ctx->bq_ready, bit, __ATOMIC_RELEASE);
    }
    PXC_CUDA(cudaLaunchKernelEx(&config, kernel, map_b, map_q, p));
  });
  count_launch(ctx);
}

static void check_vectors(const void* x, int32_t dtype, uint64_t stride, uint32_t dim, const char* name) {
  PXC_CONFIG(x != nullptr, name, 0, "null buffer");
  PXC_CONFIG(reinterpret_cast<uintptr_t>(x) % size_of(dtype) == 0, name, reinterpret_cast<uintptr_t>(x),
             "not aligned to its type");
  PXC_CONFIG(stride >= dim && stride < (uint64_t(1) << 32), "stride", stride, "must be at least dim and below 2^32");
}

static void check_product(const pxc_bq_rows* q, const pxc_bq_rows* b, uint32_t dim, const void* out, int32_t dtype,
                          uint64_t stride, bool device) {
  check_rows(q, dim, "queries", device);
  check_rows(b, dim, "base", device);
  if (q->rows == 0 || b->rows == 0) return;
  PXC_CONFIG(out != nullptr && reinterpret_cast<uintptr_t>(out) % size_of(dtype) == 0, "out",
             reinterpret_cast<uintptr_t>(out), "null or not aligned to its type");
  PXC_CONFIG(stride >= b->rows && stride <= MAX_SIZE / q->rows, "stride", stride,
             "must be at least the base rows, and the output at most 2^48 values");
}

// The even form's rows per group.
static uint64_t check_grouped(const pxc_bq_rows* q, const void* qo, const pxc_bq_rows* b, const void* bo, uint32_t groups,
                              uint32_t dim, const void* out, int32_t dtype, uint64_t size, bool device) {
  check_rows(q, dim, "queries", device);
  check_rows(b, dim, "base", device);
  PXC_CONFIG(groups >= 1 && groups <= (1u << 24), "groups", groups, "must be between 1 and 16777216");
  PXC_CONFIG(qo != nullptr, "offsets", 0, "null query offsets");
  PXC_CONFIG(size <= MAX_SIZE, "size", size, "at most 2^48 values");
  PXC_CONFIG(size == 0 || (out != nullptr && reinterpret_cast<uintptr_t>(out) % size_of(dtype) == 0), "out",
             reinterpret_cast<uintptr_t>(out), "null or not aligned to its type");
  if (bo) return 0;
  PXC_CONFIG(b->rows % groups == 0, "base", b->rows, "without base offsets the rows must be a multiple of the groups");
  const uint64_t each = b->rows / groups;
  PXC_CONFIG(q->rows == 0 || each <= MAX_SIZE / q->rows, "base", b->rows, "the output is at most 2^48 values");
  PXC_CONFIG(size >= q->rows * each, "size", size, "smaller than the queries times a group's rows");
  return each;
}

// `rows` rows of `width` bytes between pitches; in one piece where there is nothing between them (a 2-D copy's
// pitch is limited).
static void copy_rows(void* dst, uint64_t dst_pitch, const void* src, uint64_t src_pitch, uint64_t width, uint64_t rows,
                      cudaMemcpyKind kind, cudaStream_t s) {
  if (rows <= 1 || (dst_pitch == width && src_pitch == width))
    PXC_CUDA(cudaMemcpyAsync(dst, src, width * rows, kind, s));
  else
    PXC_CUDA(cudaMemcpy2DAsync(dst, dst_pitch, src, src_pitch, width, rows, kind, s));
}

// Device copies of host rows, with the pitches that the kernels want.
struct Staged {
  DBuf<uint8_t> codes, scales;
  pxc_bq_rows d{};
  void make(uint64_t rows, uint32_t dim) {
    d.rows = rows;
    d.ld = up(dim, 16);
    d.sld = up(blocks_of(dim), 4);
    codes.reserve(rows * d.ld);
    scales.reserve(rows * d.sld);
    d.codes = codes.p;
    d.scales = scales.p;
  }
  void load(const pxc_bq_rows& h, uint32_t dim, cudaStream_t s) {
    make(h.rows, dim);
    if (h.rows == 0) return;
    copy_rows(d.codes, d.ld, h.codes, h.ld, dim, h.rows, cudaMemcpyHostToDevice, s);
    copy_rows(d.scales, d.sld, h.scales, h.sld, blocks_of(dim), h.rows, cudaMemcpyHostToDevice, s);
  }
};

static void check_host_offsets(const int64_t* o, uint32_t groups, uint64_t rows) {
  for (uint32_t g = 0; g < groups; ++g)
    PXC_CONFIG(o[g] >= 0 && o[g + 1] >= o[g] && static_cast<uint64_t>(o[g + 1]) <= rows, "offsets", g,
               "offsets must rise and stay within the rows");
}

// ---- the device forms ----
static void encode_device(const Caller& c, const void* vectors, int32_t dtype, uint64_t stride, uint32_t dim,
                          const pxc_bq_rows* out) {
  check_common(dim, dtype);
  c.report();
  check_rows(out, dim, "out", true);
  if (out->rows == 0) return;
  check_vectors(vectors, dtype, stride, dim, "vectors");
  DeviceGuard g(c.ctx->device);
  encode(c.ctx, vectors, dtype, stride, dim, *out, c.stream);
}

static void decode_device(const Caller& c, const pxc_bq_rows* rows, uint32_t dim, void* out, int32_t dtype,
                          uint64_t stride) {
  check_common(dim, dtype);
  c.report();
  check_rows(rows, dim, "rows", true);
  if (rows->rows == 0) return;
  check_vectors(out, dtype, stride, dim, "out");
  DeviceGuard g(c.ctx->device);
  decode(c.ctx, *rows, dim, out, dtype, stride, c.stream);
}

static void product_device(const Caller& c, const pxc_bq_rows* queries, const pxc_bq_rows* base, uint32_t dim, void* out,
                           int32_t dtype, uint64_t stride) {
  check_common(dim, dtype);
  c.report();
  check_product(queries, base, dim, out, dtype, stride, true);
  if (queries->rows == 0 || base->rows == 0) return;
  DeviceGuard g(c.ctx->device);
  Groups groups{};
  groups.groups = 1;
  groups.n_each = base->rows;
  groups.stride = stride;
  product(c.ctx, *queries, *base, dim, groups, out, dtype, c.stream, c.record);
}

static void grouped_device(const Caller& c, const pxc_bq_rows* queries, const int64_t* query_offsets,
                           const pxc_bq_rows* base, const int64_t* base_offsets, uint32_t groups, uint32_t dim, void* out,
                           int32_t dtype, uint64_t size) {
  check_common(dim, dtype);
  c.report();
  const uint64_t each = check_grouped(queries, query_offsets, base, base_offsets, groups, dim, out, dtype, size, true);
  DeviceGuard g(c.ctx->device);
  Groups gr{};
  gr.nq = queries->rows;
  gr.nb = base->rows;
  gr.record = c.record;
  gr.q_offsets = query_offsets;
  gr.b_offsets = base_offsets;
  gr.groups = groups;
  gr.n_each = gr.stride = each;
  gr.size = size;
  if (queries->rows == 0 || base->rows == 0 || size == 0) {
    const unsigned grid = std::min<unsigned>((groups + 255) / 256, static_cast<unsigned>(c.ctx->sm_count) * 8);
    check_empty_kernel<<<grid, 256, 0, c.stream>>>(gr);
    PXC_CUDA(cudaGetLastError());
    count_launch(c.ctx);
    return;
  }
  product(c.ctx, *queries, *base, dim, gr, out, dtype, c.stream, c.record);
}

static void check_context(const pxc_ctx* ctx) { PXC_CONFIG(ctx != nullptr, "ctx", 0, "null context"); }

}  // namespace bq
}  // namespace pxc

using namespace pxc;

extern "C" {

pxc_status pxc_bq_encode_device(pxc_ctx* ctx, const void* d_vectors, int32_t dtype, uint64_t stride, uint32_t dim,
                                const pxc_bq_rows* d_out, void* stream, pxc_error* err) {
  return guarded(err, [&] {
    bq::encode_device(bq::Caller(ctx, 0, stream, false), d_vectors, dtype, stride, dim, d_out);
  });
}

pxc_status pxc_bq_encode(pxc_ctx* ctx, const void* vectors, int32_t dtype, uint64_t stride, uint32_t dim,
                         const pxc_bq_rows* out, pxc_error* err) {
  return guarded(err, [&] {
    bq::check_context(ctx);
    bq::check_common(dim, dtype);
    bq::check_rows(out, dim, "out", false);
    if (out->rows == 0) return;
    bq::check_vectors(vectors, dtype, stride, dim, "vectors");
    std::lock_guard<std::mutex> lock(ctx->mu);
    DeviceGuard g(ctx->device);
    cudaStream_t s = ctx->stream;
    const size_t es = bq::size_of(dtype);
    DBuf<uint8_t> x;
    x.reserve(out->rows * dim * es);
    bq::Staged c;
    c.make(out->rows, dim);
    bq::copy_rows(x.p, dim * es, vectors, stride * es, dim * es, out->rows, cudaMemcpyHostToDevice, s);
    bq::encode(ctx, x.p, dtype, dim, dim, c.d, s);
    bq::copy_rows(out->codes, out->ld, c.d.codes, c.d.ld, c.d.ld, out->rows, cudaMemcpyDeviceToHost, s);
    bq::copy_rows(out->scales, out->sld, c.d.scales, c.d.sld, c.d.sld, out->rows, cudaMemcpyDeviceToHost, s);
    PXC_CUDA(cudaStreamSynchronize(s));
  });
}

pxc_status pxc_bq_decode_device(pxc_ctx* ctx, const pxc_bq_rows* d_rows, uint32_t dim, void* d_out, int32_t dtype,
                                uint64_t stride, void* stream, pxc_error* err) {
  return guarded(err, [&] {
    bq::decode_device(bq::Caller(ctx, 0, stream, false), d_rows, dim, d_out, dtype, stride);
  });
}

pxc_status pxc_bq_decode(pxc_ctx* ctx, const pxc_bq_rows* rows, uint32_t dim, void* out, int32_t dtype, uint64_t stride,
                         pxc_error* err) {
  return guarded(err, [&] {
    bq::check_context(ctx);
    bq::check_common(dim, dtype);
    bq::check_rows(rows, dim, "rows", false);
    if (rows->rows == 0) return;
    bq::check_vectors(out, dtype, stride, dim, "out");
    std::lock_guard<std::mutex> lock(ctx->mu);
    DeviceGuard g(ctx->device);
    cudaStream_t s = ctx->stream;
    const size_t es = bq::size_of(dtype);
    bq::Staged c;
    c.load(*rows, dim, s);
    DBuf<uint8_t> x;
    x.reserve(rows->rows * dim * es);
    bq::decode(ctx, c.d, dim, x.p, dtype, dim, s);
    bq::copy_rows(out, stride * es, x.p, dim * es, dim * es, rows->rows, cudaMemcpyDeviceToHost, s);
    PXC_CUDA(cudaStreamSynchronize(s));
  });
}

pxc_status pxc_bq_product_device(pxc_ctx* ctx, const pxc_bq_rows* d_queries, const pxc_bq_rows* d_base, uint32_t dim,
                                 void* d_out, int32_t dtype, uint64_t stride, void* stream, pxc_error* err) {
  return guarded(err, [&] {
    bq::product_device(bq::Caller(ctx, 0, stream, true), d_queries, d_base, dim, d_out, dtype, stride);
  });
}

pxc_status pxc_bq_product(pxc_ctx* ctx, const pxc_bq_rows* queries, const pxc_bq_rows* base, uint32_t dim, void* out,
                          int32_t dtype, uint64_t stride, pxc_error* err) {
  return guarded(err, [&] {
    bq::check_context(ctx);
    bq::check_common(dim, dtype);
    bq::check_product(queries, base, dim, out, dtype, stride, false);
    if (queries->rows == 0 || base->rows == 0) return;
    std::lock_guard<std::mutex> lock(ctx->mu);
    DeviceGuard g(ctx->device);
    const bq::Leased mine(*ctx->bq_reports);
    cudaStream_t s = ctx->stream;
    const size_t es = bq::size_of(dtype);
    bq::Staged q, b;
    q.load(*queries, dim, s);
    b.load(*base, dim, s);
    DBuf<uint8_t> o;
    o.reserve(queries->rows * base->rows * es);
    bq::Groups groups{};
    groups.groups = 1;
    groups.n_each = groups.stride = base->rows;
    bq::product(ctx, q.d, b.d, dim, groups, o.p, dtype, s, mine.record);
    bq::copy_rows(out, stride * es, o.p, base->rows * es, base->rows * es, queries->rows, cudaMemcpyDeviceToHost, s);
    PXC_CUDA(cudaStreamSynchronize(s));
    mine.record.take();
  });
}

pxc_status pxc_bq_grouped_product_device(pxc_ctx* ctx, const pxc_bq_rows* d_queries, const int64_t* d_query_offsets,
                                         const pxc_bq_rows* d_base, const int64_t* d_base_offsets, uint32_t groups,
                                         uint32_t dim, void* d_out, int32_t dtype, uint64_t size, void* stream,
                                         pxc_error* err) {
  return guarded(err, [&] {
    bq::grouped_device(bq::Caller(ctx, 0, stream, true), d_queries, d_query_offsets, d_base, d_base_offsets, groups, dim, d_out,
                       dtype, size);
  });
}

pxc_status pxc_bq_grouped_product(pxc_ctx* ctx, const pxc_bq_rows* queries, const int64_t* query_offsets,
                                  const pxc_bq_rows* base, const int64_t* base_offsets, uint32_t groups, uint32_t dim,
                                  void* out, int32_t dtype, uint64_t size, pxc_error* err) {
  return guarded(err, [&] {
    bq::check_context(ctx);
    bq::check_common(dim, dtype);
    const uint64_t each = bq::check_grouped(queries, query_offsets, base, base_offsets, groups, dim, out, dtype, size, false);
    bq::check_host_offsets(query_offsets, groups, queries->rows);
    uint64_t need = queries->rows * each;
    if (base_offsets) {
      bq::check_host_offsets(base_offsets, groups, base->rows);
      need = 0;
      for (uint32_t g = 0; g < groups; ++g) {
        need += static_cast<uint64_t>(query_offsets[g + 1] - query_offsets[g]) *
                static_cast<uint64_t>(base_offsets[g + 1] - base_offsets[g]);
        PXC_CONFIG(need <= size, "size", size, "smaller than the groups' matrices together");
      }
    }
    if (need == 0) return;
    std::lock_guard<std::mutex> lock(ctx->mu);
    DeviceGuard g(ctx->device);
    const bq::Leased mine(*ctx->bq_reports);
    cudaStream_t s = ctx->stream;
    const size_t es = bq::size_of(dtype);
    bq::Staged q, b;
    q.load(*queries, dim, s);
    b.load(*base, dim, s);
    DBuf<int64_t> off;
    off.reserve(2 * (size_t(groups) + 1));
    PXC_CUDA(cudaMemcpyAsync(off.p, query_offsets, (size_t(groups) + 1) * 8, cudaMemcpyHostToDevice, s));
    if (base_offsets)
      PXC_CUDA(cudaMemcpyAsync(off.p + groups + 1, base_offsets, (size_t(groups) + 1) * 8, cudaMemcpyHostToDevice, s));
    DBuf<uint8_t> o;
    o.reserve(need * es);
    // the even form leaves the rows of queries in no group as they were: only the others come back
    const uint64_t first = base_offsets ? 0 : static_cast<uint64_t>(query_offsets[0]) * each;
    const uint64_t count = base_offsets ? need : static_cast<uint64_t>(query_offsets[groups]) * each - first;
    bq::Groups gr{};
    gr.q_offsets = off.p;
    gr.b_offsets = base_offsets ? off.p + groups + 1 : nullptr;
    gr.groups = groups;
    gr.n_each = gr.stride = each;
    gr.size = need;
    bq::product(ctx, q.d, b.d, dim, gr, o.p, dtype, s, mine.record);
    if (count)
      PXC_CUDA(cudaMemcpyAsync(static_cast<uint8_t*>(out) + first * es, o.p + first * es, count * es,
                               cudaMemcpyDeviceToHost, s));
    PXC_CUDA(cudaStreamSynchronize(s));
    mine.record.take();
  });
}

pxc_status pxc_bq_check(pxc_ctx* ctx, void* stream, pxc_error* err) { return pxc_bq_check_as(ctx, 0, stream, err); }

uint64_t pxc_bq_callers(uint64_t count) {
  static uint64_t next = 1;
  return __atomic_fetch_add(&next, count, __ATOMIC_RELAXED);
}

pxc_status pxc_bq_forget(pxc_ctx* ctx, const uint64_t* callers, uint64_t count, pxc_error* err) {
  return guarded(err, [&] {
    bq::check_context(ctx);
    PXC_CONFIG(callers != nullptr || count == 0, "callers", 0, "null callers");
    ctx->bq_reports->forget(callers, count);
  });
}

pxc_status pxc_bq_encode_as(pxc_ctx* ctx, uint64_t caller, const void* d_vectors, int32_t dtype, uint64_t stride,
                            uint32_t dim, const pxc_bq_rows* d_out, void* stream, pxc_error* err) {
  return guarded(err, [&] {
    bq::encode_device(bq::Caller(ctx, caller, stream, false), d_vectors, dtype, stride, dim, d_out);
  });
}

pxc_status pxc_bq_decode_as(pxc_ctx* ctx, uint64_t caller, const pxc_bq_rows* d_rows, uint32_t dim, void* d_out,
                            int32_t dtype, uint64_t stride, void* stream, pxc_error* err) {
  return guarded(err, [&] {
    bq::decode_device(bq::Caller(ctx, caller, stream, false), d_rows, dim, d_out, dtype, stride);
  });
}

pxc_status pxc_bq_product_as(pxc_ctx* ctx, uint64_t caller, const pxc_bq_rows* d_queries, const pxc_bq_rows* d_base,
                             uint32_t dim, void* d_out, int32_t dtype, uint64_t stride, void* stream, pxc_error* err) {
  return guarded(err, [&] {
    bq::product_device(bq::Caller(ctx, caller, stream, true), d_queries, d_base, dim, d_out, dtype, stride);
  });
}

pxc_status pxc_bq_grouped_product_as(pxc_ctx* ctx, uint64_t caller, const pxc_bq_rows* d_queries,
                                     const int64_t* d_query_offsets, const pxc_bq_rows* d_base,
                                     const int64_t* d_base_offsets, uint32_t groups, uint32_t dim, void* d_out,
                                     int32_t dtype, uint64_t size, void* stream, pxc_error* err) {
  return guarded(err, [&] {
    bq::grouped_device(bq::Caller(ctx, caller, stream, true), d_queries, d_query_offsets, d_base, d_base_offsets, groups, dim,
                       d_out, dtype, size);
  });
}

pxc_status pxc_bq_report_as(pxc_ctx* ctx, uint64_t caller, pxc_error* err) {
  return guarded(err, [&] { bq::Caller(ctx, caller, nullptr, false).report(); });
}

pxc_status pxc_bq_check_as(pxc_ctx* ctx, uint64_t caller, void* stream, pxc_error* err) {
  return guarded(err, [&] {
    const bq::Caller c(ctx, caller, stream, false);
    DeviceGuard g(ctx->device);
    PXC_CUDA(cudaStreamSynchronize(c.stream));
    c.report();
    if (caller != 0) ctx->bq_reports->of_stream(c.stream).take();
    ctx->bq_reports->take_left();
  });
}

}  // extern "C"
