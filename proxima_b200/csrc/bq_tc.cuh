// bq_tc.cuh — the block product on tcgen05 tensor cores (kind::mxf8f6f4, block scales in TMEM).
//
//   out[q][r] = sum over blocks j of 2^(s_qj + s_rj) * sum over i in j of c_qi * c_ri
//
// The instruction multiplies 32 components at a time and scales them by one E8M0 byte per row of
// either operand, inside the f32 accumulation. A block of 128 is four such steps with the
// same byte, so the power-of-two scales cost no pass over the accumulators: a tile's whole sum
// over the dimension stays in TMEM.
//
// The base rows are the M side (128 per tile, a TMEM lane each) and the queries the N side (16 to
// MAX_Q columns in steps of 16). One query then costs a 16-column tile and not a padded 128-row
// one, and a lane holds one base row, so that a warp's stores of a column are 32
// consecutive outputs.
//
// One persistent CTA per SM; roles by warp:
//   0    TMA producer: 128 bytes x 128 base rows and x the tile's queries per stage, 128-byte
//        swizzle, through a ring of as many stages as fit;
//   1    allocates TMEM and issues the MMAs: two accumulators of MAX_Q columns in turn, so
//        that a tile's epilogue runs under the next tile's MMAs;
//   2    scales: the words of four blocks (512 components) per row go from global memory through
//        registers to shared memory in the order tcgen05.cp wants (row 32 j + i of 128 at
//        16 i + 4 j); the next words are in flight while the current ones are multiplied;
//   3    the walk over tiles, a few ahead of the others;
//   4-7  epilogue, a TMEM lane quarter each.
// A scale slot in TMEM is written again only after the MMAs that read it have completed
// (sf_empty), so nothing hangs on the order of copies and MMAs beyond the documented one.
// Every wait is bounded; when one runs out the CTA leaves FAULT_TIMEOUT, drains its copies and
// MMAs, frees TMEM and returns.
#pragma once
#include "bq.cuh"
#include "sm100.cuh"

namespace pxc {
namespace bq_tc {

using namespace bq;

constexpr uint32_t BM = 128;     // base rows per tile
constexpr uint32_t MAX_Q = 224;  // queries per tile: 2 x 224 accumulator columns and the scales fit 512
constexpr uint32_t KB = 128;     // bytes of the dimension per stage: one scale block, one swizzle atom
constexpr uint32_t MMA_K = 32;
constexpr uint32_t THREADS = 256;
constexpr uint32_t BASE_BYTES = BM * KB;
constexpr uint32_t SF_SLOTS = 2;
constexpr uint32_t SF_BYTES = 3 * 512;  // base atom, two query atoms
constexpr uint32_t SF_COL = 2 * MAX_Q;  // TMEM columns of the scales: 16 per slot (base 4, queries from 8)
constexpr uint32_t TILE_SLOTS = 4;
constexpr uint32_t SMEM_LIMIT = 227 * 1024;
constexpr uint32_t MAX_STAGES = 12;

struct TileSlot {
  Tile tile;
  uint32_t valid;
  uint32_t pad;
};

struct Params {
  Groups groups;
  const uint8_t* q_scales;
  const uint8_t* b_scales;
  uint64_t q_sld, b_sld;
  void* out;
  uint32_t dim, kblocks;
  uint32_t stages;
  uint32_t q_rows;  // queries that a stage has room for: a multiple of 16
  uint32_t q_box;   // queries per TMA box
  uint64_t wait_ns;
};

// Shared memory behind the stages.
struct Control {
  unsigned char sf[SF_SLOTS][SF_BYTES];
  TileSlot tiles[TILE_SLOTS];
  uint64_t full[MAX_STAGES], empty[MAX_STAGES];
  uint64_t sf_full[SF_SLOTS], sf_empty[SF_SLOTS];
  uint64_t acc_full[2], acc_empty[2];
  uint64_t tile_full[TILE_SLOTS], tile_empty[TILE_SLOTS];
  uint64_t done;
  uint32_t tmem;
  volatile uint32_t failed;
};

__host__ __device__ constexpr uint32_t stage_bytes(uint32_t q_rows) { return BASE_BYTES + q_rows * KB; }
__host__ inline uint32_t pick_stages(uint32_t q_rows) {
  const uint32_t s = (SMEM_LIMIT - 1024 - (uint32_t)sizeof(Control)) / stage_bytes(q_rows);
  return s < MAX_STAGES ? s : MAX_STAGES;
}
__host__ inline uint32_t smem_bytes(uint32_t q_rows, uint32_t stages) {
  return stages * stage_bytes(q_rows) + (uint32_t)sizeof(Control) + 1024;
}

// ---- tcgen05 forms of this kernel ----
// e4m3 x e4m3 -> f32, E8M0 scales, both K-major; `sf` picks the byte of the scale words.
__device__ __forceinline__ uint32_t idesc_mxf8(uint32_t n, uint32_t sf) {
  return (sf << 4) | ((n >> 3) << 17) | (1u << 23) | ((BM >> 4) << 24) | (sf << 29);
}
__device__ __forceinline__ void mma_mxf8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                         uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}
// 32 rows of 16 bytes of shared memory (8-row groups 128 bytes apart, no swizzle) to four TMEM
// columns, the same in each quarter of the lanes.
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint32_t smem) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem >> 4) & 0x3FFFu);
  d |= static_cast<uint64_t>(128u >> 4) << 32;  // SBO
  d |= static_cast<uint64_t>(1u) << 46;         // descriptor version (sm100)
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(d) : "memory");
}

// The next tile of the ring for one of its readers (a warp). False at the end or after a failure.
struct Reader {
  Control& c;
  const uint64_t wait_ns;
  uint32_t i = 0;
  __device__ __forceinline__ bool next(Tile& t) {
    const uint32_t s = i % TILE_SLOTS, ph = (i / TILE_SLOTS) & 1;
    if (!__all_sync(0xFFFFFFFFu, sm100::mbar_wait(&c.tile_full[s], ph, wait_ns) && !c.failed)) {
      c.failed = 1;
      return false;
    }
    const bool any = c.tiles[s].valid != 0;
    t = c.tiles[s].tile;
    __syncwarp();
    if ((threadIdx.x & 31) == 0) sm100::mbar_arrive(&c.tile_empty[s]);
    ++i;
    return any;
  }
};

__device__ __forceinline__ uint32_t round16(uint32_t x) { return (x + 15) & ~15u; }

template <class T>
__global__ void __launch_bounds__(THREADS, 1)
    product_kernel(const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_q,
                   const __grid_constant__ Params p) {
  using namespace sm100;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t stages = p.stages, kblocks = p.kblocks;
  const uint32_t per_stage = stage_bytes(p.q_rows);
  Control& c = *reinterpret_cast<Control*>(smem + static_cast<size_t>(stages) * per_stage);
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (warp == 1) {
    tmem_alloc<512>(&c.tmem);
    tmem_relinquish();
  }
  if (threadIdx.x == 0) {
    c.failed = 0;
    for (uint32_t s = 0; s < stages; ++s) mbar_init(&c.full[s], 1), mbar_init(&c.empty[s], 1);
    for (uint32_t s = 0; s < SF_SLOTS; ++s) mbar_init(&c.sf_full[s], 1), mbar_init(&c.sf_empty[s], 1);
    for (uint32_t s = 0; s < 2; ++s) mbar_init(&c.acc_full[s], 1), mbar_init(&c.acc_empty[s], 4);
    // readers of a tile: the producer, the MMA warp, the scales, four epilogue warps
    for (uint32_t s = 0; s < TILE_SLOTS; ++s) mbar_init(&c.tile_full[s], 1), mbar_init(&c.tile_empty[s], 7);
    mbar_init(&c.done, 1);
    fence_barrier_init();
    tma_prefetch_desc(&map_b);
    tma_prefetch_desc(&map_q);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = c.tmem;

  // A bounded wait of a whole warp; on expiry the CTA's failure flag goes up.
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    const bool ok = __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity, p.wait_ns) && !c.failed);
    if (!ok) c.failed = 1;
    return ok;
  };
  Reader reader{c, p.wait_ns};
  Tile t;

  if (warp == 0) {
    // ---- producer ----
    uint32_t it = 0;
    bool ok = true;
    while (ok && reader.next(t)) {
      const uint32_t boxes = (round16(t.queries) + p.q_box - 1) / p.q_box;
      for (uint32_t kb = 0; kb < kblocks; ++kb, ++it) {
        const uint32_t s = it % stages;
        if (!(ok = wait(&c.empty[s], ((it / stages) & 1) ^ 1))) break;
        if (lane == 0) {
          unsigned char* dst = smem + static_cast<size_t>(s) * per_stage;
          mbar_arrive_expect_tx(&c.full[s], BASE_BYTES + boxes * p.q_box * KB);
          tma_load_2d(dst, &map_b, &c.full[s], kb * KB, t.b0);
          for (uint32_t i = 0; i < boxes; ++i)
            tma_load_2d(dst + BASE_BYTES + i * p.q_box * KB, &map_q, &c.full[s], kb * KB, t.q0 + i * p.q_box);
        }
        __syncwarp();
      }
    }
    // every copy has landed before the CTA exits
    for (uint32_t j = it > stages ? it - stages : 0; j < it; ++j)
      mbar_wait(&c.full[j % stages], (j / stages) & 1, p.wait_ns);
  } else if (warp == 1) {
    // ---- MMA ----
    uint32_t it = 0, quad = 0, n = 0;
    bool ok = true;
    const uint32_t base = smem_u32(smem), sf_smem = smem_u32(c.sf);
    while (ok && reader.next(t)) {
      const uint32_t acc = n & 1, width = round16(t.queries);
      if (!(ok = wait(&c.acc_empty[acc], ((n >> 1) & 1) ^ 1))) break;
      tc_fence_after();
      const uint32_t d = tmem + acc * MAX_Q;
      for (uint32_t kb = 0; kb < kblocks; ++kb, ++it) {
        const uint32_t s = it % stages, slot = quad % SF_SLOTS;
        const uint32_t sfa = tmem + SF_COL + slot * 16, sfb = sfa + 8;
        if ((kb & 3) == 0) {
          if (!(ok = wait(&c.sf_full[slot], (quad / SF_SLOTS) & 1))) break;
          if (lane == 0) {
            tc_fence_after();
            copy_scales(sfa, sf_smem + slot * SF_BYTES);
            copy_scales(sfb, sf_smem + slot * SF_BYTES + 512);
            if (width > 128) copy_scales(sfb + 4, sf_smem + slot * SF_BYTES + 1024);
          }
          __syncwarp();
        }
        if (!(ok = wait(&c.full[s], (it / stages) & 1))) break;
        tc_fence_after();
        if (lane == 0) {
          const uint64_t a = smem_desc_k_sw128(base + s * per_stage);
          const uint64_t b = smem_desc_k_sw128(base + s * per_stage + BASE_BYTES);
          const uint32_t idesc = idesc_mxf8(width, kb & 3);
          const uint32_t steps = min((p.dim - kb * KB + MMA_K - 1) / MMA_K, KB / MMA_K);
          for (uint32_t k = 0; k < steps; ++k) mma_mxf8(d, a + 2 * k, b + 2 * k, idesc, sfa, sfb, (kb | k) != 0);
          mma_commit(&c.empty[s]);
          if ((kb & 3) == 3 || kb + 1 == kblocks) mma_commit(&c.sf_empty[slot]);
          if (kb + 1 == kblocks) mma_commit(&c.acc_full[acc]);
        }
        __syncwarp();
        if ((kb & 3) == 3 || kb + 1 == kblocks) ++quad;
      }
      ++n;
    }
    if (lane == 0) mma_commit(&c.done);
    __syncwarp();
    mbar_wait(&c.done, 0, p.wait_ns);
  } else if (warp == 2) {
    // ---- scales ----
    uint32_t quad = 0;
    bool ok = true;
    while (ok && reader.next(t)) {
      const uint32_t groups4 = (kblocks + 3) / 4;
      for (uint32_t g = 0; g < groups4; ++g, ++quad) {
        uint32_t w[12];
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
          const uint64_t r = static_cast<uint64_t>(t.b0) + 32 * j + lane;
          w[j] = r < p.groups.nb ? __ldg(reinterpret_cast<const uint32_t*>(p.b_scales + r * p.b_sld) + g) : 0u;
        }
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
          const uint64_t r = static_cast<uint64_t>(t.q0) + 32 * j + lane;
          w[4 + j] = 32 * j < t.queries && r < p.groups.nq
                         ? __ldg(reinterpret_cast<const uint32_t*>(p.q_scales + r * p.q_sld) + g)
                         : 0u;
        }
        const uint32_t slot = quad % SF_SLOTS;
        if (!(ok = wait(&c.sf_empty[slot], ((quad / SF_SLOTS) & 1) ^ 1))) break;
        uint4* dst = reinterpret_cast<uint4*>(c.sf[slot]) + lane;
#pragma unroll
        for (uint32_t a = 0; a < 3; ++a) dst[a * 32] = make_uint4(w[4 * a], w[4 * a + 1], w[4 * a + 2], w[4 * a + 3]);
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&c.sf_full[slot]);
      }
    }
  } else if (warp == 3) {
    // ---- the walk over tiles ----
    Walk<MAX_Q, BM> walk(p.groups, lane);
    uint32_t i = 0;
    for (uint64_t k = blockIdx.x;; k += gridDim.x, ++i) {
      const bool any = walk.find(k, t);
      const uint32_t s = i % TILE_SLOTS;
      if (!wait(&c.tile_empty[s], ((i / TILE_SLOTS) & 1) ^ 1)) break;
      if (lane == 0) {
        c.tiles[s].tile = t;
        c.tiles[s].valid = any;
        mbar_arrive(&c.tile_full[s]);
      }
      __syncwarp();
      if (!any) break;
    }
  } else {
    // ---- epilogue ----
    const uint32_t quarter = warp & 3, row = quarter * 32 + lane;
    T* out = static_cast<T*>(p.out);
    uint32_t n = 0;
    while (reader.next(t)) {
      const uint32_t acc = n & 1;
      if (!wait(&c.acc_full[acc], (n >> 1) & 1)) break;
      tc_fence_after();
      const uint32_t addr = tmem + ((quarter * 32) << 16) + acc * MAX_Q;
      const bool mine = row < t.rows;
      T* dst = out + t.at + row;
      for (uint32_t q = 0; q < t.queries; q += 32) {
        uint32_t v[32];
        tmem_ld_32x32b_x32(addr + q, v);
        tmem_ld_wait();
        if (mine) {
#pragma unroll
          for (uint32_t j = 0; j < 32; ++j) {
            if (q + j < t.queries) *dst = from_f32<T>(__uint_as_float(v[j]));
            dst += t.stride;
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&c.acc_empty[acc]);
      ++n;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc<512>(tmem);
  if (threadIdx.x == 0 && c.failed) leave_fault(p.groups.faults, FAULT_TIMEOUT);
}

}  // namespace bq_tc
}  // namespace pxc
