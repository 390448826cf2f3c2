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
//   1    allocates TMEM and issues the MMAs: two to eight accumulators in turn, so that a
//        tile's epilogue runs under the next tiles' MMAs;
//   2    scales: the words of four blocks (512 components) per row, copied asynchronously from
//        global to shared memory in the order tcgen05.cp wants (row 32 j + i of 128 at
//        16 i + 4 j), several copies of words ahead: a word's latency is that of HBM, and a tile
//        of one block takes 0.3 us of bandwidth;
//   3    the walk over tiles, ahead of the others;
//   4-7  epilogue, a TMEM lane quarter each.
// A scale slot, in shared memory or TMEM, is written again only after the MMAs that read it have
// completed (sf_empty), so nothing hangs on the order of copies and MMAs beyond the documented one.
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
constexpr uint32_t MAX_SF = 8;          // scale slots in shared memory
constexpr uint32_t SF_TMEM = 4;         // and in TMEM: 16 columns each (base 4, queries from 8)
constexpr uint32_t SF_COL = 2 * MAX_Q;  // the first of them
constexpr uint32_t MAX_ACC = 8;
constexpr uint32_t TILE_SLOTS = 16;  // more than stages, so that the walk never holds the loads of short tiles back
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
  uint32_t sf_slots;
  uint32_t accs, acc_cols;  // accumulators (a power of two) and the columns of each
  uint64_t wait_cycles;
};

// Shared memory behind the stages and the scale slots.
struct Control {
  TileSlot tiles[TILE_SLOTS];
  uint64_t full[MAX_STAGES], empty[MAX_STAGES];
  uint64_t sf_full[MAX_SF], sf_empty[MAX_SF];
  uint64_t acc_full[MAX_ACC], acc_empty[MAX_ACC];
  uint64_t tile_full[TILE_SLOTS], tile_empty[TILE_SLOTS];
  uint64_t done;
  uint32_t tmem;
  volatile uint32_t failed;
};

__host__ __device__ constexpr uint32_t stage_bytes(uint32_t q_rows) { return BASE_BYTES + q_rows * KB; }
// base atom, and one atom per 128 queries
__host__ __device__ constexpr uint32_t sf_bytes(uint32_t q_rows) { return 512 * (1 + (q_rows + 127) / 128); }
// Fills in the rings for tiles of up to p.q_rows queries; the bytes of shared memory.
__host__ inline uint32_t plan(Params& p) {
  // narrow tiles are short, so more of them have to be in flight
  p.sf_slots = p.q_rows <= 128 ? MAX_SF : 3;
  p.accs = p.q_rows <= 48 ? 8 : p.q_rows <= 112 ? 4 : 2;
  p.acc_cols = p.accs == 8 ? 48 : p.accs == 4 ? 112 : MAX_Q;
  const uint32_t rest = 1024 + (uint32_t)sizeof(Control) + p.sf_slots * sf_bytes(p.q_rows);
  const uint32_t fit = (SMEM_LIMIT - rest) / stage_bytes(p.q_rows);
  p.stages = fit < MAX_STAGES ? fit : MAX_STAGES;
  return rest + p.stages * stage_bytes(p.q_rows);
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

// A bounded wait of one thread: a ready barrier costs one test, and only a late one looks at the
// clock and at the CTA's failure flag. Waits are made by one lane: tests by all 32 take turns
// in the shared-memory pipe and cost every role of the CTA some 200 cycles each.
__device__ __forceinline__ bool wait_one(Control& c, uint64_t* bar, uint32_t parity, uint64_t limit) {
  if (sm100::mbar_try_wait(bar, parity)) return true;
  const uint64_t start = clock64();
  for (;;) {
    if (sm100::mbar_try_wait(bar, parity)) return true;
    if (c.failed) return false;
    if (clock64() - start > limit) {
      c.failed = 1;
      return false;
    }
  }
}
// The same for a whole warp.
__device__ __forceinline__ bool wait_warp(Control& c, uint64_t* bar, uint32_t parity, uint64_t limit) {
  bool ok = true;
  if ((threadIdx.x & 31) == 0) ok = wait_one(c, bar, parity, limit);
  return __shfl_sync(0xFFFFFFFFu, ok, 0);
}

// Four bytes to shared memory, zero where `from` has none to give; arrive() signals `bar` once
// this thread's copies so far have landed (counted by the barrier's init).
__device__ __forceinline__ void copy_word(uint32_t smem, const uint8_t* from, bool any) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem), "l"(from), "r"(any ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copies_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(sm100::smem_u32(bar)) : "memory");
}

// The next tile of the ring for one of its readers, a thread or a warp. False at the end or after
// a failure.
struct Reader {
  Control& c;
  const uint64_t limit;
  uint32_t slot = 0, ph = 0;
  __device__ __forceinline__ bool next_one(Tile& t) {
    if (!wait_one(c, &c.tile_full[slot], ph, limit)) return false;
    const bool any = c.tiles[slot].valid != 0;
    t = c.tiles[slot].tile;
    sm100::mbar_arrive(&c.tile_empty[slot]);
    step();
    return any;
  }
  __device__ __forceinline__ bool next_warp(Tile& t) {
    if (!wait_warp(c, &c.tile_full[slot], ph, limit)) return false;
    const bool any = c.tiles[slot].valid != 0;
    t = c.tiles[slot].tile;
    __syncwarp();
    if ((threadIdx.x & 31) == 0) sm100::mbar_arrive(&c.tile_empty[slot]);
    step();
    return any;
  }
  __device__ __forceinline__ void step() {
    if (++slot == TILE_SLOTS) slot = 0, ph ^= 1;
  }
};

// One lane of a converged warp, in a form from which the compiler knows that it is one: the operands of
// the tensor instructions then need no loop over lanes.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xFFFFFFFF;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one != 0;
}

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
  const uint32_t per_sf = sf_bytes(p.q_rows);
  unsigned char* sf_ring = smem + static_cast<size_t>(stages) * per_stage;
  Control& c = *reinterpret_cast<Control*>(sf_ring + static_cast<size_t>(p.sf_slots) * per_sf);
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (warp == 1) {
    tmem_alloc<512>(&c.tmem);
    tmem_relinquish();
  }
  if (threadIdx.x == 0) {
    c.failed = 0;
    for (uint32_t s = 0; s < stages; ++s) mbar_init(&c.full[s], 1), mbar_init(&c.empty[s], 1);
    for (uint32_t s = 0; s < p.sf_slots; ++s) mbar_init(&c.sf_full[s], 32), mbar_init(&c.sf_empty[s], 1);
    for (uint32_t s = 0; s < p.accs; ++s) mbar_init(&c.acc_full[s], 1), mbar_init(&c.acc_empty[s], 4);
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

  const uint64_t limit = p.wait_cycles;
  Reader reader{c, limit};
  Tile t;

  if (warp == 0) {
    // ---- producer ----
    if (elect_one()) {
      uint32_t issued = 0, s = 0, ph = 0;
      bool ok = true;
      while (ok && reader.next_one(t)) {
        const uint32_t boxes = (round16(t.queries) + p.q_box - 1) / p.q_box;
        const uint32_t bytes = BASE_BYTES + boxes * p.q_box * KB;
        for (uint32_t kb = 0; kb < kblocks; ++kb) {
          if (!(ok = wait_one(c, &c.empty[s], ph ^ 1, limit))) break;
          unsigned char* dst = smem + static_cast<size_t>(s) * per_stage;
          mbar_arrive_expect_tx(&c.full[s], bytes);
          tma_load_2d(dst, &map_b, &c.full[s], kb * KB, t.b0);
          for (uint32_t i = 0; i < boxes; ++i)
            tma_load_2d(dst + BASE_BYTES + i * p.q_box * KB, &map_q, &c.full[s], kb * KB, t.q0 + i * p.q_box);
          ++issued;
          if (++s == stages) s = 0, ph ^= 1;
        }
      }
      // every copy has landed before the CTA exits: the last use of each stage, oldest first
      for (uint32_t j = issued > stages ? issued - stages : 0; j < issued; ++j) {
        const uint64_t start = clock64();
        while (!mbar_try_wait(&c.full[j % stages], (j / stages) & 1) && clock64() - start <= limit) {
        }
      }
    }
  } else if (warp == 1) {
    // ---- MMA ----
    if (elect_one()) {
      uint32_t s = 0, ph = 0;                // stage ring
      uint32_t quad = 0, sf = 0, sf_ph = 0;  // scale words: number, slot
      uint32_t acc = 0, acc_ph = 0;
      bool ok = true;
      const uint32_t base = smem_u32(smem), sf_base = smem_u32(sf_ring);
      const uint32_t last_steps = (p.dim - (kblocks - 1) * KB + MMA_K - 1) / MMA_K;
      while (ok && reader.next_one(t)) {
        const uint32_t width = round16(t.queries);
        if (!(ok = wait_one(c, &c.acc_empty[acc], acc_ph ^ 1, limit))) break;
        tc_fence_after();
        const uint32_t d = tmem + acc * p.acc_cols;
        for (uint32_t kb = 0; kb < kblocks; ++kb) {
          const uint32_t sfa = tmem + SF_COL + (quad % SF_TMEM) * 16, sfb = sfa + 8;
          if ((kb & 3) == 0) {
            if (!(ok = wait_one(c, &c.sf_full[sf], sf_ph, limit))) break;
            if (p.sf_slots > SF_TMEM && quad >= SF_TMEM) {
              // the words SF_TMEM before, in the same TMEM columns, are done with
              const uint32_t old = quad - SF_TMEM;
              if (!(ok = wait_one(c, &c.sf_empty[old % MAX_SF], (old / MAX_SF) & 1, limit))) break;
            }
            fence_proxy_async();  // the words came by generic copies
            tc_fence_after();
            const uint32_t from = sf_base + sf * per_sf;
            copy_scales(sfa, from);
            copy_scales(sfb, from + 512);
            if (width > 128) copy_scales(sfb + 4, from + 1024);
          }
          if (!(ok = wait_one(c, &c.full[s], ph, limit))) break;
          tc_fence_after();
          const uint64_t a = smem_desc_k_sw128(base + s * per_stage);
          const uint64_t b = smem_desc_k_sw128(base + s * per_stage + BASE_BYTES);
          const uint32_t idesc = idesc_mxf8(width, kb & 3);
          const uint32_t steps = kb + 1 == kblocks ? last_steps : KB / MMA_K;
#pragma unroll
          for (uint32_t k = 0; k < KB / MMA_K; ++k)
            if (k < steps) mma_mxf8(d, a + 2 * k, b + 2 * k, idesc, sfa, sfb, (kb | k) != 0);
          mma_commit(&c.empty[s]);
          if (++s == stages) s = 0, ph ^= 1;
          if ((kb & 3) == 3 || kb + 1 == kblocks) {
            mma_commit(&c.sf_empty[sf]);
            ++quad;
            if (++sf == p.sf_slots) sf = 0, sf_ph ^= 1;
          }
        }
        if (!ok) break;
        mma_commit(&c.acc_full[acc]);
        if (++acc == p.accs) acc = 0, acc_ph ^= 1;
      }
      // all MMAs complete before TMEM is released
      mma_commit(&c.done);
      const uint64_t start = clock64();
      while (!mbar_try_wait(&c.done, 0) && clock64() - start <= limit) {
      }
    }
  } else if (warp == 2) {
    // ---- scales ----
    uint32_t sf = 0, sf_ph = 0;
    bool ok = true;
    while (ok && reader.next_warp(t)) {
      const uint32_t words = (kblocks + 3) / 4, columns = (t.queries + 31) / 32;
      for (uint32_t w = 0; w < words; ++w) {
        if (!(ok = wait_warp(c, &c.sf_empty[sf], sf_ph ^ 1, limit))) break;
        const uint32_t to = smem_u32(sf_ring) + sf * per_sf + lane * 16;
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
          const uint64_t r = static_cast<uint64_t>(t.b0) + 32 * j + lane;
          const bool any = r < p.groups.nb;
          copy_word(to + 4 * j, p.b_scales + (any ? r * p.b_sld + 4 * w : 0), any);
        }
        for (uint32_t j = 0; j < columns; ++j) {
          const uint64_t r = static_cast<uint64_t>(t.q0) + 32 * j + lane;
          const bool any = r < p.groups.nq;
          copy_word(to + 512 * (1 + j / 4) + 4 * (j & 3), p.q_scales + (any ? r * p.q_sld + 4 * w : 0), any);
        }
        copies_arrive(&c.sf_full[sf]);
        if (++sf == p.sf_slots) sf = 0, sf_ph ^= 1;
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");  // landed before the CTA exits
  } else if (warp == 3) {
    // ---- the walk over tiles ----
    Walk<MAX_Q, BM> walk(p.groups, lane);
    uint32_t s = 0, ph = 0;
    for (uint64_t k = blockIdx.x;; k += gridDim.x) {
      const bool any = walk.find(k, t);
      if (!wait_warp(c, &c.tile_empty[s], ph ^ 1, limit)) break;
      if (lane == 0) {
        c.tiles[s].tile = t;
        c.tiles[s].valid = any;
        mbar_arrive(&c.tile_full[s]);
      }
      if (!any) break;
      if (++s == TILE_SLOTS) s = 0, ph ^= 1;
    }
  } else {
    // ---- epilogue ----
    const uint32_t quarter = warp & 3, row = quarter * 32 + lane;
    T* out = static_cast<T*>(p.out);
    uint32_t acc = 0, acc_ph = 0;
    while (reader.next_warp(t)) {
      if (!wait_warp(c, &c.acc_full[acc], acc_ph, limit)) break;
      tc_fence_after();
      const uint32_t addr = tmem + ((quarter * 32) << 16) + acc * p.acc_cols;
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
      if (++acc == p.accs) acc = 0, acc_ph ^= 1;
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc<512>(tmem);
  if (threadIdx.x == 0 && c.failed) leave_fault(p.groups.faults, FAULT_TIMEOUT);
}

}  // namespace bq_tc
}  // namespace pxc
