// bq_tc.cuh — the block product on tcgen05 tensor cores (kind::mxf8f6f4, block scales in TMEM).
//
//   out[q][r] = sum over blocks j of 2^(s_qj + s_rj) * sum over i in j of c_qi * c_ri
//
// The instruction multiplies 32 components at a time and scales them by one E8M0 byte per row of
// either operand, inside the f32 accumulation. A block of 128 is four such steps with the
// same byte, so the power-of-two scales cost no pass over the accumulators: a tile's whole sum
// over the dimension stays in TMEM.
//
// The base rows are the M side (a TMEM lane each) and the queries the N side (16 to MAX_Q columns
// in steps of 16). One query then costs a 16-column tile and not a padded 128-row one, and a
// lane holds one base row, so that a warp's stores of a column are 32 consecutive outputs.
//
// One persistent CTA per SM; roles by warp:
//   0    TMA producer: 128 bytes x the tile's base rows and queries per stage, 128-byte swizzle,
//        through a ring of as many stages as fit;
//   1    allocates TMEM and issues the MMAs into a ring of accumulators, so that a tile's
//        epilogue runs under the next tiles' MMAs;
//   2    scales: the words of four blocks (512 components) per row, copied asynchronously from
//        global to shared memory in the order tcgen05.cp wants (row 32 j + i of 128 at
//        16 i + 4 j), several copies of words ahead: a word's latency is that of HBM, and a tile
//        of one block takes 0.3 us of bandwidth;
//   3    the walk over tiles, ahead of the others;
//   4-11 epilogue: a TMEM lane quarter and every other 32 columns each. Two warps per scheduler
//        and four address chains: with one, the stores' addresses bound tiles of few blocks.
//
// Three shapes of tile, by what bounds the product:
//   - up to MAX_Q queries x 128 rows;
//   - narrow (few queries, many rows): 128 * subs rows per tile, so that the waits and commits of
//     a tile, some 1,000 cycles, are spent once for `subs` times 16 KB of rows;
//   - PAIR (many queries): two CTAs of a cluster work on 256 rows x the queries as one
//     (cta_group::2). Each brings its 128 rows and half of the queries, so that a stage reads and
//     writes a third less shared memory and L2 for the same products.
//
// A scale slot, in shared memory or TMEM, is written again only after the MMAs that read it have
// completed (sf_empty), so nothing hangs on the order of copies and MMAs beyond the documented one.
// Every wait is bounded. When one runs out, the CTA (of a pair: both) stops, waits for its copies and
// MMAs in flight, leaves FAULT_TIMEOUT, frees TMEM and returns. Both CTAs of a pair count their copies
// on the leader's barriers, and after a failure they may have stopped at different stages: the
// leader makes up the share of each stage that never comes and waits for the one that does (drain()).
#pragma once
#include "bq.cuh"
#include "sm100.cuh"

namespace pxc {
namespace bq_tc {

using namespace bq;

constexpr uint32_t BM = 128;     // base rows per accumulator: the TMEM lanes
constexpr uint32_t MAX_Q = 224;  // queries per tile: 2 x 224 accumulator columns and the scales fit 512
constexpr uint32_t KB = 128;     // bytes of the dimension per stage: one scale block, one swizzle atom
constexpr uint32_t MMA_K = 32;
constexpr uint32_t EPI_WARPS = 8;
constexpr uint32_t THREADS = 32 * (4 + EPI_WARPS);
constexpr uint32_t BASE_BYTES = BM * KB;
constexpr uint32_t ATOM = 512;     // scale words of 128 rows: 4 TMEM columns
constexpr uint32_t MAX_SF = 8;     // scale slots in shared memory
constexpr uint32_t SF_TMEM = 4;    // and in TMEM
constexpr uint32_t MAX_ACC = 8;
constexpr uint32_t TMEM_COLS = 512;
constexpr uint32_t TILE_SLOTS = 16;  // more than stages, so that the walk never holds the loads of short tiles back
constexpr uint32_t SMEM_LIMIT = 227 * 1024;
constexpr uint32_t MAX_STAGES = 12;
// For copies and MMAs in flight, which end by themselves: not the caller's limit, or a short one would
// let a CTA go before them.
constexpr uint64_t DRAIN_CYCLES = 2000000000;

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
  uint64_t wait_cycles;
  uint32_t dim, kblocks;
  uint32_t tile_q;     // the most queries of a tile
  uint32_t tile_log2;  // log2 of its base rows: BM * subs, or 2 * BM for a pair
  uint32_t subs;       // accumulators of a tile in this CTA
  uint32_t q_rows;     // queries of the widest tile, a multiple of 16
  uint32_t q_load;     // and those of them that a stage of this CTA has room for
  uint32_t q_box;      // queries per TMA box
  uint32_t stages, sf_slots;
  uint32_t accs, acc_cols;  // accumulators and the TMEM columns of one (of all its subs)
  uint32_t sf_col, sf_cols; // the first TMEM column of the scales, and the columns of a slot
};

// Shared memory behind the stages and the scale slots.
struct Control {
  TileSlot tiles[TILE_SLOTS];
  uint64_t full[MAX_STAGES], empty[MAX_STAGES];
  uint64_t sf_full[MAX_SF], sf_peer[MAX_SF], sf_empty[MAX_SF];
  uint64_t acc_full[MAX_ACC], acc_empty[MAX_ACC];
  uint64_t tile_full[TILE_SLOTS], tile_empty[TILE_SLOTS];
  uint64_t done;
  uint32_t tmem;
  volatile uint32_t failed;
  uint32_t peer_failed;  // of a pair: the cluster address of the other CTA's `failed`
  uint32_t issued, loaded[MAX_STAGES];  // stages that the producer filled, and the bytes of each slot's last
};

__host__ __device__ inline uint32_t q_atoms(const Params& p) { return (p.q_rows + 127) / 128; }
__host__ __device__ inline uint32_t stage_bytes(const Params& p) { return p.subs * BASE_BYTES + p.q_load * KB; }
__host__ __device__ inline uint32_t sf_bytes(const Params& p) { return ATOM * (p.subs + q_atoms(p)); }

// Fills in the rings for tiles of p.q_rows queries; the bytes of shared memory.
__host__ inline uint32_t plan(Params& p) {
  p.sf_cols = (4 * (p.subs + q_atoms(p)) + 7) / 8 * 8;
  p.sf_col = TMEM_COLS - SF_TMEM * p.sf_cols;
  p.acc_cols = p.subs * p.q_rows;
  p.accs = p.sf_col / p.acc_cols < MAX_ACC ? p.sf_col / p.acc_cols : MAX_ACC;
  // stages first, then as many scale slots as still fit: their words come from far, and a pair's second
  // CTA announces its own with a round trip more
  const uint32_t fixed = 1024 + (uint32_t)sizeof(Control), stage = stage_bytes(p), slot = sf_bytes(p);
  const uint32_t least = p.q_rows <= 128 ? MAX_SF : 3;
  const uint32_t fit = (SMEM_LIMIT - fixed - least * slot) / stage;
  p.stages = fit < MAX_STAGES ? fit : MAX_STAGES;
  const uint32_t slots = (SMEM_LIMIT - fixed - p.stages * stage) / slot;
  p.sf_slots = slots < MAX_SF ? slots : MAX_SF;
  return fixed + p.sf_slots * slot + p.stages * stage;
}

// ---- tcgen05 forms of this kernel; G is the CTA group ----
// e4m3 x e4m3 -> f32, E8M0 scales, both K-major; `sf` picks the byte of the scale words.
__device__ __forceinline__ uint32_t idesc_mxf8(uint32_t m, uint32_t n, uint32_t sf) {
  return (sf << 4) | ((n >> 3) << 17) | (1u << 23) | ((m >> 4) << 24) | (sf << 29);
}
template <int G>
__device__ __forceinline__ void mma_mxf8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                         uint32_t accumulate) {
  if constexpr (G == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}
// 32 rows of 16 bytes of shared memory (8-row groups 128 bytes apart, no swizzle) to four TMEM
// columns, the same in each quarter of the lanes. As a pair: in both CTAs, each from its own.
template <int G>
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint32_t smem) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem >> 4) & 0x3FFFu);
  d |= static_cast<uint64_t>(128u >> 4) << 32;  // SBO
  d |= static_cast<uint64_t>(1u) << 46;         // descriptor version (sm100)
  if constexpr (G == 1)
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(d) : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(d) : "memory");
}
// Signals `bar`, as a pair in both CTAs, once this thread's MMAs and copies so far have completed.
template <int G>
__device__ __forceinline__ void commit(uint64_t* bar) {
  if constexpr (G == 1)
    sm100::mma_commit(bar);
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            sm100::smem_u32(bar)),
        "h"(static_cast<uint16_t>(3))
        : "memory");
}
template <int G>
__device__ __forceinline__ void tmem_alloc(uint32_t* slot) {
  if constexpr (G == 1) {
    sm100::tmem_alloc<TMEM_COLS>(slot);
    sm100::tmem_relinquish();
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(sm100::smem_u32(slot)),
                 "r"(TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
}
template <int G>
__device__ __forceinline__ void tmem_free(uint32_t tmem) {
  if constexpr (G == 1)
    sm100::tmem_dealloc<TMEM_COLS>(tmem);
  else
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
}

// ---- the pair's other CTA ----
// The cluster address of a barrier of the leader (rank 0).
__device__ __forceinline__ uint32_t leaders(uint64_t* bar) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(sm100::smem_u32(bar)));
  return a;
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// An arrival that carries nothing but itself: a release would wait for the output stores before it.
__device__ __forceinline__ void arrive_relaxed(uint64_t* bar) {
  asm volatile("mbarrier.arrive.relaxed.cta.shared::cta.b64 _, [%0];" ::"r"(sm100::smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void arrive_cluster_relaxed(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ uint32_t in_peer(const volatile void* here, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
               : "=r"(a)
               : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(const_cast<const void*>(here)))), "r"(rank ^ 1));
  return a;
}
__device__ __forceinline__ uint32_t load_cluster(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}
// Bytes that no copy will bring, counted as arrived.
__device__ __forceinline__ void complete_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(sm100::smem_u32(bar)), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// A tile into this CTA's shared memory, counted on a barrier of either CTA of the pair.
__device__ __forceinline__ void tma_load_pair(void* dst, const CUtensorMap* map, uint32_t bar, int32_t x, int32_t y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(sm100::smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y)
      : "memory");
}

// ---- waits ----
// PEER: a barrier that threads of the other CTA of a pair arrive on. Its wider scope costs, so the others do
// without.
template <bool PEER>
__device__ __forceinline__ bool try_wait(uint64_t* bar, uint32_t parity) {
  if constexpr (!PEER) {
    return sm100::mbar_try_wait(bar, parity);
  } else {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(sm100::smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
  }
}
// Stops this CTA's roles at their next late wait, and the other CTA's of a pair.
template <bool PAIR>
__device__ __forceinline__ void fail(Control& c) {
  c.failed = 1;
  if constexpr (PAIR) asm volatile("st.relaxed.cluster.shared::cluster.u32 [%0], 1;" ::"r"(c.peer_failed) : "memory");
}
// A bounded wait of one thread: a ready barrier costs one test, and only a late one looks at the
// clock and at the CTA's failure flag. Waits are made by one lane: tests by all 32 take turns
// in the shared-memory pipe and cost every role of the CTA some 200 cycles each.
template <bool PAIR, bool PEER = false>
__device__ __forceinline__ bool wait_one(Control& c, uint64_t* bar, uint32_t parity, uint64_t limit) {
  if (try_wait<PEER>(bar, parity)) return true;
  const uint64_t start = clock64();
  for (;;) {
    if (try_wait<PEER>(bar, parity)) return true;
    if (c.failed) return false;
    if (clock64() - start > limit) {
      fail<PAIR>(c);
      return false;
    }
  }
}
// The same for a whole warp. A shuffle orders no memory: what the barrier's signal makes visible to the waiting
// lane is so for the others behind the warp's barrier.
template <bool PAIR>
__device__ __forceinline__ bool wait_warp(Control& c, uint64_t* bar, uint32_t parity, uint64_t limit) {
  bool ok = true;
  if ((threadIdx.x & 31) == 0) ok = wait_one<PAIR>(c, bar, parity, limit);
  ok = __shfl_sync(0xFFFFFFFFu, ok, 0);
  __syncwarp();
  return ok;
}
// Before the CTA ends, regardless of failures: for what is in flight, at the latest DRAIN_CYCLES after `start`.
__device__ __forceinline__ void wait_drained(uint64_t* bar, uint32_t parity, uint64_t start) {
  while (!try_wait<false>(bar, parity) && clock64() - start <= DRAIN_CYCLES) {
  }
}
// After a failure, by one thread of the CTA (of a pair: of the leader, once both CTAs' roles have ended): waits
// until every copy that was issued has landed. The last use of each slot, oldest first; earlier ones have been waited
// for, since a slot is filled again only after its MMAs. Of a pair, either producer may be up to a
// ring ahead of the other. Where only the leader filled a stage, the half that it expects of
// the other is made up; where only the other did, its half alone is expected.
template <bool PAIR>
__device__ __forceinline__ void drain(Control& c, uint32_t stages) {
  const uint64_t start = clock64();
  const uint32_t mine = c.issued, theirs = PAIR ? load_cluster(in_peer(&c.issued, 0)) : mine;
  const uint32_t most = max(mine, theirs);
  for (uint32_t j = most > stages ? most - stages : 0; j < most; ++j) {
    const uint32_t i = j % stages;
    if (PAIR && j >= theirs)
      complete_tx(&c.full[i], c.loaded[i]);
    else if (PAIR && j >= mine)
      sm100::mbar_arrive_expect_tx(&c.full[i], load_cluster(in_peer(&c.loaded[i], 0)));
    wait_drained(&c.full[i], (j / stages) & 1, start);
  }
}

// Four bytes to shared memory, zero where `from` has none to give; copies_arrive() signals `bar`
// once this thread's copies so far have landed (counted by the barrier's init).
__device__ __forceinline__ void copy_word(uint32_t smem, const uint8_t* from, bool any) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem), "l"(from), "r"(any ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copies_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(sm100::smem_u32(bar)) : "memory");
}

// A place in a ring of `n` slots and the parity of its current round.
struct Ring {
  uint32_t i = 0, ph = 0;
  __device__ __forceinline__ void step(uint32_t n) {
    if (++i == n) i = 0, ph ^= 1;
  }
};

// The next tile of the ring for one of its readers, a thread or a warp. False at the end or after
// a failure.
template <bool PAIR>
struct Reader {
  Control& c;
  const uint64_t limit;
  Ring at = {};
  __device__ __forceinline__ bool next_one(Tile& t) {
    if (!wait_one<PAIR>(c, &c.tile_full[at.i], at.ph, limit)) return false;
    const bool any = c.tiles[at.i].valid != 0;
    t = c.tiles[at.i].tile;
    sm100::mbar_arrive(&c.tile_empty[at.i]);
    at.step(TILE_SLOTS);
    return any;
  }
  __device__ __forceinline__ bool next_warp(Tile& t) {
    if (!wait_warp<PAIR>(c, &c.tile_full[at.i], at.ph, limit)) return false;
    const bool any = c.tiles[at.i].valid != 0;
    t = c.tiles[at.i].tile;
    __syncwarp();
    if ((threadIdx.x & 31) == 0) sm100::mbar_arrive(&c.tile_empty[at.i]);
    at.step(TILE_SLOTS);
    return any;
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

template <class T, bool PAIR, uint32_t SUBS>
__global__ void __launch_bounds__(THREADS, 1)
    product_kernel(const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_q,
                   const __grid_constant__ Params p) {
  using namespace sm100;
  constexpr int G = PAIR ? 2 : 1;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  constexpr uint32_t subs = SUBS;
  static_assert(!PAIR || SUBS == 1);
  const uint32_t kblocks = p.kblocks;
  const uint32_t per_stage = stage_bytes(p), per_sf = sf_bytes(p);
  unsigned char* sf_ring = smem + static_cast<size_t>(p.stages) * per_stage;
  Control& c = *reinterpret_cast<Control*>(sf_ring + static_cast<size_t>(p.sf_slots) * per_sf);
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? blockIdx.x & 1 : 0;  // in the cluster: 0 leads

  if (warp == 1) tmem_alloc<G>(&c.tmem);
  Walk walk(p.groups, lane, p.tile_q, p.tile_log2);
  if (warp == 3) walk.start();  // the offsets are on their way while the others set up
  if (threadIdx.x == 0) {
    c.failed = 0;
    if constexpr (PAIR) c.peer_failed = in_peer(&c.failed, rank);
    for (uint32_t s = 0; s < p.stages; ++s) mbar_init(&c.full[s], 1), mbar_init(&c.empty[s], 1);
    for (uint32_t s = 0; s < p.sf_slots; ++s)
      mbar_init(&c.sf_full[s], 32), mbar_init(&c.sf_peer[s], 1), mbar_init(&c.sf_empty[s], 1);
    for (uint32_t s = 0; s < p.accs; ++s) mbar_init(&c.acc_full[s], 1), mbar_init(&c.acc_empty[s], EPI_WARPS * G);
    // readers of a tile: the producer, the MMA warp, the scales, the epilogue
    for (uint32_t s = 0; s < TILE_SLOTS; ++s) mbar_init(&c.tile_full[s], 1), mbar_init(&c.tile_empty[s], 3 + EPI_WARPS);
    mbar_init(&c.done, 1);
    fence_barrier_init();
    tma_prefetch_desc(&map_b);
    tma_prefetch_desc(&map_q);
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync();  // the other CTA's barriers are there
  tc_fence_after();
  const uint32_t tmem = c.tmem;
  const uint64_t limit = p.wait_cycles;
  Reader<PAIR> reader{c, limit};
  Tile t;

  if (warp == 0) {
    // ---- producer ----
    if (elect_one()) {
      uint32_t issued = 0;
      Ring s;
      bool ok = true;
      while (ok && reader.next_one(t)) {
        const uint32_t width = round16(t.queries), load = width / G;
        const uint32_t boxes = (load + p.q_box - 1) / p.q_box;
        const uint32_t bytes = subs * BASE_BYTES + boxes * p.q_box * KB;  // this CTA's
        const int32_t b0 = t.b0 + rank * BM, q0 = t.q0 + rank * load;
        for (uint32_t kb = 0; kb < kblocks; ++kb) {
          if (!(ok = wait_one<PAIR>(c, &c.empty[s.i], s.ph ^ 1, limit))) break;
          unsigned char* dst = smem + static_cast<size_t>(s.i) * per_stage;
          unsigned char* dst_q = dst + subs * BASE_BYTES;
          if constexpr (PAIR) {
            // both CTAs' bytes are counted on the leader's barrier
            const uint32_t bar = leaders(&c.full[s.i]);
            if (rank == 0) mbar_arrive_expect_tx(&c.full[s.i], G * bytes);
            tma_load_pair(dst, &map_b, bar, kb * KB, b0);
            for (uint32_t i = 0; i < boxes; ++i)
              tma_load_pair(dst_q + i * p.q_box * KB, &map_q, bar, kb * KB, q0 + i * p.q_box);
          } else {
            mbar_arrive_expect_tx(&c.full[s.i], bytes);
            for (uint32_t i = 0; i < subs; ++i)
              tma_load_2d(dst + i * BASE_BYTES, &map_b, &c.full[s.i], kb * KB, b0 + i * BM);
            for (uint32_t i = 0; i < boxes; ++i)
              tma_load_2d(dst_q + i * p.q_box * KB, &map_q, &c.full[s.i], kb * KB, q0 + i * p.q_box);
          }
          c.loaded[s.i] = bytes;
          ++issued;
          s.step(p.stages);
        }
      }
      c.issued = issued;
    }
  } else if (warp == 1 && rank == 0) {
    // ---- MMA ----
    if (elect_one()) {
      Ring s, sf, acc, old;
      uint32_t quad = 0;  // number of the scale words; old: the slot of those SF_TMEM before
      bool ok = true;
      bool ready = false;  // the next stage is known to be full
      const uint32_t sf_base = smem_u32(sf_ring);
      const uint64_t desc_a = smem_desc_k_sw128(smem_u32(smem));
      const uint64_t desc_b = smem_desc_k_sw128(smem_u32(smem) + subs * BASE_BYTES);
      const uint32_t last_steps = (p.dim - (kblocks - 1) * KB + MMA_K - 1) / MMA_K;
      while (ok && reader.next_one(t)) {
        const uint32_t width = round16(t.queries);
        if (!(ok = wait_one<PAIR, PAIR>(c, &c.acc_empty[acc.i], acc.ph ^ 1, limit))) break;
        tc_fence_after();
        const uint32_t d = tmem + acc.i * p.acc_cols, idesc0 = idesc_mxf8(G * BM, width, 0);
        for (uint32_t kb = 0; kb < kblocks; ++kb) {
          const uint32_t sfa = tmem + p.sf_col + (quad % SF_TMEM) * p.sf_cols, sfb = sfa + 4 * subs;
          if ((kb & 3) == 0) {
            if (!(ok = wait_one<PAIR>(c, &c.sf_full[sf.i], sf.ph, limit))) break;
            if constexpr (PAIR)
              if (!(ok = wait_one<PAIR, true>(c, &c.sf_peer[sf.i], sf.ph, limit))) break;
            if (p.sf_slots > SF_TMEM && quad >= SF_TMEM) {
              // the words in the same TMEM columns before are done with
              if (!(ok = wait_one<PAIR>(c, &c.sf_empty[old.i], old.ph, limit))) break;
              old.step(p.sf_slots);
            }
            fence_proxy_async();  // the words came by generic copies
            tc_fence_after();
            const uint32_t from = sf_base + sf.i * per_sf;
#pragma unroll
            for (uint32_t i = 0; i < subs; ++i) copy_scales<G>(sfa + 4 * i, from + i * ATOM);
            copy_scales<G>(sfb, from + subs * ATOM);
            if (width > 128) copy_scales<G>(sfb + 4, from + (subs + 1) * ATOM);
          }
          if (!ready && !(ok = wait_one<PAIR>(c, &c.full[s.i], s.ph, limit))) break;
          tc_fence_after();
          // look at the next stage now: the answer is there once these MMAs are issued
          Ring following = s;
          following.step(p.stages);
          ready = try_wait<false>(&c.full[following.i], following.ph);
          const uint64_t at = static_cast<uint64_t>(s.i * (per_stage >> 4));
          const uint64_t a = desc_a + at, b = desc_b + at;
          const uint32_t idesc = idesc0 + ((kb & 3) << 4) + ((kb & 3) << 29);
          const uint32_t steps = kb + 1 == kblocks ? last_steps : KB / MMA_K;
#pragma unroll
          for (uint32_t i = 0; i < subs; ++i) {
#pragma unroll
            for (uint32_t k = 0; k < KB / MMA_K; ++k)
              if (k < steps)
                mma_mxf8<G>(d + i * p.q_rows, a + i * (BASE_BYTES >> 4) + 2 * k, b + 2 * k, idesc, sfa + 4 * i, sfb,
                            (kb | k) != 0);
          }
          commit<G>(&c.empty[s.i]);
          s = following;
          if ((kb & 3) == 3 || kb + 1 == kblocks) {
            commit<G>(&c.sf_empty[sf.i]);
            ++quad;
            sf.step(p.sf_slots);
          }
        }
        if (!ok) break;
        commit<G>(&c.acc_full[acc.i]);
        acc.step(p.accs);
      }
      // all MMAs complete before TMEM is released
      commit<G>(&c.done);
      wait_drained(&c.done, 0, clock64());
    }
  } else if (PAIR && warp == 1) {
    // ---- the second CTA of a pair: tells the leader of its scale words ----
    if (elect_one()) {
      Ring sf;
      bool ok = true;
      while (ok && reader.next_one(t)) {
        for (uint32_t w = 0; w < (kblocks + 3) / 4; ++w) {
          if (!(ok = wait_one<PAIR>(c, &c.sf_full[sf.i], sf.ph, limit))) break;
          fence_proxy_async();
          arrive_cluster(leaders(&c.sf_peer[sf.i]));
          sf.step(p.sf_slots);
        }
      }
    }
  } else if (warp == 2) {
    // ---- scales ----
    Ring sf;
    bool ok = true;
    while (ok && reader.next_warp(t)) {
      const uint32_t words = (kblocks + 3) / 4, columns = (t.queries + 31) / 32;
      const uint64_t b0 = static_cast<uint64_t>(t.b0) + rank * BM;
      for (uint32_t w = 0; w < words; ++w) {
        if (!(ok = wait_warp<PAIR>(c, &c.sf_empty[sf.i], sf.ph ^ 1, limit))) break;
        const uint32_t to = smem_u32(sf_ring) + sf.i * per_sf + lane * 16;
        for (uint32_t i = 0; i < subs; ++i) {
#pragma unroll
          for (uint32_t j = 0; j < 4; ++j) {
            const uint64_t r = b0 + i * BM + 32 * j + lane;
            const bool any = r < p.groups.nb;
            copy_word(to + i * ATOM + 4 * j, p.b_scales + (any ? r * p.b_sld + 4 * w : 0), any);
          }
        }
        for (uint32_t j = 0; j < columns; ++j) {
          const uint64_t r = static_cast<uint64_t>(t.q0) + 32 * j + lane;
          const bool any = r < p.groups.nq;
          copy_word(to + (subs + j / 4) * ATOM + 4 * (j & 3), p.q_scales + (any ? r * p.q_sld + 4 * w : 0), any);
        }
        copies_arrive(&c.sf_full[sf.i]);
        sf.step(p.sf_slots);
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");  // landed before the CTA exits
  } else if (warp == 3) {
    // ---- the walk over tiles: the same in both CTAs of a pair ----
    Ring s;
    for (uint64_t k = blockIdx.x / G;; k += gridDim.x / G) {
      const bool any = walk.find(k, t);
      if (!wait_warp<PAIR>(c, &c.tile_empty[s.i], s.ph ^ 1, limit)) break;
      if (lane == 0) {
        c.tiles[s.i].tile = t;
        c.tiles[s.i].valid = any;
        mbar_arrive(&c.tile_full[s.i]);
      }
      if (!any) break;
      s.step(TILE_SLOTS);
    }
  } else if (warp >= 4) {
    // ---- epilogue ----
    const uint32_t quarter = warp & 3, row0 = rank * BM + quarter * 32 + lane;
    T* out = static_cast<T*>(p.out);
    Ring acc;
    while (reader.next_warp(t)) {
      if (!wait_warp<PAIR>(c, &c.acc_full[acc.i], acc.ph, limit)) break;
      tc_fence_after();
      // Outputs are stored with the streaming hint: without it a large one drives the operands out of L2
      // (4096 x 65536 x 768 f32: 290 us, with it 270; x 256: 212 and 193; few queries: no difference).
      // This warp's chunks of 32 columns, numbered through the subs: every other one. The accumulator goes
      // back once the last of them is in registers, before it is stored.
      const uint32_t chunks = (t.queries + 31) / 32, first = (warp - 4) >> 2, all = subs * chunks;
      const uint64_t stride4 = 4 * t.stride;
      for (uint32_t k = first; k < all || k == first; k += EPI_WARPS / 4) {
        uint32_t v[32];
        const uint32_t i = subs == 1 ? 0 : k / chunks, q = (k - i * chunks) * 32;
        if (k < all) {
          tmem_ld_32x32b_x32(tmem + ((quarter * 32) << 16) + acc.i * p.acc_cols + i * p.q_rows + q, v);
          tmem_ld_wait();
        }
        if (k + EPI_WARPS / 4 >= all) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (PAIR && rank != 0)
              arrive_cluster_relaxed(leaders(&c.acc_empty[acc.i]));
            else
              arrive_relaxed(&c.acc_empty[acc.i]);
          }
        }
        const uint32_t row = row0 + i * BM;
        if (k < all && row < t.rows) {
          T* dst[4];
          dst[0] = out + t.at + row + q * t.stride;
          dst[1] = dst[0] + t.stride, dst[2] = dst[0] + 2 * t.stride, dst[3] = dst[1] + 2 * t.stride;
          if (q + 32 <= t.queries) {
#pragma unroll
            for (uint32_t j = 0; j < 32; ++j) {
              __stcs(dst[j & 3], from_f32<T>(__uint_as_float(v[j])));
              dst[j & 3] += stride4;
            }
          } else {
#pragma unroll
            for (uint32_t j = 0; j < 32; ++j) {
              if (q + j < t.queries) __stcs(dst[j & 3], from_f32<T>(__uint_as_float(v[j])));
              dst[j & 3] += stride4;
            }
          }
        }
        __syncwarp();
      }
      acc.step(p.accs);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync();  // both have issued all that they will, and `failed` is the same in both
  // without a failure the MMAs waited for every copy
  if (c.failed) {
    if (rank == 0 && threadIdx.x == 0) drain<PAIR>(c, p.stages);
    __syncwarp();
    if constexpr (PAIR) cluster_sync();  // neither CTA goes while copies into it or signals of it are in flight
  }
  // the leader's signals to the other CTA are on their way until its last one is here
  if (PAIR && rank != 0 && warp == 1) {
    if (lane == 0) wait_drained(&c.done, 0, clock64());
    __syncwarp();
  }
  tc_fence_after();
  if (warp == 1) tmem_free<G>(tmem);
  if (threadIdx.x == 0 && c.failed) leave_fault(p.groups.record, FAULT_TIMEOUT);
}

}  // namespace bq_tc
}  // namespace pxc
