// Product of rows in 8-bit floating point: out[m, n] = sum over blocks b of 128 of 2^(ex[m, b] + ew[n, b]) times the sum over
// the block of X[m, k] W[n, k], plus bias[n].
//
// tcgen05.mma kind::mxf8f6f4 with a block scale: the tensor core multiplies by the powers of two as it goes (they lie in
// tensor memory, a byte for each row and block; the instruction's scale of 32 elements is given four times the same
// byte). One block a SM, persistent over units of work: a tile of 128 tokens and 64, 128 or 192 channels, or a part of its
// K range. Warp 0 loads by TMA into a ring of four steps of 128 of K (pairs: five), warp 1 issues the MMAs, the others read TMEM:
// each has 32 tokens, a lane a token, and 64 channels, in registers.
//
// For many tiles two blocks of a cluster share one of 256 tokens (cta_group::2) and load a third less for it.
//
// The tensor core cuts, and does not round, what it adds to an accumulator: over 16384 of K sums came out 6.5e-6 of
// their size too small. So an accumulator takes 1024 of K, and the warps add up those sums in float32, rounded.
// Two accumulators: one is read while the other is filled.
//
// Measured: 8192 x 8192 x 8192 in 406 us, 2.71 PFLOP/s, 1.65 times the bf16 product's measured rate: bound by the tensor cores, 79% busy at the 1.49 GHz
// to which the power limit takes the clock (L2 53%). 16384 x 768 x 32000 in 463, held up by its output: a plain fill of the output's 1.05 GB
// takes 273, this product with a K of 128 345, and each further 128 of K another 25, half of what its MMAs take. 1 x 768 x 32000 in 8.8 us with the weight in L2, 3.8 us of
// it the weight's bytes from memory: a chain of latencies and a second round of tiles.
#include <cmath>
#include "fp8.cuh"
#include "sm100.cuh"
#include "tma_host.cuh"

namespace flb {

using namespace sm100;
using namespace fp8;

namespace {

constexpr int kTokens = 128;      // a tile's rows of X
constexpr int kStep = 128;        // of K a stage: one block
constexpr int kChunk = 8;         // steps that one accumulator takes
constexpr int kCols = 64;         // channels of an epilogue warp
constexpr int kStaged = 4096;     // bytes a warp stages for a store: 32 tokens of 128 bytes
constexpr uint32_t kWaitLimit = 1u << 20;   // polls, each held for about 4 us by the hardware: 4 s
constexpr uint32_t kDrainLimit = 1u << 20;  // the same for what is still in flight when a block ends early

template <int NC> constexpr int epilogue_warps() { return NC / 16; }  // 4 quarters of TMEM's lanes x NC / 64
template <int NC> constexpr int threads() { return 64 + 32 * epilogue_warps<NC>(); }
// PAIR: two blocks of a cluster share a tile of 256 tokens, each with its own 128 and half of the channels' weight rows.
template <bool PAIR, int NC> constexpr int weight_rows() { return PAIR ? NC / 2 : NC; }
template <bool PAIR, int NC> constexpr int stage_bytes() { return (kTokens + weight_rows<PAIR, NC>()) * kStep; }
template <bool PAIR> constexpr int stages() { return PAIR ? 5 : 4; }
// ring | its powers of two | staged tiles | biases
constexpr int kExpBytes = 3 * kTileBytes;  // a stage's: of the tokens, and of up to two groups of 128 channels
template <bool PAIR, int NC> constexpr int smem_bytes() {
  return stages<PAIR>() * (stage_bytes<PAIR, NC>() + kExpBytes) + epilogue_warps<NC>() * (kStaged + kCols * 4) + 1024;
}
// Tensor memory: two accumulators, then a set of powers of two a stage (4 columns of the tokens', 8 of the channels')
constexpr int kExpCols = 12;
template <bool PAIR, int NC> constexpr uint32_t tmem_cols() { return 2 * NC + stages<PAIR>() * kExpCols > 256 ? 512 : 256; }

struct Args {
  const void* bias;    // null, or [N]
  int bias_dtype;
  void* out;           // [M, N]
  int64_t M, N;
  bool tma_store;      // rows of out start on 16 bytes
  bool early;          // the kernel before this one wrote no weight
  int a_rows;          // of X that a stage loads: 128, or fewer where there are no more
  int k_blocks, quads;
  int n_tiles, tiles, splits;
  int group;           // tiles of tokens that go through all channels together
  bool stream_out;     // the output leaves L2 before the operands do
  float* parts;        // [tiles][splits][NC][128], splits > 1
  uint32_t* counts;    // [tiles], zero
  uint32_t* error;
  uint32_t limit;      // polls of a wait (kWaitLimit)
  int drop;            // a step whose copies the first worker waits for in vain (a test of the waits), or -1
};

__device__ __forceinline__ bool step_wait(uint64_t* bar, uint32_t phase, uint32_t limit) { return mbar_try_wait(bar, phase) || mbar_wait(bar, phase, limit); }
// The step `drop` expects 16 bytes more than it is sent, until the MMAs have been given up.
constexpr uint32_t kNeverSent = 16;

// One block, or a pair of them: the instructions that differ.
template <bool PAIR> struct Blocks;
template <> struct Blocks<false> {
  static constexpr int kCount = 1;
  static __device__ __forceinline__ void alloc(uint32_t* dst, uint32_t n) { tmem_alloc(dst, n); }
  static __device__ __forceinline__ void relinquish() { tmem_relinquish(); }
  static __device__ __forceinline__ void dealloc(uint32_t t, uint32_t n) { tmem_dealloc(t, n); }
  static __device__ __forceinline__ void load(void* dst, const void* tmap, uint64_t* bar, int c0, int c1) { tma_load_2d(dst, tmap, bar, c0, c1); }
  static __device__ __forceinline__ void copy_exps(uint32_t tmem, uint64_t d) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(d) : "memory");
  }
  static __device__ __forceinline__ void mma(uint32_t d, uint64_t da, uint64_t db, uint32_t desc, uint32_t ea, uint32_t eb, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(da), "l"(db), "r"(desc), "r"(ea), "r"(eb), "r"(accumulate)
        : "memory");
  }
  static __device__ __forceinline__ void commit(uint64_t* bar) { umma_commit(bar); }
  static __device__ __forceinline__ void arrive_all(uint64_t* bar) { mbar_arrive(bar); }
  static __device__ __forceinline__ void arrive_first(uint64_t* bar) { mbar_arrive(bar); }
  static __device__ __forceinline__ void meet() { __syncthreads(); }
};
template <> struct Blocks<true> {
  static constexpr int kCount = 2;
  static __device__ __forceinline__ void alloc(uint32_t* dst, uint32_t n) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst)), "r"(n) : "memory");
  }
  static __device__ __forceinline__ void relinquish() { asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory"); }
  static __device__ __forceinline__ void dealloc(uint32_t t, uint32_t n) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(t), "r"(n) : "memory");
  }
  // this barrier in one of the pair's blocks
  static __device__ __forceinline__ uint32_t in_block(uint64_t* bar, int block) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(bar)), "r"(block));
    return r;
  }
  // into this block's shared memory; the bytes count at the first block's barrier
  static __device__ __forceinline__ void load(void* dst, const void* tmap, uint64_t* bar, int c0, int c1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
            smem_u32(dst)),
        "l"(tmap), "r"(in_block(bar, 0)), "r"(c0), "r"(c1)
        : "memory");
  }
  // issued by the first block for both: each block's powers of two to its own tensor memory, each block's tokens, the two halves of the channels
  static __device__ __forceinline__ void copy_exps(uint32_t tmem, uint64_t d) {
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(d) : "memory");
  }
  static __device__ __forceinline__ void mma(uint32_t d, uint64_t da, uint64_t db, uint32_t desc, uint32_t ea, uint32_t eb, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(da), "l"(db), "r"(desc), "r"(ea), "r"(eb), "r"(accumulate)
        : "memory");
  }
  // arrives at this barrier in both blocks
  static __device__ __forceinline__ void commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
                 "h"((uint16_t)3)
                 : "memory");
  }
  static __device__ __forceinline__ void arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
  }
  static __device__ __forceinline__ void arrive_all(uint64_t* bar) { arrive(in_block(bar, 0)), arrive(in_block(bar, 1)); }
  static __device__ __forceinline__ void arrive_first(uint64_t* bar) { arrive(in_block(bar, 0)); }
  static __device__ __forceinline__ void meet() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
};
// 32 rows of 16 bytes, for TMEM lanes 0 to 31 and again for the other three quarters
__device__ __forceinline__ uint64_t exps_desc(const void* src) { return make_smem_desc(smem_u32(src), 16, 128, kSwizzleNone); }
// e4m3 operands, both K-major, float32 accumulators, powers of two as scales; which of the four bytes of a scale's word
template <int M, int NC> __device__ __forceinline__ uint32_t idesc(uint32_t byte) {
  return (byte << 4) | ((uint32_t)(NC >> 3) << 17) | (1u << 23) | ((uint32_t)(M >> 7) << 27) | (byte << 29);
}
// true in one thread of the warp, the same each time
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ void tma_store_2d(const void* tmap, const void* src, int c0, int c1, uint64_t policy) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group.L2::cache_hint [%0, {%2, %3}], [%1], %4;" ::"l"(tmap),
               "r"(smem_u32(src)), "r"(c0), "r"(c1), "l"(policy)
               : "memory");
}
template <int NC> __device__ __forceinline__ void epilogue_barrier() {
  asm volatile("bar.sync 1, %0;" ::"n"(epilogue_warps<NC>() * 32) : "memory");
}

template <bool PAIR, int NC, typename T>
__global__ void __launch_bounds__(threads<NC>(), 1)
    fp8_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_ex,
               const __grid_constant__ CUtensorMap tm_ew, const __grid_constant__ CUtensorMap tm_out, const Args a) {
  using B = Blocks<PAIR>;
  constexpr int S = stages<PAIR>(), EW = epilogue_warps<NC>(), ROWS = weight_rows<PAIR, NC>(), kStage = stage_bytes<PAIR, NC>();
  constexpr uint32_t kExpTmem = 2 * NC;
  extern __shared__ uint8_t dyn[];
  // other_done: in the first block, the second one's loader has issued its last load
  __shared__ __align__(8) uint64_t full[S], empty[S], acc_full[2], acc_empty[2], drain, other_done;
  __shared__ uint32_t tmem_base, last_flag;
  uint8_t* const ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dyn) + 1023) & ~(uintptr_t)1023);
  uint8_t* const staged_all = ring + (size_t)S * kStage;  // 1024-byte aligned: 128-byte swizzled tiles
  uint8_t* const exps = staged_all + EW * kStaged;
  float* const bias_all = reinterpret_cast<float*>(exps + S * kExpBytes);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = PAIR ? blockIdx.x & 1 : 0, worker = blockIdx.x / B::kCount, workers = gridDim.x / B::kCount;

  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tm_x);
    tma_prefetch_desc(&tm_w);
    for (int i = 0; i < S; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&acc_full[i], 1), mbar_init(&acc_empty[i], B::kCount * EW);
    mbar_init(&drain, 1), mbar_init(&other_done, 1);
    fence_mbar_init();
  }
  if (warp == 1) {
    B::alloc(&tmem_base, tmem_cols<PAIR, NC>());
    B::relinquish();
  }
  tc_fence_before();
  __syncwarp();
  B::meet();
  tc_fence_after();
  const uint32_t tmem = tmem_base;

  const int units = a.tiles * a.splits, m_tiles = a.tiles / a.n_tiles;
  // a unit's tokens (this block's), channels and steps of K
  auto place = [&](int u, int& m0, int& n0, int& k0, int& k1) {
    const int tile = u / a.splits, split = u - tile * a.splits;
    const int g = tile / (a.group * a.n_tiles), in = tile - g * a.group * a.n_tiles, rows = min(a.group, m_tiles - g * a.group);
    m0 = ((g * a.group + in % rows) * B::kCount + rank) * kTokens;
    n0 = in / rows * NC;
    k0 = (int)((int64_t)a.k_blocks * split / a.splits);
    k1 = (int)((int64_t)a.k_blocks * (split + 1) / a.splits);
  };
  const int groups_w = (int)blocks_of(a.N);
  // groups of 128 channels' powers of two that a tile reaches: one or two, from n0 / 128 on
  auto groups_of = [&](int n0) { return min((n0 + NC - 1) / kBlock, groups_w - 1) - n0 / kBlock + 1; };

  if (warp == 0) {
    // as below, the whole warp goes through the loop and one thread issues
    const bool issues = elect_one();
    bool ok = true;
    uint32_t it = 0, early = 0;
    // the powers of two of four steps come with the first of them. Both blocks of a pair need those of all the tile's channels.
    auto load_w = [&](int s, int n0, int groups, int k, bool first) {
      B::load(ring + s * kStage + kTokens * kStep, &tm_w, &full[s], k * kStep, n0 + rank * ROWS);
      if (first) {
        const int row = n0 / kBlock * a.quads + k / 4;
        B::load(exps + s * kExpBytes + kTileBytes, &tm_ew, &full[s], 0, row);
        if (groups > 1) B::load(exps + s * kExpBytes + 2 * kTileBytes, &tm_ew, &full[s], 0, row + a.quads);
      }
    };
    // the first block expects both blocks' bytes (the other's may land before: the count goes below zero)
    const uint32_t codes_bytes = (uint32_t)((a.a_rows + ROWS) * kStep);
    const uint32_t drop = worker == 0 ? (uint32_t)a.drop : ~0u;
    auto expect = [&](int s, int groups, bool first, uint32_t step) {
      if (rank == 0)
        mbar_arrive_expect_tx(&full[s], B::kCount * (codes_bytes + (first ? (1 + groups) * kTileBytes : 0)) + (step == drop ? kNeverSent : 0));
    };
    // Where the kernel that this one may overlap is the one that makes X's codes, the weight was written before that
    // kernel started: a first ring of weight tiles is on its way before the wait.
    for (int u = worker; a.early && u < units && early < (uint32_t)S; u += workers) {
      int m0, n0, k0, k1;
      place(u, m0, n0, k0, k1);
      const int groups = groups_of(n0);
      for (int k = k0; k < k1 && early < (uint32_t)S; ++k, ++early) {
        const bool first = k == k0 || (k & 3) == 0;
        if (issues) {
          expect(early, groups, first, early);
          load_w(early, n0, groups, k, first);
        }
      }
    }
    wait_predecessor();
    int s = 0;
    uint32_t phase = 0;
    for (int u = worker; u < units && ok; u += workers) {
      int m0, n0, k0, k1;
      place(u, m0, n0, k0, k1);
      const int groups = groups_of(n0), row_x = m0 / kBlock * a.quads;
      for (int k = k0; k < k1; ++k, ++it) {
        const bool first = k == k0 || (k & 3) == 0, whole = it >= early;
        if (it >= (uint32_t)S && !step_wait(&empty[s], phase ^ 1, a.limit)) {
          ok = false;
          break;
        }
        if (issues) {
          if (whole) {
            expect(s, groups, first, it);
            load_w(s, n0, groups, k, first);
          }
          B::load(ring + s * kStage, &tm_x, &full[s], k * kStep, m0);
          if (first) B::load(exps + s * kExpBytes, &tm_ex, &full[s], 0, row_x + k / 4);
        }
        s = s + 1 == S ? 0 : s + 1;
        phase ^= s == 0;
      }
    }
    __syncwarp();
    const uint32_t last = it > (uint32_t)S ? it - S : 0;
    const bool complete = ok;
    if (rank == 0) {
      // both blocks' copies count here: the other block waits for this one at the end
      uint32_t landed = 0;  // of the ring's stages
      if (drop >= last && drop < it) {
        mbar_wait(&drain, 0, kDrainLimit);
        if (issues)
          asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(&full[drop % S])), "n"(kNeverSent) : "memory");
        __syncwarp();
      }
      for (uint32_t i = last; i < it; ++i) {
        if (mbar_wait(&full[i % S], (i / S) & 1, kDrainLimit)) landed |= 1u << (i % S);
        else ok = false;
      }
      if (PAIR && !complete && mbar_wait(&other_done, 0, kDrainLimit)) {
        // The other block's wait may have seen what this one's gave up on: its copies for up to a ring of further steps come down on
        // barriers where nothing expects them yet. (It issued none where the last one there has not landed.) Where powers of two are among
        // them the bytes do not add up, and the wait runs out, long after they are down; so it does where it issued none.
        for (uint32_t i = it; i < it + S; ++i) {
          if (!(landed >> (i % S) & 1)) continue;
          if (issues) mbar_arrive_expect_tx(&full[i % S], codes_bytes);
          mbar_wait(&full[i % S], (i / S) & 1, kDrainLimit >> 6);
        }
      }
    } else if (issues) {
      B::arrive_first(&other_done);
    }
    if (PAIR) {
      // the first block's arrivals at this block's barriers are all in before the block ends
      if (complete)
        for (uint32_t i = last; i < it; ++i)
          if (!step_wait(&empty[i % S], (i / S) & 1, a.limit)) ok = false;
      if (rank == 1 && !mbar_wait(&drain, 0, kDrainLimit)) ok = false;
    }
    if (!ok && lane == 0) atomicExch(a.error, 1u);
  } else if (warp == 1) {
    if (rank == 0) {
      // The whole warp goes through the loop and one thread of it issues, so that the operands are known to be uniform; nothing is divided, and
      // stages are counted: one thread alone, with remainders, took 820 cycles a step where the MMAs take 384.
      // A set of powers of two is written again after S others, so S steps at least: the step that does it has waited for
      // a stage whose copies began when all MMAs up to S steps before, its readers among them, were done.
      const bool issues = elect_one();
      uint32_t s = 0, phase = 0, set = 0, b = 0, acc_phase = 0, started = 0;  // started: accumulators, up to two
      bool ok = true, any = false;
      const uint64_t da0 = make_smem_desc(smem_u32(ring), 16, 1024, kSwizzle128B), db0 = make_smem_desc(smem_u32(ring + kTokens * kStep), 16, 1024, kSwizzle128B);
      const uint64_t de0 = exps_desc(exps);
      wait_predecessor();
      for (int u = worker; u < units && ok; u += workers) {
        int m0, n0, k0, k1;
        place(u, m0, n0, k0, k1);
        const int groups = groups_of(n0);
        const uint32_t skip = 4 + n0 % kBlock / 32;
        uint32_t at = 0;
        int chunk = 0;  // steps of the accumulator so far
        for (int k = k0; k < k1; ++k) {
          if (chunk == 0 && started >= 2 && !step_wait(&acc_empty[b], acc_phase, a.limit)) {
            ok = false;
            break;
          }
          if (!step_wait(&full[s], phase, a.limit)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t byte = k & 3, desc = idesc<B::kCount * kTokens, NC>(0) | byte << 4 | byte << 29;
          const bool copies = k == k0 || byte == 0;
          if (copies) {
            at = tmem + kExpTmem + set * kExpCols;
            set = set + 1 == (uint32_t)S ? 0 : set + 1;
          }
          const bool closes = chunk == kChunk - 1 || k == k1 - 1;
          if (issues) {
            if (copies) {
              const uint64_t de = de0 + s * (kExpBytes >> 4);
              B::copy_exps(at, de);
              B::copy_exps(at + 4, de + (kTileBytes >> 4));
              if (groups > 1) B::copy_exps(at + 8, de + 2 * (kTileBytes >> 4));
            }
            const uint64_t da = da0 + s * (kStage >> 4), db = db0 + s * (kStage >> 4);
#pragma unroll
            for (int i = 0; i < kStep / 32; ++i) B::mma(tmem + b * NC, da + 2 * i, db + 2 * i, desc, at, at + skip, (chunk > 0 || i > 0) ? 1u : 0u);
            B::commit(&empty[s]);
            if (closes) B::commit(&acc_full[b]);
          }
          any = true;
          s = s + 1 == (uint32_t)S ? 0 : s + 1;
          phase ^= s == 0;
          ++chunk;
          if (closes) {
            chunk = 0, b ^= 1;
            if (started < 2) ++started;
            else acc_phase ^= b == 0;
          }
        }
      }
      __syncwarp();
      if (issues) {
        if (any) B::commit(&drain);
        else B::arrive_all(&drain);
      }
      if (!mbar_wait(&drain, 0, kDrainLimit)) ok = false;
      if (!ok && lane == 0) atomicExch(a.error, 1u);
    }
  } else {
    const int q = warp & 3, part = (warp - 2) / 4;  // this warp's 32 tokens and 64 channels
    uint8_t* const staged = staged_all + (warp - 2) * kStaged;
    float* const bias = bias_all + (warp - 2) * kCols;
    uint32_t local = 0;
    bool ok = true;
    uint64_t policy;
    if (a.stream_out) asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
    else asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(policy));
    wait_predecessor();
    for (int u = worker; u < units; u += workers) {
      int m0, n0, k0, k1;
      place(u, m0, n0, k0, k1);
      m0 += q * 32, n0 += part * kCols;
      __syncwarp();
#pragma unroll
      for (int c = 0; c < kCols; c += 32) {
        const int64_t n = n0 + c + lane;
        float v = 0;
        if (a.bias && n < a.N) {
          v = a.bias_dtype == FLB_F32 ? ld(reinterpret_cast<const float*>(a.bias) + n)
              : a.bias_dtype == FLB_F16 ? ld(reinterpret_cast<const __half*>(a.bias) + n) : ld(reinterpret_cast<const __nv_bfloat16*>(a.bias) + n);
        }
        bias[c + lane] = v;
      }
      __syncwarp();
      float sum[kCols];
#pragma unroll 1
      for (int k = k0; k < k1; k += kChunk, ++local) {
        const uint32_t b = local & 1;
        if (ok && !step_wait(&acc_full[b], (local >> 1) & 1, a.limit)) {
          ok = false;  // carries on with what is there, so that the warps meet at every barrier below
          if (lane == 0) atomicExch(a.error, 1u);
        }
        tc_fence_after();
        const uint32_t acc = tmem + b * NC + part * kCols + ((uint32_t)(q * 32) << 16);
        // (both halves at once took 160 bytes of spills with 192 channels)
        uint32_t v[32];
        tmem_ld32(acc, v);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 32; ++j) sum[j] = k == k0 ? __uint_as_float(v[j]) : sum[j] + __uint_as_float(v[j]);
        tmem_ld32(acc + 32, v);
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        // (a warp that has given up no longer stands in for one that is still reading: the MMAs then end too)
        if (lane == 0 && ok) B::arrive_first(&acc_empty[b]);
#pragma unroll
        for (int j = 0; j < 32; ++j) sum[32 + j] = k == k0 ? __uint_as_float(v[j]) : sum[32 + j] + __uint_as_float(v[j]);
      }
      if (!ok) {  // what did not come is NaN, for callers that do not wait for the error word: a training step sees it in its loss
#pragma unroll
        for (int j = 0; j < kCols; ++j) sum[j] = __uint_as_float(0x7fffffffu);
      }
      if (a.splits > 1) {
        const int tile = u / a.splits, split = u % a.splits;
        float* const parts = a.parts + ((int64_t)tile * a.splits * NC + part * kCols) * kTokens + q * 32 + lane;
        const bool some = m0 < a.M && n0 < a.N;
        if (some) {
          float* const mine = parts + (int64_t)split * NC * kTokens;
#pragma unroll
          for (int j = 0; j < kCols; ++j) mine[j * kTokens] = sum[j];
        }
        __threadfence();
        epilogue_barrier<NC>();
        if (threadIdx.x == 64) last_flag = atomicAdd(a.counts + tile, 1u) == (uint32_t)a.splits - 1 ? 1u : 0u;
        epilogue_barrier<NC>();
        if (!last_flag) continue;
        __threadfence();
        // the parts' sums in their order: the same bits whichever block comes last
        if (some) {
#pragma unroll
          for (int j = 0; j < kCols; ++j) sum[j] = __ldcg(parts + j * kTokens);
#pragma unroll 1
          for (int i = 1; i < a.splits; ++i) {
#pragma unroll
            for (int j = 0; j < kCols; ++j) sum[j] += __ldcg(parts + ((int64_t)i * NC + j) * kTokens);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < kCols; j += 4) {
        const float4 t = *reinterpret_cast<const float4*>(bias + j);
        sum[j] += t.x, sum[j + 1] += t.y, sum[j + 2] += t.z, sum[j + 3] += t.w;
      }
      // 128 bytes a token at a time: staged in shared memory, from where a TMA store, or coalesced ones, take them
      constexpr int kPer = 128 / (int)sizeof(T);
#pragma unroll
      for (int c = 0; c < kCols; c += kPer) {
        if (n0 + c >= a.N || m0 >= a.M) break;
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        __syncwarp();
#pragma unroll
        for (int w = 0; w < 8; ++w) {
          uint4 x;
          if constexpr (sizeof(T) == 4)
            x = make_uint4(__float_as_uint(sum[c + 4 * w]), __float_as_uint(sum[c + 4 * w + 1]), __float_as_uint(sum[c + 4 * w + 2]),
                           __float_as_uint(sum[c + 4 * w + 3]));
          else
            x = make_uint4(rows::pack2<T>(sum[c + 8 * w], sum[c + 8 * w + 1]), rows::pack2<T>(sum[c + 8 * w + 2], sum[c + 8 * w + 3]),
                           rows::pack2<T>(sum[c + 8 * w + 4], sum[c + 8 * w + 5]), rows::pack2<T>(sum[c + 8 * w + 6], sum[c + 8 * w + 7]));
          *reinterpret_cast<uint4*>(staged + sw128_offset(lane, w)) = x;
        }
        if (a.tma_store) {
          fence_async_shared();
          __syncwarp();
          if (lane == 0) {  // a store that ends outside the output is cut there
            tma_store_2d(&tm_out, staged, n0 + c, m0, policy);
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
        } else {
          __syncwarp();
          const int rows_here = (int)min((int64_t)32, a.M - m0);
          for (int r = 0; r < rows_here; ++r) {
            T* const to = reinterpret_cast<T*>(a.out) + (m0 + r) * a.N + n0 + c;
#pragma unroll
            for (int j = lane; j < kPer; j += 32)
              if (n0 + c + j < a.N)
                to[j] = *reinterpret_cast<const T*>(staged + sw128_offset(r, j * (int)sizeof(T) / 16) + j * sizeof(T) % 16);
          }
        }
      }
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  tc_fence_before();
  __syncwarp();
  B::meet();
  if (warp == 1) {
    tc_fence_after();
    B::dealloc(tmem, tmem_cols<PAIR, NC>());
  }
}

struct Shape {
  int width, n_tiles, tiles, splits;
  bool pair;
};
// The tile's channels, parts of K and blocks a tile whose rounds over the SMs cost least. In units of which about 850 take a microsecond: a step 100 and
// 0.8 for each row that it loads, a unit 600 for its start and epilogue; parts 1200 for their meeting and what they
// write and the last one adds up; a pair's start 1000. What decides (us, the product alone, operands from memory): 1 x 768 x 32000 with 128
// channels 11.5, 192 12.7, 64 14.3; 16 x 4096 x 4096 with 64 in two parts 12.7, whole 14.0; 500 x 8000 x 500 with 64 in four parts 13.4, 128 in
// eight 15.5; 1003 x 769 x 517 with 64 whole 7.7, in two parts 9.7; 768 x 16384 x 768 with 128 in four parts 22.2, 192 in four 24.6; 300 x 4096 x
// 4096 with 128 16.5, 192 in two parts 17.8; 2931 x 1001 x 2304 by pairs 14.0, by one block 15.2; 2931 x 768 x 2304 11.9 and 11.2;
// 8192 x 4096 x 4096 by pairs 110, by one block 134.
Shape shape_of(int64_t M, int64_t N, int64_t K) {
  const int64_t sms = num_sms(), m_tiles = (M + kTokens - 1) / kTokens, blocks = blocks_of(K), rows = std::min<int64_t>(M, kTokens);
  Shape best = {};
  double least = INFINITY;
  for (int nc : {192, 128, 64}) {
    const int64_t n_tiles = (N + nc - 1) / nc, tiles = m_tiles * n_tiles;
    for (int64_t splits = 1; splits <= std::min<int64_t>(blocks, std::max<int64_t>(1, sms / tiles)); ++splits) {
      const int64_t rounds = (tiles * splits + sms - 1) / sms, steps = (blocks + splits - 1) / splits;
      double cost = rounds * (steps * (100 + 0.8 * (rows + nc)) + 600);
      if (splits > 1) cost += 1200 + nc * ((rows + 31) / 32 / 4.0) * (16 + 5 * splits);
      if (cost < least) least = cost, best = Shape{nc, (int)n_tiles, (int)tiles, (int)splits, false};
    }
  }
  if (sms % 2 == 0) {
    const int64_t n_tiles = (N + 191) / 192, tiles = (M + 255) / 256 * n_tiles;
    const double cost = (tiles + sms / 2 - 1) / (sms / 2) * (blocks * (100 + 0.8 * 224) + 600) + 1000;
    if (cost < least) best = Shape{192, (int)n_tiles, (int)tiles, 1, true};
  }
  return best;
}

// Workspace: [error, counts] | codes and powers of two of X (when they are made here) | parts
struct Ws {
  size_t counts, codes, exps, parts, bytes;
};
Ws ws_of(const Shape& g, int64_t M, int64_t K, bool quantise) {
  auto al = [](size_t x) { return (x + 255) & ~(size_t)255; };
  Ws w;
  w.counts = 4;
  size_t off = al(4 + (g.splits > 1 ? (size_t)g.tiles * 4 : 0));
  w.codes = off;
  off += quantise ? al((size_t)M * rows::code_pitch(K)) : 0;
  w.exps = off;
  off += quantise ? al((size_t)exps_bytes(M, K)) : 0;
  w.parts = off;
  off += g.splits > 1 ? (size_t)g.tiles * g.splits * g.width * kTokens * 4 : 0;
  w.bytes = off;
  return w;
}

struct Maps {
  CUtensorMap x, w, ex, ew, out;
};

template <bool PAIR, int NC, typename T> int launch_t(const Maps& m, const Args& a, bool overlap, cudaStream_t s) {
  const auto kernel = fp8_kernel<PAIR, NC, T>;
  constexpr int kBlocks = PAIR ? 2 : 1;
  const int st = ensure_dyn_smem(reinterpret_cast<const void*>(kernel), smem_bytes<PAIR, NC>(), "fp8_linear shared memory");
  if (st != FLB_OK) return st;
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)std::min<int64_t>((int64_t)a.tiles * a.splits * kBlocks, num_sms() / kBlocks * kBlocks));
  cfg.blockDim = dim3(threads<NC>());
  cfg.dynamicSmemBytes = smem_bytes<PAIR, NC>();
  cfg.stream = s;
  cfg.attrs = attr;
  if (overlap) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (PAIR) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = 2;
    attr[cfg.numAttrs].val.clusterDim.y = 1;
    attr[cfg.numAttrs++].val.clusterDim.z = 1;
  }
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, m.x, m.w, m.ex, m.ew, m.out, a);
  count_launches(1);
  return check_cuda(e, "fp8_linear launch");
}

template <typename T> int launch(const Shape& g, const Maps& m, const Args& a, bool overlap, cudaStream_t s) {
  if (g.pair) return launch_t<true, 192, T>(m, a, overlap, s);
  switch (g.width) {
    case 64: return launch_t<false, 64, T>(m, a, overlap, s);
    case 128: return launch_t<false, 128, T>(m, a, overlap, s);
    default: return launch_t<false, 192, T>(m, a, overlap, s);
  }
}

// Powers of two as rows of 128 words: 128 rows' of four blocks
int exps_map(CUtensorMap* m, const uint8_t* exps, int64_t R, int64_t K) {
  const uint64_t dims[2] = {kTileBytes / 4, (uint64_t)(exps_bytes(R, K) / kTileBytes)};
  const uint64_t strides[1] = {kTileBytes};
  const uint32_t box[2] = {kTileBytes / 4, 1};
  return make_tmap(m, exps, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE);
}
int code_map(CUtensorMap* m, const int8_t* codes, int64_t rows, int64_t ld, int64_t K, int box_rows) {
  const uint64_t dims[2] = {(uint64_t)K, (uint64_t)rows};
  const uint64_t strides[1] = {(uint64_t)ld};
  const uint32_t box[2] = {kStep, (uint32_t)box_rows};
  return make_tmap(m, codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Of 126 MB of L2: a weight that stays there is gone through once for each tile of tokens, for a larger one 16 of them go together; an output that
// does not fit beside it leaves first.
constexpr int64_t kWeightInL2 = 48 << 20;
constexpr size_t kOutputInL2 = 64 << 20;

}  // namespace

int fp8_rows(const void* x, int64_t ldx, int8_t* codes, uint8_t* exps, int64_t R, int64_t K, int dtype, bool whole, uint32_t* zero, int n_zero,
             cudaStream_t s);

size_t fp8_linear_workspace_bytes(int64_t M, int64_t N, int64_t K, bool quantise) { return ws_of(shape_of(M, N, K), M, K, quantise).bytes; }

int fp8_linear(const void* x, int64_t ldx, const int8_t* x_codes, int64_t ldc, const uint8_t* x_exps, const int8_t* w_codes, int64_t ldw,
               const uint8_t* w_exps, const void* bias, int bias_dtype, void* out, int64_t M, int64_t N, int64_t K, int dtype, void* ws,
               int check_timeout, int drop, uint32_t limit, cudaStream_t s) {
  const Shape g = shape_of(M, N, K);
  const Ws l = ws_of(g, M, K, x != nullptr);
  uint8_t* const p = reinterpret_cast<uint8_t*>(ws);
  const int n_zero = 1 + (g.splits > 1 ? g.tiles : 0);
  const bool reset = !x && (g.splits > 1 || check_timeout);
  int st;
  if (x) {
    // the rows' kernel clears the error word and the counts too
    int8_t* const codes = reinterpret_cast<int8_t*>(p + l.codes);
    if ((st = fp8_rows(x, ldx, codes, p + l.exps, M, K, dtype, false, reinterpret_cast<uint32_t*>(p), n_zero, s)) != FLB_OK) return st;
    x_codes = codes, x_exps = p + l.exps, ldc = rows::code_pitch(K);
  } else if (reset) {  // otherwise nothing reads those words
    if ((st = check_cuda(cudaMemsetAsync(p, 0, (size_t)n_zero * 4, s), "fp8_linear reset")) != FLB_OK) return st;
  }
  Args a = {};
  a.a_rows = (int)std::min<int64_t>(kTokens, (M + 7) / 8 * 8);
  Maps m = {};
  if ((st = code_map(&m.w, w_codes, N, ldw, K, g.pair ? g.width / 2 : g.width)) != FLB_OK) return st;
  if ((st = code_map(&m.x, x_codes, M, ldc, K, a.a_rows)) != FLB_OK) return st;
  if ((st = exps_map(&m.ex, x_exps, M, K)) != FLB_OK || (st = exps_map(&m.ew, w_exps, N, K)) != FLB_OK) return st;
  const int es = dtype_size(dtype);
  a.tma_store = N * es % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
  if (a.tma_store) {
    const uint64_t dims[2] = {(uint64_t)N, (uint64_t)M};
    const uint64_t strides[1] = {(uint64_t)N * es};
    const uint32_t box[2] = {(uint32_t)(128 / es), 32};
    const CUtensorMapDataType dt = dtype == FLB_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : dtype == FLB_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                                                         : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    if ((st = make_tmap(&m.out, out, dt, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) != FLB_OK) return st;
  }
  a.bias = bias, a.bias_dtype = bias_dtype, a.out = out, a.M = M, a.N = N;
  a.early = x != nullptr;
  a.limit = limit ? limit : kWaitLimit, a.drop = drop;
  a.k_blocks = (int)blocks_of(K), a.quads = (int)quads_of(K), a.n_tiles = g.n_tiles, a.tiles = g.tiles, a.splits = g.splits;
  a.group = N * K <= kWeightInL2 ? 1 : 16;
  a.stream_out = (size_t)M * N * es > kOutputInL2;
  a.parts = reinterpret_cast<float*>(p + l.parts), a.counts = reinterpret_cast<uint32_t*>(p + l.counts), a.error = reinterpret_cast<uint32_t*>(p);
  switch (dtype) {
    case FLB_F32: st = launch<float>(g, m, a, x != nullptr, s); break;
    case FLB_F16: st = launch<__half>(g, m, a, x != nullptr, s); break;
    default: st = launch<__nv_bfloat16>(g, m, a, x != nullptr, s); break;
  }
  if (st != FLB_OK || !check_timeout) return st;
  uint32_t err = 0;
  if ((st = check_cuda(cudaMemcpyAsync(&err, p, 4, cudaMemcpyDeviceToHost, s), "fp8_linear error word")) != FLB_OK) return st;
  if ((st = check_cuda(cudaStreamSynchronize(s), "fp8_linear error word")) != FLB_OK) return st;
  return err ? fail(FLB_ERR_TIMEOUT, "fp8_linear: a bounded wait in the kernel gave up") : FLB_OK;
}

}  // namespace flb
