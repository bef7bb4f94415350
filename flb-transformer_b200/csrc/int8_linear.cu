// Product of 8-bit integer rows, each with a scale: out[m, n] = (sum_k X[m, k] W[n, k]) sx[m] sw[n] + bias[n].
//
// tcgen05.mma kind::i8, 32-bit integer accumulators in TMEM (exact for K <= 32768: K 127^2 < 2^31). One block
// a SM, persistent over units of work. Warp 0 loads by TMA into a ring, warp 1 issues the MMAs, warps 2-9 read
// TMEM (two accumulators, so that a tile's epilogue runs beside the next one's MMAs). Three kernels:
//
// int8_few_kernel, for few tokens or tiles. The weight rows are the M side of the instruction, 128 output
// channels a tile, and the tokens its N side, NT of 16 to 128: a decoding step wastes little of a tile.
// With fewer tiles than SMs a unit is a part of a tile's K range; the parts leave integer sums in the
// workspace, and the block that counts itself last adds them up: integers, the same in any order. Any N and
// alignment. Bound by its chain of latencies (launch, first copies, MMAs, sums: 16 x 4096 x 4096 10.7 us with the
// rows' kernel, 2.6 us of it the weight's bytes).
//
// int8_step_kernel, the same for up to 16 tokens of x itself, whose integer rows it makes on the way: 1 x 768 x 32000
// in 8.4 us, 3.8 us of it the weight's bytes.
//
// int8_many_kernel, for tiles enough to fill the SMs. The tokens are the M side, 128 a block, and 256 or 128
// channels the N side: a thread of the epilogue has a token's consecutive channels, packs them and leaves
// them in shared memory for a TMA store. (With the other orientation a thread has one channel of many
// tokens; pairing them up by shuffles took three times the instructions and bound the kernel.) For long K two
// blocks of a cluster share a tile of 256 x 256 (cta_group::2). Bound by the tensor cores, and over seconds by the power that
// they draw (995 W, the SMs at 1430 to 1490 MHz then): 8192 x 8192 x 8192 in 349 us in a short run and 404 in a long
// one, 3.15 and 2.72 POPS, 1.9 times the bf16 product's measured rates for each. With small K the output's way to memory takes
// its share: 16384 x 768 x 32000 in 397 and 461 us, 2.03 and 1.75 POPS, of which 160 us would write the output alone.
// Times below are of short runs / of runs of seconds where there are two.
#include <cmath>
#include "rows.cuh"
#include "sm100.cuh"
#include "tma_host.cuh"

namespace flb {

using namespace sm100;

namespace {

constexpr int kChannels = 128;   // a tile's weight rows
constexpr int kStep = 128;       // bytes of K a stage
constexpr int kRing = 198 * 1024;
constexpr int kEpilogue = 256;   // threads that read TMEM and store
constexpr int kGemmThreads = 64 + kEpilogue;
constexpr uint32_t kWaitLimit = 1u << 20;  // polls, each held for about 4 us by the hardware: 4 s
// A wait that gives up leaves wrong numbers behind it, but nothing in flight: every kernel's loader waits for its last copies and
// the thread that issues MMAs for its own (the barrier `drain`), with this limit, before the block gives up its shared
// memory and TMEM.
constexpr uint32_t kDrainLimit = 1u << 20;

template <int NT> constexpr int stage_bytes() { return (kChannels + NT) * kStep; }
template <int NT> constexpr int stages() { return kRing / stage_bytes<NT>(); }
template <int NT> constexpr uint32_t tmem_cols() { return 2 * NT < 32 ? 32 : 2 * NT; }

struct Int8Args {
  const float *sx, *sw;
  const void* bias;   // null, or out's type (bias32: float32)
  bool bias32;
  void* out;          // [M, N]
  int64_t M, N;
  bool pairs;         // 16-bit outputs two channels at a time
  bool early;         // the kernel before this one wrote no weight
  int k_blocks;       // of kStep
  int n_tiles, tiles, splits;
  int group;          // many tokens: tiles of tokens that go through all channels together
  bool stream_out;    // and the output leaves L2 before the operands do
  int32_t* parts;     // [tiles][splits][NT][128], splits > 1
  uint32_t* counts;   // [tiles], zero
  uint32_t* error;
  uint32_t limit;     // polls of a wait (kWaitLimit)
  int drop;           // a step whose copies the first block, or pair, waits for in vain (a test of the waits), or -1
};

// A bounded wait whose first poll is not behind the limit, an argument: 8192 x 4096 x 4096 in 93 us, 96 with it in front
__device__ __forceinline__ bool step_wait(uint64_t* bar, uint32_t phase, uint32_t limit) {
  return mbar_try_wait(bar, phase) || mbar_wait(bar, phase, limit);
}

// One thread's MMAs so far are done when this returns, or the limit has run out. issued: there are any.
__device__ __forceinline__ void drain_mma(uint64_t* drain, bool issued, uint32_t* error) {
  if (issued) umma_commit(drain);
  else mbar_arrive(drain);
  if (!mbar_wait(drain, 0, kDrainLimit)) atomicExch(error, 1u);
}

// The step `drop` expects 16 bytes more than it is sent, until the MMA thread has given up on it. (In the expected count,
// because a test of its own in the loader's loop took 0.7 us of 10.5 for 16 x 4096 x 4096.)
constexpr uint32_t kNeverSent = 16;
__device__ __forceinline__ uint32_t expected(uint32_t bytes, uint32_t step, uint32_t drop) { return bytes + (step == drop ? kNeverSent : 0); }
__device__ __forceinline__ void forgive(uint64_t* full, uint64_t* drain, uint32_t stages, uint32_t first, uint32_t end, uint32_t drop) {
  if (drop < first || drop >= end) return;
  mbar_wait(drain, 0, kDrainLimit);
  asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(&full[drop % stages])), "n"(kNeverSent) : "memory");
}

// signed 8-bit operands, both K-major, 32-bit integer accumulators
template <int NT> constexpr uint32_t idesc_i8() {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(NT >> 3) << 17) | ((uint32_t)(kChannels >> 4) << 24);
}
__device__ __forceinline__ void umma_i8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void load_cols(uint32_t taddr, uint32_t (&r)[32]) { tmem_ld32(taddr, r); }
__device__ __forceinline__ void load_cols(uint32_t taddr, uint32_t (&r)[16]) { tmem_ld16(taddr, r); }

__device__ __forceinline__ void epilogue_barrier() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// Sum times a token's scale, times a channel's: of an integer of up to 2^29 the first product passes float32 for scales from 2^99
// on, also where the second would bring it back. For such tokens the channel's scale comes first.
constexpr float kLargeScale = 0x1p96f;
__device__ __forceinline__ float scaled(uint32_t sum, float sx, float sw, float bias) {
  const bool large = fabsf(sx) > kLargeScale;
  return fmaf(__int2float_rn((int)sum) * (large ? sw : sx), large ? sx : sw, bias);
}

// One channel's values of CW tokens from token t0 on: scaled, with the bias, stored. FULL: the tile is
// inside the output.
template <typename T, int CW, bool FULL>
__device__ __forceinline__ void store_tokens(const Int8Args& a, const uint32_t (&acc)[CW], const float* sx, float sw, float bias,
                                             int64_t t0, int64_t channel) {
  T* out = reinterpret_cast<T*>(a.out);
  const int lane = threadIdx.x & 31;
  float v[CW];
#pragma unroll
  for (int j = 0; j < CW; j += 4) {
    const float4 s = *reinterpret_cast<const float4*>(sx + j);
    v[j] = scaled(acc[j], s.x, sw, bias);
    v[j + 1] = scaled(acc[j + 1], s.y, sw, bias);
    v[j + 2] = scaled(acc[j + 2], s.z, sw, bias);
    v[j + 3] = scaled(acc[j + 3], s.w, sw, bias);
  }
  if (sizeof(T) == 2 && a.pairs) {
    // two channels a store: an even lane takes both channels of an even token, its neighbour of the odd one
    const int odd = lane & 1;
    const int64_t c = channel - odd;
    T* p = out + (t0 + odd) * a.N + c;
    const bool in = FULL || c < a.N;
    const int left = FULL ? CW : (int)min((int64_t)CW, a.M - t0 - odd);  // tokens from this lane's first on
#pragma unroll
    for (int j = 0; j < CW; j += 2) {
      const float other = __shfl_xor_sync(0xffffffffu, odd ? v[j] : v[j + 1], 1);
      const float lo = odd ? other : v[j], hi = odd ? v[j + 1] : other;
      if constexpr (sizeof(T) == 2) {
        if (FULL || (in && j < left)) *reinterpret_cast<uint32_t*>(p) = rows::pack2<T>(lo, hi);
      }
      p += 2 * a.N;
    }
  } else {
    T* p = out + t0 * a.N + channel;
    const int left = FULL ? CW : channel < a.N ? (int)min((int64_t)CW, a.M - t0) : 0;
#pragma unroll
    for (int j = 0; j < CW; ++j) {
      if (FULL || j < left) st(p, v[j]);
      p += a.N;
    }
  }
}

template <int NT, typename T>
__global__ void __launch_bounds__(kGemmThreads, 1)
    int8_few_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, const Int8Args a) {
  constexpr int S = stages<NT>();
  constexpr uint32_t kBytes = stage_bytes<NT>();
  extern __shared__ uint8_t dyn[];
  __shared__ __align__(8) uint64_t full[S], empty[S], acc_full[2], acc_empty[2], drain;
  __shared__ uint32_t tmem_base, last_flag;
  __shared__ __align__(16) float scales[kEpilogue / 32][NT > 64 ? NT / 2 : 32];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dyn) + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tm_w);
    tma_prefetch_desc(&tm_x);
    for (int i = 0; i < S; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&acc_full[i], 1), mbar_init(&acc_empty[i], kEpilogue);
    mbar_init(&drain, 1);
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(&tmem_base, tmem_cols<NT>());
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base;

  const int units = a.tiles * a.splits;
  auto k_range = [&](int split, int& k0, int& k1) {
    k0 = (int)((int64_t)a.k_blocks * split / a.splits);
    k1 = (int)((int64_t)a.k_blocks * (split + 1) / a.splits);
  };

  if (warp == 0) {
    if (lane == 0) {
      // Where the kernel that this one may overlap is the one that makes the tokens' codes here, the weight was
      // written before that kernel started: a first ring of weight tiles, of the first units' steps, is on
      // its way before the wait.
      bool ok = true;
      uint32_t it = 0, early = 0;
      const uint32_t drop = blockIdx.x == 0 ? (uint32_t)a.drop : ~0u;
      for (int u = blockIdx.x; a.early && u < units && early < (uint32_t)S; u += gridDim.x) {
        int k0, k1;
        k_range(u % a.splits, k0, k1);
        for (int k = k0; k < k1 && early < (uint32_t)S; ++k, ++early) {
          mbar_arrive_expect_tx(&full[early], expected(kBytes, early, drop));
          tma_load_2d(ring + (size_t)early * kBytes, &tm_w, &full[early], k * kStep, (u / a.splits) % a.n_tiles * kChannels);
        }
      }
      wait_predecessor();
      for (int u = blockIdx.x; u < units && ok; u += gridDim.x) {
        const int tile = u / a.splits;
        const int n0 = (tile % a.n_tiles) * kChannels, m0 = (tile / a.n_tiles) * NT;
        int k0, k1;
        k_range(u % a.splits, k0, k1);
        for (int k = k0; k < k1; ++k, ++it) {
          const int s = it % S;
          uint8_t* st = ring + (size_t)s * kBytes;
          if (it >= early) {
            if (it >= (uint32_t)S && !step_wait(&empty[s], ((it / S) & 1) ^ 1, a.limit)) {
              ok = false;
              break;
            }
            mbar_arrive_expect_tx(&full[s], expected(kBytes, it, drop));
            tma_load_2d(st, &tm_w, &full[s], k * kStep, n0);
          }
          tma_load_2d(st + kChannels * kStep, &tm_x, &full[s], k * kStep, m0);
        }
      }
      // (every early step is among these: their x tiles were issued without a wait)
      const uint32_t last = it > (uint32_t)S ? it - S : 0;
      forgive(full, &drain, S, last, it, drop);
      for (uint32_t i = last; i < it; ++i)
        if (!mbar_wait(&full[i % S], (i / S) & 1, kDrainLimit)) ok = false;
      if (!ok) atomicExch(a.error, 1u);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_i8<NT>();
      uint32_t it = 0, local = 0;
      bool ok = true;
      // every warp waits for the predecessor before its first bounded wait: the polls are not spent on what that one has left
      wait_predecessor();
      for (int u = blockIdx.x; u < units && ok; u += gridDim.x, ++local) {
        const uint32_t b = local & 1;
        if (local >= 2 && !step_wait(&acc_empty[b], ((local >> 1) & 1) ^ 1, a.limit)) {
          ok = false;
          break;
        }
        tc_fence_after();
        int k0, k1;
        k_range(u % a.splits, k0, k1);
        for (int k = k0; k < k1; ++k, ++it) {
          const int s = it % S;
          if (!step_wait(&full[s], (it / S) & 1, a.limit)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t at = smem_u32(ring + (size_t)s * kBytes);
          // rows of 128 bytes, 128-byte swizzle: 8-row groups 1024 bytes apart, 32 bytes of K an instruction
          uint64_t da = make_smem_desc(at, 16, 1024, kSwizzle128B);
          uint64_t db = make_smem_desc(at + kChannels * kStep, 16, 1024, kSwizzle128B);
#pragma unroll
          for (int i = 0; i < kStep / 32; ++i, da += 2, db += 2)
            umma_i8(tmem + b * NT, da, db, idesc, (k > k0 || i > 0) ? 1u : 0u);
          umma_commit(&empty[s]);
        }
        if (ok) umma_commit(&acc_full[b]);
      }
      if (!ok) atomicExch(a.error, 1u);
      drain_mma(&drain, it > 0, a.error);
    }
  } else {
    // each epilogue warp has the 32 TMEM lanes, here channels, of its number mod 4, and half of the tokens
    // (the first four warps all of 16)
    constexpr int COLS = NT >= 32 ? NT / 2 : NT, CW = COLS < 32 ? COLS : 32, STEPS = COLS / CW;
    const int q = warp & 3, first = (warp - 2) / 4 * COLS;
    const bool has_cols = first < NT;
    float* sx = scales[warp - 2];
    uint32_t local = 0, limit = a.limit;
    wait_predecessor();
    for (int u = blockIdx.x; u < units; u += gridDim.x, ++local) {
      const uint32_t b = local & 1;
      const int tile = u / a.splits, split = u % a.splits;
      const int64_t n0 = (int64_t)(tile % a.n_tiles) * kChannels, m0 = (int64_t)(tile / a.n_tiles) * NT + first;
      const int64_t channel = n0 + q * 32 + lane;
      const bool there = channel < a.N, full_tile = n0 + kChannels <= a.N && m0 + COLS <= a.M;
      const float sw = there ? ld(a.sw + channel) : 0.f;
      float bias = 0.f;
      if (a.bias && there)
        bias = a.bias32 ? ld(reinterpret_cast<const float*>(a.bias) + channel) : ld(reinterpret_cast<const T*>(a.bias) + channel);
      __syncwarp();
#pragma unroll
      for (int c = 0; c < COLS; c += 32)
        if (c + lane < COLS) sx[c + lane] = m0 + c + lane < a.M ? ld(a.sx + m0 + c + lane) : 0.f;
      __syncwarp();
      if (!step_wait(&acc_full[b], (local >> 1) & 1, limit)) {
        // carries on with what is there, so that the warps meet at every barrier below
        limit = 1;
        if (lane == 0) atomicExch(a.error, 1u);
      }
      tc_fence_after();
      const uint32_t acc = tmem + b * NT + first + ((uint32_t)(q * 32) << 16);
      int32_t* part = a.parts + (((int64_t)tile * a.splits + split) * NT + first) * kChannels + q * 32 + lane;
      if (has_cols) {
        uint32_t v[2][CW];  // the next columns on their way from TMEM while these are stored
        load_cols(acc, v[0]);
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
          tmem_wait_ld();
          if (i + 1 < STEPS) {
            load_cols(acc + (i + 1) * CW, v[(i + 1) & 1]);
          } else {
            tc_fence_before();
            mbar_arrive(&acc_empty[b]);
          }
          if (a.splits > 1) {
            // tokens beyond M have no reader
#pragma unroll
            for (int j = 0; j < CW; ++j)
              if (m0 + i * CW + j < a.M) part[(i * CW + j) * kChannels] = (int32_t)v[i & 1][j];
          } else if (full_tile) {
            store_tokens<T, CW, true>(a, v[i & 1], sx + i * CW, sw, bias, m0 + i * CW, channel);
          } else if (m0 + i * CW < a.M) {
            store_tokens<T, CW, false>(a, v[i & 1], sx + i * CW, sw, bias, m0 + i * CW, channel);
          }
        }
      } else {
        mbar_arrive(&acc_empty[b]);
      }
      if (a.splits > 1) {
        __threadfence();
        epilogue_barrier();
        if (threadIdx.x == 64) last_flag = atomicAdd(a.counts + tile, 1u) == (uint32_t)a.splits - 1 ? 1u : 0u;
        epilogue_barrier();
        if (last_flag && has_cols) {
          __threadfence();
          const int32_t* p0 = a.parts + ((int64_t)tile * a.splits * NT + first) * kChannels + q * 32 + lane;
#pragma unroll 1
          for (int c = 0; c < COLS && m0 + c < a.M; c += CW) {
            uint32_t v[CW];
#pragma unroll
            for (int j = 0; j < CW; ++j) v[j] = 0;
            // the loads of several parts under way together
#pragma unroll 4
            for (int i = 0; i < a.splits; ++i) {
#pragma unroll
              for (int j = 0; j < CW; ++j)
                if (m0 + c + j < a.M) v[j] += (uint32_t)__ldcg(p0 + ((int64_t)i * NT + c + j) * kChannels);
            }
            store_tokens<T, CW, false>(a, v, sx + c, sw, bias, m0 + c, channel);
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, tmem_cols<NT>());
  }
}

// Two blocks that work on one tile (PAIR) or one: the instructions that differ.
template <bool PAIR> struct Group;
template <> struct Group<false> {
  static __device__ __forceinline__ void alloc(uint32_t* dst, uint32_t n) { tmem_alloc(dst, n); }
  static __device__ __forceinline__ void relinquish() { tmem_relinquish(); }
  static __device__ __forceinline__ void dealloc(uint32_t t, uint32_t n) { tmem_dealloc(t, n); }
  static __device__ __forceinline__ void load(void* dst, const void* tmap, uint64_t* bar, int c0, int c1) { tma_load_2d(dst, tmap, bar, c0, c1); }
  static __device__ __forceinline__ void mma(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t acc) { umma_i8(d, da, db, idesc, acc); }
  static __device__ __forceinline__ void commit(uint64_t* bar) { umma_commit(bar); }
  static __device__ __forceinline__ void arrive_all(uint64_t* bar) { mbar_arrive(bar); }
  static __device__ __forceinline__ void arrive_first(uint64_t* bar) { mbar_arrive(bar); }
  static __device__ __forceinline__ void meet() { __syncthreads(); }
};
template <> struct Group<true> {
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
  static __device__ __forceinline__ uint32_t first(uint64_t* bar) { return in_block(bar, 0); }
  // into this block's shared memory; the bytes count at the first block's barrier
  static __device__ __forceinline__ void load(void* dst, const void* tmap, uint64_t* bar, int c0, int c1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
            smem_u32(dst)),
        "l"(tmap), "r"(first(bar)), "r"(c0), "r"(c1)
        : "memory");
  }
  // issued by the first block for both: each block's tokens, the two halves of the channels
  static __device__ __forceinline__ void mma(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(da), "l"(db), "r"(idesc), "r"(acc)
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
  static __device__ __forceinline__ void arrive_first(uint64_t* bar) { arrive(first(bar)); }
  static __device__ __forceinline__ void meet() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
};

// ---- a decoding step ------------------------------------------------------------------------------------

// Up to 16 tokens of up to 4096 elements, straight from x: each block makes the integer rows that it needs itself, in
// the layout of the MMA's operand, while its weight tiles are on their way: one launch instead of two. With
// fewer tiles than SMs the blocks of a cluster, up to eight, share a tile's K range; the first one adds up their
// sums, which the others leave in its shared memory.
constexpr int kStepTokens = 16;
constexpr int kStepWidest = 4096;
constexpr int kStepStages = 6;
constexpr int kStepTile = kChannels * kStep;
constexpr int kMostParts = 8;
// ring | integer rows [K / 128][16][128 bytes] | the other blocks' sums [7][16][128]
constexpr int kStepSmem = kStepStages * kStepTile + kStepTokens * kStepWidest + (kMostParts - 1) * kStepTokens * kChannels * 4 + 1024;

struct StepArgs {
  const void* x;
  int64_t ldx;
  bool vec;  // rows that start on 16 bytes, a multiple of 8 wide
  int K;
};

// Eight elements of a row from k on, zeros beyond K. By ordinary loads, as everything here that a predecessor may have
// written: this kernel may start beside it, and the read-only path is for what does not change while a kernel runs.
template <typename T> __device__ __forceinline__ void load_row8(rows::Raw8<T>& r, const T* row, int k, int K, bool vec) {
  if (vec) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
      const uint4 v = k < K ? reinterpret_cast<const uint4*>(row + k)[i] : make_uint4(0, 0, 0, 0);
      r.w[4 * i] = v.x, r.w[4 * i + 1] = v.y, r.w[4 * i + 2] = v.z, r.w[4 * i + 3] = v.w;
    }
  } else {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = k + j < K ? ld(row + k + j) : 0.f;
#pragma unroll
    for (int j = 0; j < (int)sizeof(T) * 2; ++j) {
      if constexpr (sizeof(T) == 4) r.w[j] = __float_as_uint(v[j]);
      else r.w[j] = rows::pack2<T>(v[2 * j], v[2 * j + 1]);
    }
  }
}

// A channel's sums of the tokens, scaled, with the bias, stored
template <typename T> __device__ __forceinline__ void finish_step(const Int8Args& a, const uint32_t (&acc)[kStepTokens], const float* scale, int64_t channel) {
  const bool there = channel < a.N;
  float bias = 0.f;
  if (a.bias && there)
    bias = a.bias32 ? ld(reinterpret_cast<const float*>(a.bias) + channel) : ld(reinterpret_cast<const T*>(a.bias) + channel);
  store_tokens<T, kStepTokens, false>(a, acc, scale, there ? ld(a.sw + channel) : 0.f, bias, 0, channel);
}

template <typename T>
__global__ void __launch_bounds__(kGemmThreads, 1)
    int8_step_kernel(const __grid_constant__ CUtensorMap tm_w, const StepArgs x, const Int8Args a) {
  constexpr int S = kStepStages, NT = kStepTokens;
  extern __shared__ uint8_t dyn[];
  __shared__ __align__(8) uint64_t full[S], empty[S], acc_full[2], acc_empty[2], rows_ready, drain;
  __shared__ uint32_t tmem_base, amax[NT];
  __shared__ __align__(16) float scale[NT], factor[NT];
  uint8_t* const ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dyn) + 1023) & ~(uintptr_t)1023);
  uint8_t* const codes = ring + S * kStepTile;
  int32_t* const sums = reinterpret_cast<int32_t*>(codes + kStepTokens * kStepWidest);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // a cluster's blocks are the parts of one tile, and work on no other
  const int part = a.splits > 1 ? blockIdx.x % a.splits : 0, first_tile = blockIdx.x / a.splits, stride = gridDim.x / a.splits;
  const int k0 = (int)((int64_t)a.k_blocks * part / a.splits), k1 = (int)((int64_t)a.k_blocks * (part + 1) / a.splits);

  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tm_w);
    for (int i = 0; i < S; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&acc_full[i], 1), mbar_init(&acc_empty[i], 128);
    mbar_init(&rows_ready, 1), mbar_init(&drain, 1);
    fence_mbar_init();
  }
  if (threadIdx.x >= 64 && threadIdx.x < 64 + NT) amax[threadIdx.x - 64] = 0;
  if (warp == 1) {
    tmem_alloc(&tmem_base, 2 * NT);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncwarp();
  if (a.splits > 1) Group<true>::meet();  // every block of the cluster runs before its memory is written to
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base;
  wait_predecessor();

  uint32_t acc_values[NT];  // a part's sums, kept for the meeting below
  if (warp == 0) {
    if (lane == 0) {
      bool ok = true;
      uint32_t it = 0;
      const uint32_t drop = blockIdx.x == 0 ? (uint32_t)a.drop : ~0u;
      for (int tile = first_tile; tile < a.tiles && ok; tile += stride) {
        for (int k = k0; k < k1; ++k, ++it) {
          const int s = it % S;
          if (it >= (uint32_t)S && !step_wait(&empty[s], ((it / S) & 1) ^ 1, a.limit)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(&full[s], expected(kStepTile, it, drop));
          tma_load_2d(ring + s * kStepTile, &tm_w, &full[s], k * kStep, tile * kChannels);
        }
      }
      const uint32_t last = it > (uint32_t)S ? it - S : 0;
      forgive(full, &drain, S, last, it, drop);
      for (uint32_t i = last; i < it; ++i)
        if (!mbar_wait(&full[i % S], (i / S) & 1, kDrainLimit)) ok = false;
      if (!ok) atomicExch(a.error, 1u);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_i8<NT>();
      uint32_t it = 0, local = 0;
      bool ok = step_wait(&rows_ready, 0, a.limit);
      for (int tile = first_tile; tile < a.tiles && ok; tile += stride, ++local) {
        const uint32_t b = local & 1;
        if (local >= 2 && !step_wait(&acc_empty[b], ((local >> 1) & 1) ^ 1, a.limit)) {
          ok = false;
          break;
        }
        tc_fence_after();
        for (int k = k0; k < k1; ++k, ++it) {
          const int s = it % S;
          if (!step_wait(&full[s], (it / S) & 1, a.limit)) {
            ok = false;
            break;
          }
          tc_fence_after();
          uint64_t da = make_smem_desc(smem_u32(ring + s * kStepTile), 16, 1024, kSwizzle128B);
          uint64_t db = make_smem_desc(smem_u32(codes + (k - k0) * NT * kStep), 16, 1024, kSwizzle128B);
#pragma unroll
          for (int i = 0; i < kStep / 32; ++i, da += 2, db += 2) umma_i8(tmem + b * NT, da, db, idesc, (k > k0 || i > 0) ? 1u : 0u);
          umma_commit(&empty[s]);
        }
        if (ok) umma_commit(&acc_full[b]);
      }
      if (!ok) atomicExch(a.error, 1u);
      drain_mma(&drain, it > 0, a.error);
    }
  } else {
    const int et = threadIdx.x - 64, M = (int)a.M;
    const T* const xp = reinterpret_cast<const T*>(x.x);
    // the rows' largest magnitudes: all rows' loads of a step under way together
    uint32_t m[NT];
#pragma unroll
    for (int r = 0; r < NT; ++r) m[r] = 0;
    for (int k = et * 8; k < x.K; k += kEpilogue * 8) {
      rows::Raw8<T> v[NT];
#pragma unroll
      for (int r = 0; r < NT; ++r)
        if (r < M) load_row8<T>(v[r], xp + r * x.ldx, k, x.K, x.vec);
#pragma unroll
      for (int r = 0; r < NT; ++r)
        if (r < M) {
          uint32_t h[1];
          rows::max_bits<T, rows::EIGHT>(v[r], h);
          m[r] = max(m[r], h[0]);
        }
    }
#pragma unroll
    for (int r = 0; r < NT; ++r)
      if (r < M) {
        const uint32_t v = __reduce_max_sync(0xffffffffu, m[r]);
        if (lane == 0) atomicMax(&amax[r], v);
      }
    epilogue_barrier();
    if (et < NT) scale[et] = et < M ? rows::int8_scale(amax[et]) : 0.f, factor[et] = et < M ? rows::int8_factor(amax[et]) : 0.f;
    epilogue_barrier();
    const int groups = (k1 - k0) * (kStep / 8), all = M * groups;  // of eight elements: a row's, all rows'
    auto convert = [&](auto batch) {
      constexpr int B = decltype(batch)::value;  // groups of a thread whose loads are under way together
      for (int g0 = et; g0 < all; g0 += B * kEpilogue) {
        rows::Raw8<T> v[B];
        int r[B], at[B];
#pragma unroll
        for (int i = 0; i < B; ++i) {
          const int g = min(g0 + i * kEpilogue, all - 1);  // the last one again, with the same result
          r[i] = (uint32_t)g / (uint32_t)groups;
          at[i] = (g - r[i] * groups) * 8;
          load_row8<T>(v[i], xp + r[i] * x.ldx, k0 * kStep + at[i], x.K, x.vec);
        }
#pragma unroll
        for (int i = 0; i < B; ++i) {
          rows::F2 f[4];
          uint32_t q[8];
          rows::to_float<T>(v[i], f);
          rows::int8_codes(f, factor[r[i]], q);
          *reinterpret_cast<uint2*>(codes + (at[i] / kStep) * NT * kStep + sw128_offset(r[i], (at[i] % kStep) / 16) + at[i] % 16) =
              make_uint2(rows::bytes4(q[0], q[1], q[2], q[3]), rows::bytes4(q[4], q[5], q[6], q[7]));
        }
      }
    };
    if (all <= kEpilogue) convert(std::integral_constant<int, 1>());
    else convert(std::integral_constant<int, 4>());
    fence_async_shared();
    epilogue_barrier();
    if (et == 0) mbar_arrive(&rows_ready);

    if (warp < 6) {
      // these four warps have the 32 TMEM lanes, here channels, of their number mod 4
      const int q = warp & 3;
      uint32_t local = 0, limit = a.limit;
      for (int tile = first_tile; tile < a.tiles; tile += stride, ++local) {
        const uint32_t b = local & 1;
        if (!step_wait(&acc_full[b], (local >> 1) & 1, limit)) {
          limit = 1;  // carries on with what is there
          if (lane == 0) atomicExch(a.error, 1u);
        }
        tc_fence_after();
        tmem_ld16(tmem + b * NT + ((uint32_t)(q * 32) << 16), acc_values);
        tmem_wait_ld();
        tc_fence_before();
        mbar_arrive(&acc_empty[b]);
        const int channel = q * 32 + lane;
        if (a.splits == 1) {
          finish_step<T>(a, acc_values, scale, (int64_t)tile * kChannels + channel);
        } else if (part > 0) {
          // to the first block's shared memory
          uint32_t to;
          asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(to) : "r"(smem_u32(sums + (part - 1) * NT * kChannels + channel)));
#pragma unroll
          for (int j = 0; j < NT; ++j)
            if (j < M) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to + j * kChannels * 4), "r"(acc_values[j]) : "memory");
        }
      }
    }
  }
  if (a.splits > 1) {
    __syncwarp();
    Group<true>::meet();  // every part's sums are there
    if (part == 0 && warp >= 2 && warp < 6) {
      const int channel = (warp & 3) * 32 + lane;
      for (int i = 0; i < a.splits - 1; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
          if (j < a.M) acc_values[j] += (uint32_t)sums[(i * NT + j) * kChannels + channel];
      finish_step<T>(a, acc_values, scale, (int64_t)first_tile * kChannels + channel);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 2 * NT);
  }
}

// ---- many tokens ----------------------------------------------------------------------------------------

constexpr int kTokens = 128;    // a block's tokens of a tile
constexpr int kStaged = 4096;   // bytes a warp hands to one TMA store: 32 tokens of 128 bytes
template <bool PAIR, int NC> constexpr int many_rows() { return PAIR ? NC / 2 : NC; }  // weight rows a block loads a stage
template <bool PAIR, int NC> constexpr int many_stage_bytes() { return (kTokens + many_rows<PAIR, NC>()) * kStep; }
template <bool PAIR, int NC> constexpr int many_stages() { return many_rows<PAIR, NC>() == 256 ? 3 : 4; }
// ring | two staged tiles a warp | a warp's channel scales and biases
template <bool PAIR, int NC> constexpr int many_smem() {
  return many_stages<PAIR, NC>() * many_stage_bytes<PAIR, NC>() + kEpilogue / 32 * (2 * kStaged + NC / 2 * 8) + 1024;
}

__device__ __forceinline__ void tma_store_2d(const void* tmap, const void* src, int c0, int c1, uint64_t policy) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group.L2::cache_hint [%0, {%2, %3}], [%1], %4;" ::"l"(tmap),
               "r"(smem_u32(src)), "r"(c0), "r"(c1), "l"(policy)
               : "memory");
}

// A tile is 128 tokens x NC channels, or with PAIR 256 x NC for two blocks of a cluster: each loads its own tokens
// and half of the channels' weight rows.
template <bool PAIR, int NC, typename T>
__global__ void __launch_bounds__(kGemmThreads, 1)
    int8_many_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x,
                     const __grid_constant__ CUtensorMap tm_out, const Int8Args a) {
  using G = Group<PAIR>;
  constexpr int S = many_stages<PAIR, NC>(), BLOCKS = PAIR ? 2 : 1, ROWS = many_rows<PAIR, NC>();
  constexpr uint32_t kBytes = many_stage_bytes<PAIR, NC>();
  extern __shared__ uint8_t dyn[];
  // other_done: in the first block, the second one's loader has issued its last load
  __shared__ __align__(8) uint64_t full[S], empty[S], acc_full[2], acc_empty[2], drain, other_done;
  __shared__ uint32_t tmem_base;
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dyn) + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int place_in_pair = PAIR ? blockIdx.x & 1 : 0, worker = blockIdx.x / BLOCKS, workers = gridDim.x / BLOCKS;

  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tm_w);
    tma_prefetch_desc(&tm_x);
    tma_prefetch_desc(&tm_out);
    for (int i = 0; i < S; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&acc_full[i], 1), mbar_init(&acc_empty[i], BLOCKS * kEpilogue / 32);
    mbar_init(&drain, 1), mbar_init(&other_done, 1);
    fence_mbar_init();
  }
  if (warp == 1) {
    G::alloc(&tmem_base, 2 * NC);
    G::relinquish();
  }
  tc_fence_before();
  __syncwarp();
  G::meet();
  tc_fence_after();
  const uint32_t tmem = tmem_base;
  const int m_tiles = a.tiles / a.n_tiles;
  // this block's tokens, and the tile's channels
  auto place = [&](int tile, int& m0, int& n0) {
    // a.group tiles of tokens go through all channels together
    const int g = tile / (a.group * a.n_tiles), in = tile - g * a.group * a.n_tiles;
    const int rows = min(a.group, m_tiles - g * a.group);
    m0 = ((g * a.group + in % rows) * BLOCKS + place_in_pair) * kTokens;
    n0 = in / rows * NC;
  };

  if (warp == 0) {
    if (lane == 0) {
      bool ok = true;
      uint32_t it = 0;
      const uint32_t drop = worker == 0 && place_in_pair == 0 ? (uint32_t)a.drop : ~0u;
      wait_predecessor();
      for (int tile = worker; tile < a.tiles && ok; tile += workers) {
        int m0, n0;
        place(tile, m0, n0);
        if (PAIR) n0 += place_in_pair * ROWS;
        for (int k = 0; k < a.k_blocks; ++k, ++it) {
          const int s = it % S;
          if (it >= (uint32_t)S && !step_wait(&empty[s], ((it / S) & 1) ^ 1, a.limit)) {
            ok = false;
            break;
          }
          uint8_t* st = ring + (size_t)s * kBytes;
          // the first block expects both blocks' bytes (the other's may land before: the count goes below zero)
          if (place_in_pair == 0) mbar_arrive_expect_tx(&full[s], expected(BLOCKS * kBytes, it, drop));
          G::load(st, &tm_x, &full[s], k * kStep, m0);
          G::load(st + kTokens * kStep, &tm_w, &full[s], k * kStep, n0);
        }
      }
      const uint32_t last = it > (uint32_t)S ? it - S : 0;
      const bool complete = ok;
      if (place_in_pair == 0) {
        // both blocks' copies count here: the other block waits for this one at the end
        uint32_t landed = 0;  // of the ring's stages
        forgive(full, &drain, S, last, it, drop);
        for (uint32_t i = last; i < it; ++i) {
          if (mbar_wait(&full[i % S], (i / S) & 1, kDrainLimit)) landed |= 1u << (i % S);
          else ok = false;
        }
        if (PAIR && !complete && mbar_wait(&other_done, 0, kDrainLimit)) {
          // The other block's wait may have seen what this one's gave up on: its copies for up to a ring of further steps
          // come down on barriers where nothing expects them yet. (It issued none where the last one there has not landed.)
          for (uint32_t i = it; i < it + S; ++i) {
            if (!(landed >> (i % S) & 1)) continue;
            mbar_arrive_expect_tx(&full[i % S], kBytes);
            mbar_wait(&full[i % S], (i / S) & 1, kDrainLimit >> 6);  // runs out where it issued none
          }
        }
      } else {
        G::arrive_first(&other_done);
      }
      if (PAIR) {
        // the first block's arrivals at this block's barriers are all in before the block ends
        if (complete)
          for (uint32_t i = last; i < it; ++i)
            if (!step_wait(&empty[i % S], (i / S) & 1, a.limit)) ok = false;
        if (place_in_pair == 1 && !mbar_wait(&drain, 0, kDrainLimit)) ok = false;
      }
      if (!ok) atomicExch(a.error, 1u);
    }
  } else if (warp == 1) {
    if (lane == 0 && place_in_pair == 0) {
      constexpr uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(NC >> 3) << 17) | ((uint32_t)(BLOCKS * kTokens >> 4) << 24);
      uint32_t it = 0, local = 0;
      bool ok = true;
      wait_predecessor();
      for (int tile = worker; tile < a.tiles && ok; tile += workers, ++local) {
        const uint32_t b = local & 1;
        if (local >= 2 && !step_wait(&acc_empty[b], ((local >> 1) & 1) ^ 1, a.limit)) {
          ok = false;
          break;
        }
        tc_fence_after();
        for (int k = 0; k < a.k_blocks; ++k, ++it) {
          const int s = it % S;
          if (!step_wait(&full[s], (it / S) & 1, a.limit)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t at = smem_u32(ring + (size_t)s * kBytes);
          uint64_t da = make_smem_desc(at, 16, 1024, kSwizzle128B);
          uint64_t db = make_smem_desc(at + kTokens * kStep, 16, 1024, kSwizzle128B);
#pragma unroll
          for (int i = 0; i < kStep / 32; ++i, da += 2, db += 2) G::mma(tmem + b * NC, da, db, idesc, (k > 0 || i > 0) ? 1u : 0u);
          G::commit(&empty[s]);
        }
        if (ok) G::commit(&acc_full[b]);
      }
      if (it > 0) G::commit(&drain);
      else G::arrive_all(&drain);
      if (!mbar_wait(&drain, 0, kDrainLimit)) ok = false;
      if (!ok) atomicExch(a.error, 1u);
    }
  } else {
    // a warp has the 32 TMEM lanes, here tokens, of its number mod 4, and half of the channels. (16 warps with a quarter
    // each and one staged tile took 423 us instead of 369, in short runs, for 16384 x 768 x 32000.)
    constexpr int COLS = NC / 2, STEPS = COLS / 32, kWords = 32 * (int)sizeof(T) / 16;  // 16-byte words a lane stages a step
    const int q = warp & 3, first = (warp - 2) / 4 * COLS;
    uint8_t* const mine = ring + (size_t)S * kBytes + (size_t)(warp - 2) * (2 * kStaged);
    float* const sw = reinterpret_cast<float*>(ring + (size_t)S * kBytes + (size_t)(kEpilogue / 32) * (2 * kStaged)) + (warp - 2) * 2 * COLS;
    float* const sb = sw + COLS;
    uint32_t local = 0, limit = a.limit, stores = 0;
    uint64_t policy;
    if (a.stream_out) asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
    else asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(policy));
    wait_predecessor();
    for (int tile = worker; tile < a.tiles; tile += workers, ++local) {
      const uint32_t b = local & 1;
      int m0, n0;
      place(tile, m0, n0);
      n0 += first;
      const int token = m0 + q * 32 + lane;
      const float sx = token < a.M ? ld(a.sx + token) : 0.f;
      const bool any_large = __any_sync(0xffffffffu, fabsf(sx) > kLargeScale);
      // all loads before the first store, which they might otherwise have to wait for
      float channel_scale[COLS / 32], channel_bias[COLS / 32];
#pragma unroll
      for (int c = 0; c < COLS / 32; ++c) {
        const int64_t n = n0 + c * 32 + lane;
        const bool there = n < a.N;
        channel_scale[c] = there ? ld(a.sw + n) : 0.f;
        channel_bias[c] = 0.f;
        if (a.bias && there) channel_bias[c] = a.bias32 ? ld(reinterpret_cast<const float*>(a.bias) + n) : ld(reinterpret_cast<const T*>(a.bias) + n);
      }
      __syncwarp();
#pragma unroll
      for (int c = 0; c < COLS / 32; ++c) sw[c * 32 + lane] = channel_scale[c], sb[c * 32 + lane] = channel_bias[c];
      __syncwarp();
      if (!step_wait(&acc_full[b], (local >> 1) & 1, limit)) {
        limit = 1;  // carries on with what is there
        if (lane == 0) atomicExch(a.error, 1u);
      }
      tc_fence_after();
      const uint32_t acc = tmem + b * NC + first + ((uint32_t)(q * 32) << 16);
      uint32_t v[2][32];
      tmem_ld32(acc, v[0]);
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        tmem_wait_ld();
        if (i + 1 < STEPS) {
          tmem_ld32(acc + (i + 1) * 32, v[(i + 1) & 1]);
        } else {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) G::arrive_first(&acc_empty[b]);
        }
        // the staged tile of 32 tokens x 128 bytes is full after one step of float32, two of 16-bit types
        constexpr int kPer = 128 / (kWords * 16);
        uint8_t* const staged = mine + (stores & 1) * kStaged;
        if (i % kPer == 0) {
          // the store before the last one has read its bytes
          if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
          __syncwarp();
        }
        uint32_t w[kWords * 4];
        auto put = [&](int j, float2 p, float2 r) {
          if constexpr (sizeof(T) == 4) {
            w[j] = __float_as_uint(p.x), w[j + 1] = __float_as_uint(p.y), w[j + 2] = __float_as_uint(r.x), w[j + 3] = __float_as_uint(r.y);
          } else {
            w[j / 2] = rows::pack2<T>(p.x, p.y), w[j / 2 + 1] = rows::pack2<T>(r.x, r.y);
          }
        };
        if (!any_large) {
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const float4 s = *reinterpret_cast<const float4*>(sw + i * 32 + j), t = *reinterpret_cast<const float4*>(sb + i * 32 + j);
            const rows::F2 x = rows::f2(sx);
            const rows::F2 lo = rows::fma2(rows::mul2(rows::f2(__int2float_rn((int)v[i & 1][j]), __int2float_rn((int)v[i & 1][j + 1])), x),
                                           rows::f2(s.x, s.y), rows::f2(t.x, t.y));
            const rows::F2 hi = rows::fma2(rows::mul2(rows::f2(__int2float_rn((int)v[i & 1][j + 2]), __int2float_rn((int)v[i & 1][j + 3])), x),
                                           rows::f2(s.z, s.w), rows::f2(t.z, t.w));
            put(j, rows::split(lo), rows::split(hi));
          }
        } else {
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const float4 s = *reinterpret_cast<const float4*>(sw + i * 32 + j), t = *reinterpret_cast<const float4*>(sb + i * 32 + j);
            put(j, make_float2(scaled(v[i & 1][j], sx, s.x, t.x), scaled(v[i & 1][j + 1], sx, s.y, t.y)),
                make_float2(scaled(v[i & 1][j + 2], sx, s.z, t.z), scaled(v[i & 1][j + 3], sx, s.w, t.w)));
          }
        }
#pragma unroll
        for (int j = 0; j < kWords; ++j)
          *reinterpret_cast<uint4*>(staged + sw128_offset(lane, (i % kPer) * kWords + j)) =
              make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
        if (i % kPer == kPer - 1) {
          fence_async_shared();
          __syncwarp();
          // a store that starts outside the output is left out; one that ends outside is cut there
          if (lane == 0) {
            const int c = n0 + (i / kPer) * kPer * 32;
            if (c < a.N && m0 + q * 32 < a.M) tma_store_2d(&tm_out, staged, c, m0 + q * 32, policy);
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
          ++stores;
        }
      }
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  tc_fence_before();
  __syncwarp();
  G::meet();
  if (warp == 1) {
    tc_fence_after();
    G::dealloc(tmem, 2 * NC);
  }
}

// Orders of the tiles, of 126 MB of L2. A weight that stays there is best gone through once for each tile of tokens: the
// blocks then write whole rows of the output (16384 x 768 x 32000: 398 / 463 us, with 16 tiles of tokens at once 419 / 475; an
// output too large for L2 leaves it first, with the default policy 436 / 496). A larger one would come from
// memory each time: 16 tiles of tokens at once (8192 x 4096 x 32000, 131 MB: 712 / 823 us against 857 / 1073).
constexpr int64_t kWeightInL2 = 48 << 20;
constexpr size_t kOutputInL2 = 64 << 20;

// Which kernel, its tile's other side (NT or NC), and parts of a tile's K range.
struct GemmShape {
  bool step = false, many = false, pair = false;
  int width, n_tiles, tiles, splits;
};
GemmShape gemm_shape(int64_t M, int64_t N, int64_t K, bool rows_on_16, bool from_x) {
  GemmShape g;
  const int64_t sms = num_sms(), m_tiles = (M + kTokens - 1) / kTokens;
  auto tiles = [&](int nc) { return m_tiles * ((N + nc - 1) / nc); };
  // The kernel for many tokens where its smaller tiles fill the SMs once over and its stores can be made.
  g.many = rows_on_16 && M > 64 && tiles(128) >= sms;
  if (g.many) {
    // Pairs of blocks load a third less for each product, but start later and hand over tiles between them: for more
    // tiles than SMs with K of 1024 on (8192 x 1024 x 8192: 58 / 69 us against 63 / 74, 8192 x 4096 x 4096: 93 / 107 against
    // 106 / 120; 8192 x 768 x 8192: 53 / 62 against 51 / 60, 1000 x 4096 x 4096: 17.6 / 16.9 against 16.8 / 17.0).
    g.pair = sms % 2 == 0 && K >= 1024 && tiles(256) > sms;
    // Of a block's own tiles those whose rounds over the SMs cost least, a K step of a tile costing the rows that it
    // loads (2931 x 768 x 2304: 10.1 us with 256 channels, 11.6 with 128; 300 x 4096 x 4096: 15.4 and 15.3).
    auto cost = [&](int nc) { return (tiles(nc) + sms - 1) / sms * (kTokens + nc); };
    g.width = g.pair || cost(256) <= cost(128) ? 256 : 128;
    g.n_tiles = (int)((N + g.width - 1) / g.width);
    g.tiles = (int)(g.pair ? (M + 255) / 256 * g.n_tiles : tiles(g.width));
    g.splits = 1;
    return g;
  }
  g.width = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : 128;
  g.n_tiles = (int)((N + kChannels - 1) / kChannels);
  g.tiles = (int)((M + g.width - 1) / g.width * g.n_tiles);
  // Fewer tiles than SMs: parts of K, as many as fill them, but no more than pay: of p parts each loads blocks / p steps
  // of (128 + NT) x 128 bytes, and the last one adds up p x NT x 128 sums, 4 bytes each, so that p = sqrt(blocks (128 +
  // NT) / (4 NT)) has the least of both (100 x 8000 x 100: 19 us with 6 parts, 101 with 63).
  const int64_t blocks = (K + kStep - 1) / kStep;
  const int64_t pay = std::max<int64_t>(1, std::llround(std::sqrt((double)blocks * (kChannels + g.width) / (4.0 * g.width))));
  g.splits = (int)std::max<int64_t>(1, std::min<int64_t>(std::min(blocks, pay), sms / g.tiles));
  // A decoding step's kernel while x is small: every one of its blocks goes through all of it (1 x 768 x 32000: 8.4 us
  // against 10.1 with a launch of its own for the rows, and 3 us less for the host; 8 x 2048 x 2048: 8.0 and 8.9;
  // 16 x 4096 x 4096: 12.7 and 10.8; 8 x 4096 x 16000: 18.4 and 15.9).
  g.step = from_x && M <= kStepTokens && K <= kStepWidest && M * K <= (g.tiles <= 64 ? 16384 : 8192);
  // clusters of 2, 4 or 8 blocks, no more of them than run at once (16 of 8 did not: 1 x 2048 x 2048 took 11.7 us)
  if (g.step) g.splits = g.splits >= 8 && g.tiles <= 8 ? 8 : g.splits >= 4 && g.tiles <= 32 ? 4 : g.splits >= 2 && g.tiles <= 64 ? 2 : 1;
  return g;
}

// Workspace: [error, counts] | codes and scales of the tokens (when they are quantised here) | parts
struct GemmWs {
  size_t counts, codes, scale, parts, bytes;
};
GemmWs gemm_ws(const GemmShape& g, int64_t M, int64_t K, bool quantise) {
  auto al = [](size_t x) { return (x + 255) & ~(size_t)255; };
  GemmWs w;
  w.counts = 4;
  size_t off = al(4 + (g.splits > 1 ? (size_t)g.tiles * 4 : 0));
  w.codes = off;
  off += quantise && !g.step ? al((size_t)M * rows::code_pitch(K)) : 0;
  w.scale = off;
  off += quantise && !g.step ? al((size_t)M * 4) : 0;
  w.parts = off;
  off += g.splits > 1 && !g.step ? (size_t)g.tiles * g.splits * g.width * kChannels * 4 : 0;
  w.bytes = off;
  return w;
}

// units: of work; blocks: of a cluster that shares one. overlap: the kernel may start while the one before it drains.
template <typename... K, typename... A>
int launch(void (*k)(K...), int64_t units, int blocks, int smem, const Int8Args& a, bool overlap, cudaStream_t s, const A&... args) {
  int st = ensure_dyn_smem(reinterpret_cast<const void*>(k), smem, "int8_linear shared memory");
  if (st != FLB_OK) return st;
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)std::min<int64_t>(units * blocks, num_sms() / blocks * blocks));
  cfg.blockDim = dim3(kGemmThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  if (overlap) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (blocks > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = blocks;
    attr[cfg.numAttrs].val.clusterDim.y = 1;
    attr[cfg.numAttrs++].val.clusterDim.z = 1;
  }
  const cudaError_t e = cudaLaunchKernelEx(&cfg, k, args..., a);
  count_launches(1);
  return check_cuda(e, "int8_linear launch");
}

template <int NT, typename T>
int launch_few(const CUtensorMap& tw, const CUtensorMap& tx, const Int8Args& a, bool overlap, cudaStream_t s) {
  return launch(int8_few_kernel<NT, T>, (int64_t)a.tiles * a.splits, 1, stages<NT>() * stage_bytes<NT>() + 1024, a, overlap, s, tw, tx);
}

template <bool PAIR, int NC, typename T>
int launch_many(const CUtensorMap& tw, const CUtensorMap& tx, const CUtensorMap& to, const Int8Args& a, bool overlap, cudaStream_t s) {
  return launch(int8_many_kernel<PAIR, NC, T>, a.tiles, PAIR ? 2 : 1, many_smem<PAIR, NC>(), a, overlap, s, tw,
                tx, to);
}

template <typename T>
int launch_t(const GemmShape& g, const CUtensorMap& tw, const CUtensorMap& tx, const Int8Args& a, bool overlap, cudaStream_t s) {
  if (g.many) {
    CUtensorMap to;
    const uint64_t dims[2] = {(uint64_t)a.N, (uint64_t)a.M};
    const uint64_t strides[1] = {(uint64_t)a.N * sizeof(T)};
    const uint32_t box[2] = {128 / sizeof(T), 32};
    const CUtensorMapDataType dt = sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const int st = make_tmap(&to, a.out, dt, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
    if (st != FLB_OK) return st;
    if (g.pair) return launch_many<true, 256, T>(tw, tx, to, a, overlap, s);
    if (g.width == 256) return launch_many<false, 256, T>(tw, tx, to, a, overlap, s);
    return launch_many<false, 128, T>(tw, tx, to, a, overlap, s);
  }
  switch (g.width) {
    case 16: return launch_few<16, T>(tw, tx, a, overlap, s);
    case 32: return launch_few<32, T>(tw, tx, a, overlap, s);
    case 64: return launch_few<64, T>(tw, tx, a, overlap, s);
    default: return launch_few<128, T>(tw, tx, a, overlap, s);
  }
}

int code_map(CUtensorMap* m, const int8_t* codes, int64_t rows, int64_t ld, int64_t K, int box_rows) {
  const uint64_t dims[2] = {(uint64_t)K, (uint64_t)rows};
  const uint64_t strides[1] = {(uint64_t)ld};
  const uint32_t box[2] = {kStep, (uint32_t)box_rows};
  return make_tmap(m, codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

}  // namespace

int int8_rows(const void* x, int64_t ldx, int8_t* codes, float* scale, int64_t R, int64_t D, int dtype, uint32_t* zero,
              int64_t n_zero, cudaStream_t s);

// For either kernel: which one runs also depends on where the output lies.
size_t int8_linear_workspace_bytes(int64_t M, int64_t N, int64_t K, bool quantise) {
  return std::max(gemm_ws(gemm_shape(M, N, K, false, quantise), M, K, quantise).bytes,
                  gemm_ws(gemm_shape(M, N, K, true, quantise), M, K, quantise).bytes);
}

int int8_linear(const void* x, int64_t ldx, const int8_t* x_codes, int64_t ldc, const float* x_scale, const int8_t* w_codes,
                int64_t ldw, const float* w_scale, const void* bias, int bias_dtype, void* out, int64_t M, int64_t N,
                int64_t K, int dtype, void* ws, int check_timeout, int drop, uint32_t limit, cudaStream_t s) {
  const GemmShape g = gemm_shape(M, N, K, N * dtype_size(dtype) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0,
                                 x != nullptr);
  const GemmWs l = gemm_ws(g, M, K, x != nullptr);
  uint8_t* p = reinterpret_cast<uint8_t*>(ws);
  const int64_t n_zero = 1 + (g.splits > 1 ? g.tiles : 0);
  const bool reset = g.step ? check_timeout != 0 : !x && (g.splits > 1 || check_timeout);
  int st;
  if (x && !g.step) {
    // the rows' kernel clears the error word and the counts too
    int8_t* codes = reinterpret_cast<int8_t*>(p + l.codes);
    float* scale = reinterpret_cast<float*>(p + l.scale);
    if ((st = int8_rows(x, ldx, codes, scale, M, K, dtype, reinterpret_cast<uint32_t*>(p), n_zero, s)) != FLB_OK) return st;
    x_codes = codes, x_scale = scale, ldc = rows::code_pitch(K);
  } else if (reset) {  // otherwise nothing reads those words
    if ((st = check_cuda(cudaMemsetAsync(p, 0, n_zero * 4, s), "int8_linear reset")) != FLB_OK) return st;
  }
  CUtensorMap tw, tx = {};
  if ((st = code_map(&tw, w_codes, N, ldw, K, g.many ? (g.pair ? g.width / 2 : g.width) : kChannels)) != FLB_OK) return st;
  if (!g.step && (st = code_map(&tx, x_codes, M, ldc, K, g.many ? kTokens : g.width)) != FLB_OK) return st;
  Int8Args a = {};
  a.sx = x_scale, a.sw = w_scale, a.bias = bias, a.bias32 = bias_dtype == FLB_F32;
  a.out = out, a.M = M, a.N = N;
  a.pairs = N % 2 == 0 && reinterpret_cast<uintptr_t>(out) % 4 == 0;
  a.early = x != nullptr;
  a.k_blocks = (int)((K + kStep - 1) / kStep), a.n_tiles = g.n_tiles, a.tiles = g.tiles, a.splits = g.splits;
  a.group = N * K <= kWeightInL2 ? 1 : 16;
  a.stream_out = (size_t)M * N * dtype_size(dtype) > kOutputInL2;
  a.parts = reinterpret_cast<int32_t*>(p + l.parts), a.counts = reinterpret_cast<uint32_t*>(p + l.counts);
  a.error = reinterpret_cast<uint32_t*>(p);
  a.limit = limit ? limit : kWaitLimit, a.drop = drop;
  const StepArgs sa{x, ldx, K % 8 == 0 && ldx * dtype_size(dtype) % 16 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0, (int)K};
  if (g.step) {
    switch (dtype) {
      case FLB_F32: st = launch(int8_step_kernel<float>, g.tiles, g.splits, kStepSmem, a, !reset, s, tw, sa); break;
      case FLB_F16: st = launch(int8_step_kernel<__half>, g.tiles, g.splits, kStepSmem, a, !reset, s, tw, sa); break;
      default: st = launch(int8_step_kernel<__nv_bfloat16>, g.tiles, g.splits, kStepSmem, a, !reset, s, tw, sa); break;
    }
  } else switch (dtype) {
    case FLB_F32: st = launch_t<float>(g, tw, tx, a, !reset, s); break;
    case FLB_F16: st = launch_t<__half>(g, tw, tx, a, !reset, s); break;
    default: st = launch_t<__nv_bfloat16>(g, tw, tx, a, !reset, s); break;
  }
  if (st != FLB_OK || !check_timeout) return st;
  uint32_t err = 0;
  if ((st = check_cuda(cudaMemcpyAsync(&err, p, 4, cudaMemcpyDeviceToHost, s), "int8_linear error word")) != FLB_OK) return st;
  if ((st = check_cuda(cudaStreamSynchronize(s), "int8_linear error word")) != FLB_OK) return st;
  return err ? fail(FLB_ERR_TIMEOUT, "int8_linear: a bounded wait in the kernel gave up") : FLB_OK;
}

}  // namespace flb
