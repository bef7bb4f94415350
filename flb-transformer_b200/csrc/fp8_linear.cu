// Product of rows in 8-bit floating point: out[m, n] = sum over blocks b of 128 of 2^(ex[m, b] + ew[n, b]) times the sum over
// the block of X[m, k] W[n, k], plus bias[n].
//
// tcgen05.mma kind::mxf8f6f4 with a block scale: the tensor core multiplies by the powers of two as it goes (they lie in
// tensor memory, a byte for each row and block; the instruction's scale of 32 elements is given four times the same
// byte). One block a SM, persistent over units of work: a tile of 128 tokens and 64, 128 or 192 channels, or a part of its
// K range. Warp 0 loads by TMA into a ring of four steps of 128 of K, warp 1 issues the MMAs, the others read TMEM:
// each has 32 tokens, a lane a token, and 64 channels, in registers.
//
// The tensor core cuts, and does not round, what it adds to an accumulator: over 16384 of K sums came out 6.5e-6 of
// their size too small. So an accumulator takes 1024 of K, and the warps add up those sums in float32, rounded.
// Two accumulators: one is read while the other is filled.
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
constexpr int kStages = 4;
constexpr int kChunk = 8;         // steps that one accumulator takes
constexpr int kCols = 64;         // channels of an epilogue warp
constexpr int kStaged = 4096;     // bytes a warp stages for a store: 32 tokens of 128 bytes
constexpr uint32_t kWaitLimit = 1u << 20;   // polls, each held for about 4 us by the hardware: 4 s
constexpr uint32_t kDrainLimit = 1u << 20;  // the same for what is still in flight when a block ends early

template <int NC> constexpr int epilogue_warps() { return NC / 16; }  // 4 quarters of TMEM's lanes x NC / 64
template <int NC> constexpr int threads() { return 64 + 32 * epilogue_warps<NC>(); }
template <int NC> constexpr int stage_bytes() { return (kTokens + NC) * kStep; }
// ring | its powers of two | staged tiles | biases
constexpr int kExpBytes = 3 * kTileBytes;  // a stage's: of the tokens, and of up to two groups of 128 channels
template <int NC> constexpr int smem_bytes() {
  return kStages * (stage_bytes<NC>() + kExpBytes) + epilogue_warps<NC>() * (kStaged + kCols * 4) + 1024;
}
// Tensor memory: two accumulators, then kStages sets of powers of two (4 columns of the tokens', 8 of the channels')
template <int NC> constexpr uint32_t tmem_cols() { return NC > 64 ? 512 : 256; }
constexpr int kExpCols = 12;

struct Args {
  const uint8_t *ex, *ew;
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
};

__device__ __forceinline__ bool step_wait(uint64_t* bar, uint32_t phase) { return mbar_try_wait(bar, phase) || mbar_wait(bar, phase, kWaitLimit); }

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes),
               "r"(smem_u32(bar))
               : "memory");
}
// 32 rows of 16 bytes to TMEM lanes 0 to 31, four columns, and the same to the other three quarters
__device__ __forceinline__ void copy_exps(uint32_t tmem, const void* src) {
  const uint64_t d = make_smem_desc(smem_u32(src), 16, 128, kSwizzleNone);
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(d) : "memory");
}
// e4m3 operands, both K-major, float32 accumulators, powers of two as scales; which of the four bytes of a scale's word
template <int NC> __device__ __forceinline__ uint32_t idesc(uint32_t byte) {
  return (byte << 4) | ((uint32_t)(NC >> 3) << 17) | (1u << 23) | ((uint32_t)(kTokens >> 7) << 27) | (byte << 29);
}
__device__ __forceinline__ void umma_fp8(uint32_t d, uint64_t da, uint64_t db, uint32_t desc, uint32_t ea, uint32_t eb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
      "l"(da), "l"(db), "r"(desc), "r"(ea), "r"(eb), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tma_store_2d(const void* tmap, const void* src, int c0, int c1, uint64_t policy) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group.L2::cache_hint [%0, {%2, %3}], [%1], %4;" ::"l"(tmap),
               "r"(smem_u32(src)), "r"(c0), "r"(c1), "l"(policy)
               : "memory");
}
template <int NC> __device__ __forceinline__ void epilogue_barrier() {
  asm volatile("bar.sync 1, %0;" ::"n"(epilogue_warps<NC>() * 32) : "memory");
}

template <int NC, typename T>
__global__ void __launch_bounds__(threads<NC>(), 1)
    fp8_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_out,
               const Args a) {
  constexpr int S = kStages, EW = epilogue_warps<NC>();
  constexpr uint32_t kExpTmem = 2 * NC;
  extern __shared__ uint8_t dyn[];
  __shared__ __align__(8) uint64_t full[S], empty[S], acc_full[2], acc_empty[2], drain;
  __shared__ uint32_t tmem_base, last_flag;
  uint8_t* const ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dyn) + 1023) & ~(uintptr_t)1023);
  uint8_t* const staged_all = ring + (size_t)S * stage_bytes<NC>();  // 1024-byte aligned: 128-byte swizzled tiles
  uint8_t* const exps = staged_all + EW * kStaged;
  float* const bias_all = reinterpret_cast<float*>(exps + S * kExpBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tm_x);
    tma_prefetch_desc(&tm_w);
    for (int i = 0; i < S; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&acc_full[i], 1), mbar_init(&acc_empty[i], EW);
    mbar_init(&drain, 1);
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(&tmem_base, tmem_cols<NC>());
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base;

  const int units = a.tiles * a.splits, m_tiles = a.tiles / a.n_tiles;
  // a unit's tokens, channels and steps of K
  auto place = [&](int u, int& m0, int& n0, int& k0, int& k1) {
    const int tile = u / a.splits, split = u - tile * a.splits;
    const int g = tile / (a.group * a.n_tiles), in = tile - g * a.group * a.n_tiles, rows = min(a.group, m_tiles - g * a.group);
    m0 = (g * a.group + in % rows) * kTokens;
    n0 = in / rows * NC;
    k0 = (int)((int64_t)a.k_blocks * split / a.splits);
    k1 = (int)((int64_t)a.k_blocks * (split + 1) / a.splits);
  };
  const int groups_x = (int)blocks_of(a.M), groups_w = (int)blocks_of(a.N);
  // groups of 128 channels' powers of two that a tile reaches: one or two, from n0 / 128 on
  auto groups_of = [&](int n0) { return min((n0 + NC - 1) / kBlock, groups_w - 1) - n0 / kBlock + 1; };

  if (warp == 0) {
    if (lane == 0) {
      bool ok = true;
      uint32_t it = 0, early = 0;
      auto load_w = [&](int s, int n0, int k, bool first) {
        uint8_t* const st = ring + (size_t)s * stage_bytes<NC>();
        tma_load_2d(st + kTokens * kStep, &tm_w, &full[s], k * kStep, n0);
        if (first)
          for (int g = 0; g < groups_of(n0); ++g)
            bulk_load(exps + s * kExpBytes + (1 + g) * kTileBytes, a.ew + ((int64_t)(n0 / kBlock + g) * a.quads + k / 4) * kTileBytes, kTileBytes, &full[s]);
      };
      // the powers of two of four steps come with the first of them
      auto bytes = [&](int n0, bool first) { return (uint32_t)((a.a_rows + NC) * kStep + (first ? (1 + groups_of(n0)) * kTileBytes : 0)); };
      // Where the kernel that this one may overlap is the one that makes X's codes, the weight was written before that
      // kernel started: a first ring of weight tiles is on its way before the wait.
      for (int u = blockIdx.x; a.early && u < units && early < (uint32_t)S; u += gridDim.x) {
        int m0, n0, k0, k1;
        place(u, m0, n0, k0, k1);
        for (int k = k0; k < k1 && early < (uint32_t)S; ++k, ++early) {
          const bool first = k == k0 || k % 4 == 0;
          mbar_arrive_expect_tx(&full[early], bytes(n0, first));
          load_w(early, n0, k, first);
        }
      }
      wait_predecessor();
      for (int u = blockIdx.x; u < units && ok; u += gridDim.x) {
        int m0, n0, k0, k1;
        place(u, m0, n0, k0, k1);
        for (int k = k0; k < k1; ++k, ++it) {
          const int s = it % S;
          const bool first = k == k0 || k % 4 == 0;
          if (it >= early) {
            if (it >= (uint32_t)S && !step_wait(&empty[s], ((it / S) & 1) ^ 1)) {
              ok = false;
              break;
            }
            mbar_arrive_expect_tx(&full[s], bytes(n0, first));
            load_w(s, n0, k, first);
          }
          tma_load_2d(ring + (size_t)s * stage_bytes<NC>(), &tm_x, &full[s], k * kStep, m0);
          if (first) bulk_load(exps + s * kExpBytes, a.ex + ((int64_t)(m0 / kBlock) * a.quads + k / 4) * kTileBytes, kTileBytes, &full[s]);
        }
      }
      for (uint32_t i = it > (uint32_t)S ? it - S : 0; i < it; ++i)
        if (!mbar_wait(&full[i % S], (i / S) & 1, kDrainLimit)) ok = false;
      if (!ok) atomicExch(a.error, 1u);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      // A set of powers of two is written again after S others, so S steps at least: the step that does it has waited for
      // a stage whose copies began when all MMAs up to S steps before, its readers among them, were done.
      uint32_t it = 0, local = 0, set = 0;
      bool ok = true;
      wait_predecessor();
      for (int u = blockIdx.x; u < units && ok; u += gridDim.x) {
        int m0, n0, k0, k1;
        place(u, m0, n0, k0, k1);
        uint32_t at = 0;
        for (int k = k0; k < k1; ++k, ++it) {
          const int s = it % S;
          const uint32_t b = local & 1;
          const bool opens = (k - k0) % kChunk == 0;
          if (opens) {
            if (local >= 2 && !step_wait(&acc_empty[b], ((local >> 1) & 1) ^ 1)) {
              ok = false;
              break;
            }
          }
          if (!step_wait(&full[s], (it / S) & 1)) {
            ok = false;
            break;
          }
          tc_fence_after();
          if (k == k0 || k % 4 == 0) {
            at = tmem + kExpTmem + set % S * kExpCols;
            ++set;
            copy_exps(at, exps + s * kExpBytes);
            for (int g = 0; g < groups_of(n0); ++g) copy_exps(at + 4 + 4 * g, exps + s * kExpBytes + (1 + g) * kTileBytes);
          }
          const uint32_t from = smem_u32(ring + (size_t)s * stage_bytes<NC>());
          uint64_t da = make_smem_desc(from, 16, 1024, kSwizzle128B), db = make_smem_desc(from + kTokens * kStep, 16, 1024, kSwizzle128B);
          const uint32_t desc = idesc<NC>(k & 3), eb = at + 4 + n0 % kBlock / 32;
#pragma unroll
          for (int i = 0; i < kStep / 32; ++i, da += 2, db += 2) umma_fp8(tmem + b * NC, da, db, desc, at, eb, (!opens || i > 0) ? 1u : 0u);
          umma_commit(&empty[s]);
          if ((k - k0) % kChunk == kChunk - 1 || k == k1 - 1) {
            umma_commit(&acc_full[b]);
            ++local;
          }
        }
      }
      if (it > 0) umma_commit(&drain);
      else mbar_arrive(&drain);
      if (!mbar_wait(&drain, 0, kDrainLimit)) ok = false;
      if (!ok) atomicExch(a.error, 1u);
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
    for (int u = blockIdx.x; u < units; u += gridDim.x) {
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
        if (ok && !step_wait(&acc_full[b], (local >> 1) & 1)) {
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
        if (lane == 0) mbar_arrive(&acc_empty[b]);
#pragma unroll
        for (int j = 0; j < 32; ++j) sum[32 + j] = k == k0 ? __uint_as_float(v[j]) : sum[32 + j] + __uint_as_float(v[j]);
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
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, tmem_cols<NC>());
  }
}

struct Shape {
  int width, n_tiles, tiles, splits;
};
// The tile's channels and parts of K whose rounds over the SMs cost least: a step the rows that it loads, a unit its start and
// epilogue, a part its way through memory and back.
Shape shape_of(int64_t M, int64_t N, int64_t K) {
  const int64_t sms = num_sms(), m_tiles = (M + kTokens - 1) / kTokens, blocks = blocks_of(K);
  Shape best = {};
  double least = INFINITY;
  for (int nc : {192, 128, 64}) {
    const int64_t n_tiles = (N + nc - 1) / nc, tiles = m_tiles * n_tiles;
    for (int64_t splits = 1; splits <= std::min<int64_t>(blocks, std::max<int64_t>(1, sms / tiles)); ++splits) {
      const int64_t rounds = (tiles * splits + sms - 1) / sms, steps = (blocks + splits - 1) / splits;
      const double cost = rounds * (steps * (double)(std::min<int64_t>(M, kTokens) + nc) + 600.0) + (splits > 1 ? 400.0 + splits * (double)nc : 0.0);
      if (cost < least) least = cost, best = Shape{nc, (int)n_tiles, (int)tiles, (int)splits};
    }
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

template <int NC, typename T>
int launch_t(const CUtensorMap& tx, const CUtensorMap& tw, const CUtensorMap& to, const Args& a, bool overlap, cudaStream_t s) {
  const int st = ensure_dyn_smem(reinterpret_cast<const void*>(fp8_kernel<NC, T>), smem_bytes<NC>(), "fp8_linear shared memory");
  if (st != FLB_OK) return st;
  cudaLaunchAttribute attr[1];
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)std::min<int64_t>((int64_t)a.tiles * a.splits, num_sms()));
  cfg.blockDim = dim3(threads<NC>());
  cfg.dynamicSmemBytes = smem_bytes<NC>();
  cfg.stream = s;
  cfg.attrs = attr;
  if (overlap) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 1;
  }
  const cudaError_t e = cudaLaunchKernelEx(&cfg, fp8_kernel<NC, T>, tx, tw, to, a);
  count_launches(1);
  return check_cuda(e, "fp8_linear launch");
}

template <typename T> int launch(int width, const CUtensorMap& tx, const CUtensorMap& tw, const CUtensorMap& to, const Args& a, bool overlap, cudaStream_t s) {
  switch (width) {
    case 64: return launch_t<64, T>(tx, tw, to, a, overlap, s);
    case 128: return launch_t<128, T>(tx, tw, to, a, overlap, s);
    default: return launch_t<192, T>(tx, tw, to, a, overlap, s);
  }
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

int fp8_rows(const void* x, int64_t ldx, int8_t* codes, uint8_t* exps, int64_t R, int64_t K, int dtype, uint32_t* zero, int n_zero, cudaStream_t s);

size_t fp8_linear_workspace_bytes(int64_t M, int64_t N, int64_t K, bool quantise) { return ws_of(shape_of(M, N, K), M, K, quantise).bytes; }

int fp8_linear(const void* x, int64_t ldx, const int8_t* x_codes, int64_t ldc, const uint8_t* x_exps, const int8_t* w_codes, int64_t ldw,
               const uint8_t* w_exps, const void* bias, int bias_dtype, void* out, int64_t M, int64_t N, int64_t K, int dtype, void* ws,
               int check_timeout, cudaStream_t s) {
  const Shape g = shape_of(M, N, K);
  const Ws l = ws_of(g, M, K, x != nullptr);
  uint8_t* const p = reinterpret_cast<uint8_t*>(ws);
  const int n_zero = 1 + (g.splits > 1 ? g.tiles : 0);
  const bool reset = !x && (g.splits > 1 || check_timeout);
  int st;
  if (x) {
    // the rows' kernel clears the error word and the counts too
    int8_t* const codes = reinterpret_cast<int8_t*>(p + l.codes);
    if ((st = fp8_rows(x, ldx, codes, p + l.exps, M, K, dtype, reinterpret_cast<uint32_t*>(p), n_zero, s)) != FLB_OK) return st;
    x_codes = codes, x_exps = p + l.exps, ldc = rows::code_pitch(K);
  } else if (reset) {  // otherwise nothing reads those words
    if ((st = check_cuda(cudaMemsetAsync(p, 0, (size_t)n_zero * 4, s), "fp8_linear reset")) != FLB_OK) return st;
  }
  Args a = {};
  a.a_rows = (int)std::min<int64_t>(kTokens, (M + 7) / 8 * 8);
  CUtensorMap tw, tx, to = {};
  if ((st = code_map(&tw, w_codes, N, ldw, K, g.width)) != FLB_OK) return st;
  if ((st = code_map(&tx, x_codes, M, ldc, K, a.a_rows)) != FLB_OK) return st;
  const int es = dtype_size(dtype);
  a.tma_store = N * es % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
  if (a.tma_store) {
    const uint64_t dims[2] = {(uint64_t)N, (uint64_t)M};
    const uint64_t strides[1] = {(uint64_t)N * es};
    const uint32_t box[2] = {(uint32_t)(128 / es), 32};
    const CUtensorMapDataType dt = dtype == FLB_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : dtype == FLB_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                                                         : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    if ((st = make_tmap(&to, out, dt, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) != FLB_OK) return st;
  }
  a.ex = x_exps, a.ew = w_exps, a.bias = bias, a.bias_dtype = bias_dtype, a.out = out, a.M = M, a.N = N;
  a.early = x != nullptr;
  a.k_blocks = (int)blocks_of(K), a.quads = (int)quads_of(K), a.n_tiles = g.n_tiles, a.tiles = g.tiles, a.splits = g.splits;
  a.group = N * K <= kWeightInL2 ? 1 : 16;
  a.stream_out = (size_t)M * N * es > kOutputInL2;
  a.parts = reinterpret_cast<float*>(p + l.parts), a.counts = reinterpret_cast<uint32_t*>(p + l.counts), a.error = reinterpret_cast<uint32_t*>(p);
  switch (dtype) {
    case FLB_F32: st = launch<float>(g.width, tx, tw, to, a, x != nullptr, s); break;
    case FLB_F16: st = launch<__half>(g.width, tx, tw, to, a, x != nullptr, s); break;
    default: st = launch<__nv_bfloat16>(g.width, tx, tw, to, a, x != nullptr, s); break;
  }
  if (st != FLB_OK || !check_timeout) return st;
  uint32_t err = 0;
  if ((st = check_cuda(cudaMemcpyAsync(&err, p, 4, cudaMemcpyDeviceToHost, s), "fp8_linear error word")) != FLB_OK) return st;
  if ((st = check_cuda(cudaStreamSynchronize(s), "fp8_linear error word")) != FLB_OK) return st;
  return err ? fail(FLB_ERR_TIMEOUT, "fp8_linear: a bounded wait in the kernel gave up") : FLB_OK;
}

}  // namespace flb
