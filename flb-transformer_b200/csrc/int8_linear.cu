// Product of 8-bit integer rows, each with a scale: out[m, n] = (sum_k X[m, k] W[n, k]) sx[m] sw[n] + bias[n].
//
// tcgen05.mma kind::i8, 32-bit integer accumulators in TMEM (exact for K <= 131072: K 127^2 < 2^31). The weight
// rows are the M side of the instruction, 128 output channels a tile, and the tokens its N side, NT of 16 to
// 256: a decoding step of few tokens wastes little of a tile, and in the epilogue a warp's lanes are
// consecutive channels of one token, so its stores are contiguous without a transpose.
//
// One block a SM, persistent over units of work: a unit is a tile, or with few tiles a part of the
// tile's K range. Warp 0 loads by TMA into a ring, warp 1 issues the MMAs, warps 2-9 read TMEM (two accumulators, so
// that a tile's epilogue runs beside the next one's MMAs). Parts of a tile leave integer sums in the
// workspace; the block that counts itself last adds them up: integers, the same in any order.
//
// Few tokens: bound by reading the weight, of which a ring of 11 stages keeps 176 KB a SM in flight. Many: by
// the tensor cores and the operands' way from L2 (48 KB for 512 cycles of MMA at NT = 256).
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
constexpr uint32_t kWaitLimit = 4000000u;  // polls, each of which the hardware may hold for a while

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
  int k_blocks;       // of kStep
  int n_tiles, tiles, splits;
  int32_t* parts;     // [tiles][splits][NT][128], splits > 1
  uint32_t* counts;   // [tiles], zero
  uint32_t* error;
};

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
    v[j] = fmaf(__int2float_rn((int)acc[j]) * s.x, sw, bias);
    v[j + 1] = fmaf(__int2float_rn((int)acc[j + 1]) * s.y, sw, bias);
    v[j + 2] = fmaf(__int2float_rn((int)acc[j + 2]) * s.z, sw, bias);
    v[j + 3] = fmaf(__int2float_rn((int)acc[j + 3]) * s.w, sw, bias);
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
    int8_gemm_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, const Int8Args a) {
  constexpr int S = stages<NT>();
  constexpr uint32_t kBytes = stage_bytes<NT>();
  extern __shared__ uint8_t dyn[];
  __shared__ __align__(8) uint64_t full[S], empty[S], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_base, last_flag;
  __shared__ __align__(16) float scales[kEpilogue / 32][NT > 64 ? NT / 2 : 32];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dyn) + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tm_w);
    tma_prefetch_desc(&tm_x);
    for (int i = 0; i < S; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&acc_full[i], 1), mbar_init(&acc_empty[i], kEpilogue);
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
      // the weight was written before the kernel that this one may overlap started; the tokens' codes by
      // that kernel, so the first ring of weight tiles is on its way before the wait
      bool ok = true, waited = false;
      uint32_t it = 0;
      for (int u = blockIdx.x; u < units && ok; u += gridDim.x) {
        const int tile = u / a.splits;
        const int n0 = (tile % a.n_tiles) * kChannels, m0 = (tile / a.n_tiles) * NT;
        int k0, k1;
        k_range(u % a.splits, k0, k1);
        int early = 0;  // stages of this unit whose weight part is already under way
        if (!waited) {
          early = min(k1 - k0, S);
          for (int i = 0; i < early; ++i) {
            mbar_arrive_expect_tx(&full[i], kBytes);
            tma_load_2d(ring + (size_t)i * kBytes, &tm_w, &full[i], (k0 + i) * kStep, n0);
          }
          wait_predecessor();
          waited = true;
        }
        for (int k = k0; k < k1; ++k, ++it) {
          const int s = it % S;
          uint8_t* st = ring + (size_t)s * kBytes;
          if (k - k0 >= early) {
            if (it >= (uint32_t)S && !mbar_wait(&empty[s], ((it / S) & 1) ^ 1, kWaitLimit)) {
              ok = false;
              break;
            }
            mbar_arrive_expect_tx(&full[s], kBytes);
            tma_load_2d(st, &tm_w, &full[s], k * kStep, n0);
          }
          tma_load_2d(st + kChannels * kStep, &tm_x, &full[s], k * kStep, m0);
        }
      }
      if (!ok) {
        atomicExch(a.error, 1u);
        // the copies still in flight land before the block's shared memory is given up
        for (uint32_t i = it > (uint32_t)S ? it - S : 0; i < it; ++i) mbar_wait(&full[i % S], (i / S) & 1, kWaitLimit);
      }
      if (!waited) wait_predecessor();
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_i8<NT>();
      uint32_t it = 0, local = 0;
      bool ok = true;
      for (int u = blockIdx.x; u < units && ok; u += gridDim.x, ++local) {
        const uint32_t b = local & 1;
        if (local >= 2 && !mbar_wait(&acc_empty[b], ((local >> 1) & 1) ^ 1, kWaitLimit)) {
          ok = false;
          break;
        }
        tc_fence_after();
        int k0, k1;
        k_range(u % a.splits, k0, k1);
        for (int k = k0; k < k1; ++k, ++it) {
          const int s = it % S;
          if (!mbar_wait(&full[s], (it / S) & 1, kWaitLimit)) {
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
    }
  } else {
    // each epilogue warp has the 32 TMEM lanes, here channels, of its number mod 4, and half of the tokens
    // (the first four warps all of 16)
    constexpr int COLS = NT >= 32 ? NT / 2 : NT, CW = COLS < 32 ? COLS : 32, STEPS = COLS / CW;
    const int q = warp & 3, first = (warp - 2) / 4 * COLS;
    const bool has_cols = first < NT;
    float* sx = scales[warp - 2];
    uint32_t local = 0, limit = kWaitLimit;
    wait_predecessor();
    for (int u = blockIdx.x; u < units; u += gridDim.x, ++local) {
      const uint32_t b = local & 1;
      const int tile = u / a.splits, split = u % a.splits;
      const int64_t n0 = (int64_t)(tile % a.n_tiles) * kChannels, m0 = (int64_t)(tile / a.n_tiles) * NT + first;
      const int64_t channel = n0 + q * 32 + lane;
      const bool there = channel < a.N, full_tile = n0 + kChannels <= a.N && m0 + COLS <= a.M;
      const float sw = there ? __ldg(a.sw + channel) : 0.f;
      float bias = 0.f;
      if (a.bias && there)
        bias = a.bias32 ? __ldg(reinterpret_cast<const float*>(a.bias) + channel) : ld(reinterpret_cast<const T*>(a.bias) + channel);
      __syncwarp();
#pragma unroll
      for (int c = 0; c < COLS; c += 32)
        if (c + lane < COLS) sx[c + lane] = m0 + c + lane < a.M ? __ldg(a.sx + m0 + c + lane) : 0.f;
      __syncwarp();
      if (!mbar_wait(&acc_full[b], (local >> 1) & 1, limit)) {
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
#pragma unroll 1
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

// Tokens a tile and parts of a tile's K range. Up to 128 tokens: one tile of tokens. More: the width whose
// rounds of tiles over the SMs cost least, a tile's K step costing its operands' rows. Fewer tiles than SMs:
// as many parts of K as fill them.
struct GemmShape {
  int nt, n_tiles, tiles, splits;
};
GemmShape gemm_shape(int64_t M, int64_t N, int64_t K) {
  GemmShape g;
  const int64_t sms = num_sms();
  g.n_tiles = (int)((N + kChannels - 1) / kChannels);
  g.nt = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : 128;
  if (M > 128) {
    auto cost = [&](int nt) { return (((M + nt - 1) / nt * g.n_tiles + sms - 1) / sms) * (kChannels + nt); };
    if (cost(256) <= cost(128)) g.nt = 256;
  }
  g.tiles = (int)((M + g.nt - 1) / g.nt * g.n_tiles);
  const int64_t blocks = (K + kStep - 1) / kStep;
  g.splits = (int)std::max<int64_t>(1, std::min<int64_t>(blocks, sms / g.tiles));
  return g;
}

// Workspace: [error, counts] | codes and scales of the tokens (when they are quantised here) | parts
struct GemmWs {
  size_t counts, codes, scale, parts, bytes;
};
GemmWs gemm_ws(int64_t M, int64_t N, int64_t K, bool quantise) {
  const GemmShape g = gemm_shape(M, N, K);
  auto al = [](size_t x) { return (x + 255) & ~(size_t)255; };
  GemmWs w;
  w.counts = 4;
  size_t off = al(4 + (g.splits > 1 ? (size_t)g.tiles * 4 : 0));
  w.codes = off;
  off += quantise ? al((size_t)M * rows::code_pitch(K)) : 0;
  w.scale = off;
  off += quantise ? al((size_t)M * 4) : 0;
  w.parts = off;
  off += g.splits > 1 ? (size_t)g.tiles * g.splits * g.nt * kChannels * 4 : 0;
  w.bytes = off;
  return w;
}

template <int NT, typename T>
int launch_gemm(const CUtensorMap& tw, const CUtensorMap& tx, const Int8Args& a, bool after_rows, cudaStream_t s) {
  auto k = int8_gemm_kernel<NT, T>;
  const int smem = stages<NT>() * stage_bytes<NT>() + 1024;
  int st = ensure_dyn_smem(reinterpret_cast<const void*>(k), smem, "int8_linear shared memory");
  if (st != FLB_OK) return st;
  const dim3 grid((unsigned)std::min<int64_t>((int64_t)a.tiles * a.splits, num_sms()));
  cudaError_t e;
  if (after_rows) {
    e = launch_dependent(k, grid, dim3(kGemmThreads), smem, s, tw, tx, a);
  } else {
    k<<<grid, kGemmThreads, smem, s>>>(tw, tx, a);
    e = cudaGetLastError();
  }
  count_launches(1);
  return check_cuda(e, "int8_linear launch");
}

template <typename T>
int launch_gemm_t(int nt, const CUtensorMap& tw, const CUtensorMap& tx, const Int8Args& a, bool after_rows, cudaStream_t s) {
  switch (nt) {
    case 16: return launch_gemm<16, T>(tw, tx, a, after_rows, s);
    case 32: return launch_gemm<32, T>(tw, tx, a, after_rows, s);
    case 64: return launch_gemm<64, T>(tw, tx, a, after_rows, s);
    case 128: return launch_gemm<128, T>(tw, tx, a, after_rows, s);
    default: return launch_gemm<256, T>(tw, tx, a, after_rows, s);
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

size_t int8_linear_workspace_bytes(int64_t M, int64_t N, int64_t K, bool quantise) { return gemm_ws(M, N, K, quantise).bytes; }

int int8_linear(const void* x, int64_t ldx, const int8_t* x_codes, int64_t ldc, const float* x_scale, const int8_t* w_codes,
                int64_t ldw, const float* w_scale, const void* bias, int bias_dtype, void* out, int64_t M, int64_t N,
                int64_t K, int dtype, void* ws, int check_timeout, cudaStream_t s) {
  const GemmShape g = gemm_shape(M, N, K);
  const GemmWs l = gemm_ws(M, N, K, x != nullptr);
  uint8_t* p = reinterpret_cast<uint8_t*>(ws);
  const int64_t n_zero = 1 + (g.splits > 1 ? g.tiles : 0);
  int st;
  if (x) {
    // the rows' kernel clears the error word and the counts too
    int8_t* codes = reinterpret_cast<int8_t*>(p + l.codes);
    float* scale = reinterpret_cast<float*>(p + l.scale);
    if ((st = int8_rows(x, ldx, codes, scale, M, K, dtype, reinterpret_cast<uint32_t*>(p), n_zero, s)) != FLB_OK) return st;
    x_codes = codes, x_scale = scale, ldc = rows::code_pitch(K);
  } else if ((st = check_cuda(cudaMemsetAsync(p, 0, n_zero * 4, s), "int8_linear reset")) != FLB_OK) {
    return st;
  }
  CUtensorMap tw, tx;
  if ((st = code_map(&tw, w_codes, N, ldw, K, kChannels)) != FLB_OK) return st;
  if ((st = code_map(&tx, x_codes, M, ldc, K, g.nt)) != FLB_OK) return st;
  const Int8Args a{x_scale, w_scale, bias, bias_dtype == FLB_F32, out, M, N,
                   N % 2 == 0 && reinterpret_cast<uintptr_t>(out) % 4 == 0, (int)((K + kStep - 1) / kStep), g.n_tiles, g.tiles,
                   g.splits, reinterpret_cast<int32_t*>(p + l.parts), reinterpret_cast<uint32_t*>(p + l.counts),
                   reinterpret_cast<uint32_t*>(p)};
  switch (dtype) {
    case FLB_F32: st = launch_gemm_t<float>(g.nt, tw, tx, a, x != nullptr, s); break;
    case FLB_F16: st = launch_gemm_t<__half>(g.nt, tw, tx, a, x != nullptr, s); break;
    default: st = launch_gemm_t<__nv_bfloat16>(g.nt, tw, tx, a, x != nullptr, s); break;
  }
  if (st != FLB_OK || !check_timeout) return st;
  uint32_t err = 0;
  if ((st = check_cuda(cudaMemcpyAsync(&err, p, 4, cudaMemcpyDeviceToHost, s), "int8_linear error word")) != FLB_OK) return st;
  if ((st = check_cuda(cudaStreamSynchronize(s), "int8_linear error word")) != FLB_OK) return st;
  return err ? fail(FLB_ERR_TIMEOUT, "int8_linear: a bounded wait in the kernel gave up") : FLB_OK;
}

}  // namespace flb
