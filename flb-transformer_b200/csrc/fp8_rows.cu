// Rows into 8-bit floating point (fp8.cuh), along their own axis, and a matrix along both.
//
// rows_kernel: each row's blocks alone, for inference. A block is 16 lanes' eight 16-bit values, or a warp's four float32.
// tile_kernel: a training step reads x, the weight and the output's gradient each along two axes, since its three products sum
// over three of them. A block of threads takes 128 x 128 elements, which hold a power of two's block of every row and of
// every column, from one read of them, and leaves the second kind transposed: rows of the product that sums the other way.
// For the gradient it adds up the columns too, in float32 and a fixed order: what the bias gets.
// Bound by memory: 2 bytes read and 2 written an element of 16 bits.
#include "fp8.cuh"

namespace flb {

namespace {

using namespace fp8;

// PER lanes of a warp share a row's block of 128: 16 (eight values each) or 32 (four)
template <typename T> constexpr int kPer = sizeof(T) == 2 ? 16 : 32;

template <int N> __device__ __forceinline__ uint32_t max_of(uint32_t v) {
#pragma unroll
  for (int o = N / 2; o; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// 16 bytes of a row of K from column c on, zeros beyond. VEC: rows that start on 16 bytes, whole ones of them.
template <typename T, bool VEC> __device__ __forceinline__ uint4 load_row(const T* row, int64_t c, int64_t K) {
  constexpr int N = 16 / sizeof(T);
  if constexpr (VEC) return c < K ? *reinterpret_cast<const uint4*>(row + c) : make_uint4(0, 0, 0, 0);
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if (c + j < K) {
      if constexpr (sizeof(T) == 4) w[j & 3] = __float_as_uint(row[c + j]);
      else w[j / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(row)[c + j] << (16 * (j & 1));
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename T> __device__ __forceinline__ void unpack_row(float (&v)[16 / sizeof(T)], const uint4& w) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (sizeof(T) == 4) {
      v[j] = __uint_as_float(u[j]);
    } else {
      const float2 f = rows::unpack2<T>(u[j]);
      v[2 * j] = f.x, v[2 * j + 1] = f.y;
    }
  }
}

// Codes of these values to their row, whose pitch is a multiple of 16: what lies behind K (up to the pitch) may be written.
template <int N> __device__ __forceinline__ void store_codes(int8_t* row, const float (&v)[N], float inv, int64_t c, int64_t pitch) {
  uint32_t w[N / 4];
#pragma unroll
  for (int j = 0; j < N / 4; ++j) w[j] = code4(v[4 * j] * inv, v[4 * j + 1] * inv, v[4 * j + 2] * inv, v[4 * j + 3] * inv);
  if (c >= pitch) return;
  if constexpr (N == 8) *reinterpret_cast<uint2*>(row + c) = make_uint2(w[0], w[1]);
  else *reinterpret_cast<uint32_t*>(row + c) = w[0];
}

// The float32 bits of the largest magnitude of 16 bytes a lane and PER lanes. 16-bit values as they are, two at a time: their magnitudes' bits
// are ordered as they are.
template <typename T, int PER> __device__ __forceinline__ uint32_t largest(const uint4& w) {
  if constexpr (sizeof(T) == 4) {
    return max_of<PER>(max(max(w.x & 0x7fffffffu, w.y & 0x7fffffffu), max(w.z & 0x7fffffffu, w.w & 0x7fffffffu)));
  } else {
    const uint32_t two = __vmaxu2(__vmaxu2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu), __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu));
    return __float_as_uint(rows::unpack2<T>(max_of<PER>(max(two & 0xffffu, two >> 16))).x);
  }
}

struct RowsArgs {
  const void* x;
  int64_t ldx, R, K, pitch, quads;
  int8_t* codes;
  uint8_t* exps;
  unsigned clears; // thread blocks ahead of those that make rows
  uint32_t* zero;  // words to clear, or null
  int n_zero;
};

// Zeros in the places of exps that no block has: behind each row's last one, and of the rows to the next 128. `at` of `step` threads.
__device__ __forceinline__ void clear_places(const RowsArgs& a, int64_t at, int64_t step) {
  const int64_t blocks = blocks_of(a.K), behind = a.quads * 4 - blocks, words = (blocks_of(a.R) * kBlock - a.R) * a.quads;
  for (int64_t i = at; i < words; i += step) *reinterpret_cast<uint32_t*>(a.exps + exp_at(a.R + i / a.quads, i % a.quads * 4, a.quads)) = 0;
  for (int64_t i = at; i < a.R * behind; i += step) a.exps[exp_at(i / behind, blocks + i % behind, a.quads)] = 0;
}

// WHOLE: the first thread blocks clear the places of exps that no block has. (By the threads of the last block and row 16384 x 32000 bf16 took 580 us, so
// 440, and 428 without; by thread blocks at the end of the grid 4096 x 768 took 4.7 us, so 3.8.)
template <typename T, bool VEC, bool WHOLE> __global__ void __launch_bounds__(256) rows_kernel(const RowsArgs a) {
  let_successor_start();
  if (WHOLE && blockIdx.x < a.clears) {
    clear_places(a, (int64_t)blockIdx.x * 256 + threadIdx.x, (int64_t)a.clears * 256);
    return;
  }
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < a.n_zero; i += 256) a.zero[i] = 0;
  constexpr int PER = kPer<T>, N = 16 / sizeof(T);
  const int64_t blocks = blocks_of(a.K), unit = ((int64_t)(blockIdx.x - (WHOLE ? a.clears : 0)) * 256 + threadIdx.x) / PER;
  const int lane = threadIdx.x % PER;
  const int64_t row = unit / blocks, block = unit % blocks;
  const bool there = row < a.R;
  const uint4 raw = there ? load_row<T, VEC>(reinterpret_cast<const T*>(a.x) + row * a.ldx, block * kBlock + lane * N, a.K) : make_uint4(0, 0, 0, 0);
  float v[N];
  unpack_row<T>(v, raw);
  const int u = unit_of(largest<T, PER>(raw));
  if (!there) return;
  store_codes(a.codes + row * a.pitch, v, inverse_of(u), block * kBlock + lane * N, a.pitch);
  if (lane == 0) a.exps[exp_at(row, block, a.quads)] = (uint8_t)u;
}

struct TileArgs {
  const void* x;
  int64_t ldx, R, C;
  int64_t pitch, quads;      // of the rows' form
  int64_t pitch_t, quads_t;  // of the columns'
  int8_t *codes, *codes_t;
  uint8_t *exps, *exps_t;
  float* sums;               // null, or [tiles of rows][C]: each column's sum over a tile's rows
};

constexpr int kDown = 8;

// 256 threads. As 16 or 8 rows at a time (a row's block in PER lanes), then as columns: four runs of 32 rows of 64 pairs of columns.
template <typename T, bool VEC, bool SUM> __global__ void __launch_bounds__(256, sizeof(T) == 4 ? 3 : 4) tile_kernel(const TileArgs a) {
  constexpr int PER = kPer<T>, N = 16 / sizeof(T), ROWS = 256 / PER, kPitch = kBlock + 16 / (int)sizeof(T);
  extern __shared__ __align__(16) uint8_t dyn[];
  T(*tile)[kPitch] = reinterpret_cast<T(*)[kPitch]>(dyn);
  __shared__ uint32_t tops[4][kBlock];
  __shared__ float parts[SUM ? 4 : 1][kBlock];
  // Eight tiles down, then the next ones across: columns of codes leave in pieces of 1 KB that blocks running together write, rows come in long ones.
  const unsigned across = (unsigned)blocks_of(a.C), down = (unsigned)blocks_of(a.R), group = blockIdx.x / (kDown * across), in = blockIdx.x % (kDown * across);
  const unsigned high = min((unsigned)kDown, down - group * kDown), tile_r = group * kDown + in % high, tile_c = in / high;
  const int64_t r0 = (int64_t)tile_r * kBlock, c0 = (int64_t)tile_c * kBlock;
  const int lane = threadIdx.x % PER;
  // all of the thread's loads under way together
  uint4 raw[kBlock / ROWS];
#pragma unroll
  for (int i = 0; i < kBlock / ROWS; ++i) {
    const int64_t row = r0 + i * ROWS + threadIdx.x / PER;
    raw[i] = make_uint4(0, 0, 0, 0);
    if (row < a.R) raw[i] = load_row<T, VEC>(reinterpret_cast<const T*>(a.x) + row * a.ldx, c0 + lane * N, a.C);
  }
#pragma unroll
  for (int i = 0; i < kBlock / ROWS; ++i) {
    const int r = i * ROWS + threadIdx.x / PER;
    const int64_t row = r0 + r;
    *reinterpret_cast<uint4*>(&tile[r][lane * N]) = raw[i];
    float v[N];
    unpack_row<T>(v, raw[i]);
    const int u = unit_of(largest<T, PER>(raw[i]));
    if (row < a.R) {
      store_codes(a.codes + row * a.pitch, v, inverse_of(u), c0 + lane * N, a.pitch);
      if (lane == 0) a.exps[exp_at(row, tile_c, a.quads)] = (uint8_t)u;
    }
  }
  __syncthreads();
  // columns 2p and 2p + 1, rows 32g to 32g + 31: 16-bit pairs are read once and stay in registers
  const int p = threadIdx.x % 64, g = threadIdx.x / 64;
  using Pair = std::conditional_t<sizeof(T) == 4, float2, uint32_t>;
  auto pair_at = [&](int i) { return *reinterpret_cast<const Pair*>(&tile[32 * g + i][2 * p]); };
  auto values = [](const Pair& x) {
    if constexpr (sizeof(T) == 4) return x;
    else return rows::unpack2<T>(x);
  };
  Pair kept[sizeof(T) == 4 ? 1 : 32];
  uint32_t m0 = 0, m1 = 0, both = 0;
  float s0 = 0, s1 = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const Pair x = pair_at(i);
    if constexpr (sizeof(T) == 4) {
      m0 = max(m0, __float_as_uint(x.x) & 0x7fffffffu);
      m1 = max(m1, __float_as_uint(x.y) & 0x7fffffffu);
    } else {
      kept[i] = x;
      both = __vmaxu2(both, x & 0x7fff7fffu);
    }
    if (SUM) {
      const float2 v = values(x);
      s0 += v.x, s1 += v.y;
    }
  }
  if constexpr (sizeof(T) == 2) {
    const float2 v = rows::unpack2<T>(both);
    m0 = __float_as_uint(v.x), m1 = __float_as_uint(v.y);
  }
  tops[g][2 * p] = m0, tops[g][2 * p + 1] = m1;
  if (SUM) parts[g][2 * p] = s0, parts[g][2 * p + 1] = s1;
  __syncthreads();
  const int64_t col = c0 + 2 * p;
  int unit[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int c = 2 * p + j;
    unit[j] = unit_of(max(max(tops[0][c], tops[1][c]), max(tops[2][c], tops[3][c])));
    if (g == 0 && col + j < a.C) {
      a.exps_t[exp_at(col + j, tile_r, a.quads_t)] = (uint8_t)unit[j];
      if (SUM) a.sums[(int64_t)tile_r * a.C + col + j] = (parts[0][c] + parts[1][c]) + (parts[2][c] + parts[3][c]);
    }
  }
  const float inv0 = inverse_of(unit[0]), inv1 = inverse_of(unit[1]);
  uint32_t w0[8], w1[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    float2 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (sizeof(T) == 4) v[j] = pair_at(4 * k + j);
      else v[j] = values(kept[4 * k + j]);
    }
    w0[k] = code4(v[0].x * inv0, v[1].x * inv0, v[2].x * inv0, v[3].x * inv0);
    w1[k] = code4(v[0].y * inv1, v[1].y * inv1, v[2].y * inv1, v[3].y * inv1);
  }
  // through shared memory, so that a column's 128 codes leave in one piece (16 bytes a thread to 32 columns: 1050 us for 16384 x 32000, so 390)
  constexpr int kOut = kBlock + 16;
  static_assert(kBlock * kOut <= kBlock * kPitch * (int)sizeof(T), "the codes take the elements' place");
  __syncthreads();
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    *reinterpret_cast<uint4*>(dyn + (2 * p) * kOut + 32 * g + 16 * h) = make_uint4(w0[4 * h], w0[4 * h + 1], w0[4 * h + 2], w0[4 * h + 3]);
    *reinterpret_cast<uint4*>(dyn + (2 * p + 1) * kOut + 32 * g + 16 * h) = make_uint4(w1[4 * h], w1[4 * h + 1], w1[4 * h + 2], w1[4 * h + 3]);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = i * 32 + threadIdx.x / 8, at = threadIdx.x % 8 * 16;
    if (c0 + c < a.C && r0 + at < a.pitch_t)
      *reinterpret_cast<uint4*>(a.codes_t + (c0 + c) * a.pitch_t + r0 + at) = *reinterpret_cast<const uint4*>(dyn + c * kOut + at);
  }
}

// The tiles' sums, in order, into the bias's gradient.
template <typename T> __global__ void __launch_bounds__(256) sums_kernel(const float* __restrict__ sums, T* __restrict__ out, int64_t tiles, int64_t C) {
  // 32 columns a block, eight runs of tiles
  __shared__ float part[8][32];
  const int lane = threadIdx.x & 31, run = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane, per = (tiles + 7) / 8;
  float s = 0;
  if (c < C)
    for (int64_t t = run * per; t < min(tiles, (run + 1) * per); ++t) s += sums[t * C + c];
  part[run][lane] = s;
  __syncthreads();
  if (run == 0 && c < C) {
#pragma unroll
    for (int i = 1; i < 8; ++i) s += part[i][lane];
    st(out + c, s);
  }
}

bool on16(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && bytes % 16 == 0; }

template <typename T, bool WHOLE> int rows_t(RowsArgs a, cudaStream_t s) {
  const bool vec = on16(a.x, a.ldx * sizeof(T)) && a.K * sizeof(T) % 16 == 0;
  const int64_t grid = (a.R * blocks_of(a.K) * kPer<T> + 255) / 256;
  // what no block has: bytes behind rows and 4-byte words of further rows
  const int64_t places = std::max(a.R * (a.quads * 4 - blocks_of(a.K)), (blocks_of(a.R) * kBlock - a.R) * a.quads);
  a.clears = WHOLE ? (unsigned)std::min<int64_t>((places + 255) / 256, num_sms()) : 0;
  if (grid + a.clears > INT32_MAX) return fail(FLB_ERR_SHAPE, "fp8_rows: too many rows");
  if (vec) rows_kernel<T, true, WHOLE><<<(unsigned)(grid + a.clears), 256, 0, s>>>(a);
  else rows_kernel<T, false, WHOLE><<<(unsigned)(grid + a.clears), 256, 0, s>>>(a);
  count_launches(1);
  return check_cuda(cudaGetLastError(), "fp8_rows launch");
}
template <typename T> int rows_t(const RowsArgs& a, bool whole, cudaStream_t s) { return whole ? rows_t<T, true>(a, s) : rows_t<T, false>(a, s); }

template <typename T, bool VEC, bool SUM> int launch_tiles(const TileArgs& a, unsigned grid, cudaStream_t s) {
  constexpr int smem = kBlock * (kBlock * (int)sizeof(T) + 16);
  const int st = ensure_dyn_smem(reinterpret_cast<const void*>(tile_kernel<T, VEC, SUM>), smem, "fp8_rows2 shared memory");
  if (st != FLB_OK) return st;
  tile_kernel<T, VEC, SUM><<<grid, 256, smem, s>>>(a);
  count_launches(1);
  return check_cuda(cudaGetLastError(), "fp8_rows2 launch");
}

template <typename T> int tiles_t(const TileArgs& a, void* bias_grad, int bias_dtype, cudaStream_t s) {
  const bool vec = on16(a.x, a.ldx * sizeof(T)) && a.C * sizeof(T) % 16 == 0;
  const int64_t tiles = blocks_of(a.R) * blocks_of(a.C);
  if (tiles > INT32_MAX) return fail(FLB_ERR_SHAPE, "fp8_rows2: too many elements");
  int st;
  if (a.sums) st = vec ? launch_tiles<T, true, true>(a, (unsigned)tiles, s) : launch_tiles<T, false, true>(a, (unsigned)tiles, s);
  else st = vec ? launch_tiles<T, true, false>(a, (unsigned)tiles, s) : launch_tiles<T, false, false>(a, (unsigned)tiles, s);
  if (st != FLB_OK || !a.sums) return st;
  const unsigned g = (unsigned)((a.C + 31) / 32);
  switch (bias_dtype) {
    case FLB_F32: sums_kernel<<<g, 256, 0, s>>>(a.sums, reinterpret_cast<float*>(bias_grad), blocks_of(a.R), a.C); break;
    case FLB_F16: sums_kernel<<<g, 256, 0, s>>>(a.sums, reinterpret_cast<__half*>(bias_grad), blocks_of(a.R), a.C); break;
    default: sums_kernel<<<g, 256, 0, s>>>(a.sums, reinterpret_cast<__nv_bfloat16*>(bias_grad), blocks_of(a.R), a.C); break;
  }
  count_launches(1);
  return check_cuda(cudaGetLastError(), "fp8_rows2 sums launch");
}

}  // namespace

int fp8_rows(const void* x, int64_t ldx, int8_t* codes, uint8_t* exps, int64_t R, int64_t K, int dtype, bool whole, uint32_t* zero, int n_zero,
             cudaStream_t s) {
  const RowsArgs a{x, ldx, R, K, rows::code_pitch(K), quads_of(K), codes, exps, 0, zero, n_zero};
  switch (dtype) {
    case FLB_F32: return rows_t<float>(a, whole, s);
    case FLB_F16: return rows_t<__half>(a, whole, s);
    default: return rows_t<__nv_bfloat16>(a, whole, s);
  }
}

int fp8_rows2(const void* x, int64_t ldx, int8_t* codes, uint8_t* exps, int8_t* codes_t, uint8_t* exps_t, float* sums, void* bias_grad,
              int bias_dtype, int64_t R, int64_t C, int dtype, cudaStream_t s) {
  const TileArgs a{x, ldx, R, C, rows::code_pitch(C), quads_of(C), rows::code_pitch(R), quads_of(R), codes, codes_t, exps, exps_t, sums};
  switch (dtype) {
    case FLB_F32: return tiles_t<float>(a, bias_grad, bias_dtype, s);
    case FLB_F16: return tiles_t<__half>(a, bias_grad, bias_dtype, s);
    default: return tiles_t<__nv_bfloat16>(a, bias_grad, bias_dtype, s);
  }
}

}  // namespace flb
