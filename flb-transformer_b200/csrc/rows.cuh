// Row kernels' shared parts: how the threads of a row divide its elements, vector access, reductions
// over a row, the 8-bit kept form and 8-bit integer codes, programmatic dependent launch.
#pragma once
#include <algorithm>
#include "common.cuh"

namespace flb {
namespace rows {

// A row's threads (one warp, or a whole block) cover it in chunks of 256 consecutive elements per warp,
// eight elements a lane. VEC (rows that start on 16 bytes, a multiple of 8 elements wide): a lane's eight
// are consecutive, one 16-byte access for 16-bit types, two for float32. Otherwise they lie 32 apart, so
// that a warp's scalar accesses are still one contiguous run each. Both ways a warp's chunk is two blocks
// of 128 elements: lanes 0-15 and 16-31, or a lane's first four and last four.
template <bool VEC> struct Chunk {
  // element j of the chunk that starts at `base`
  static __device__ __forceinline__ int at(int base, int lane, int j) {
    return VEC ? base + lane * 8 + j : base + j * 32 + lane;
  }
};

template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t u);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t u) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t u) {
  return __half22float2(*reinterpret_cast<__half2*>(&u));
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}

// Eight elements as they lie in memory: 4 words for 16-bit types, 8 for float32. Loading and converting
// are apart so that a loop can hold the next row's loads in flight.
template <typename T> struct Raw8 { uint32_t w[sizeof(T) * 2]; };

template <typename T, bool VEC>
__device__ __forceinline__ void load_raw(Raw8<T>& r, const T* __restrict__ row, int base, int lane, int D) {
  if constexpr (VEC) {
    const int p = base + lane * 8;
    if (p < D) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(row + p) + i);
        r.w[4 * i] = v.x, r.w[4 * i + 1] = v.y, r.w[4 * i + 2] = v.z, r.w[4 * i + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) * 2; ++i) r.w[i] = 0;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int p = base + j * 32 + lane;
      if constexpr (sizeof(T) == 4) {
        r.w[j] = p < D ? __ldg(reinterpret_cast<const uint32_t*>(row) + p) : 0u;
      } else {
        const uint32_t v = p < D ? (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(row) + p) : 0u;
        if (j & 1) r.w[j / 2] |= v << 16; else r.w[j / 2] = v;
      }
    }
  }
}
template <typename T> __device__ __forceinline__ void to_float(const Raw8<T>& r, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(r.w[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = unpack2<T>(r.w[j]);
      v[2 * j] = f.x, v[2 * j + 1] = f.y;
    }
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void load8(float (&v)[8], const T* __restrict__ row, int base, int lane, int D) {
  Raw8<T> r;
  load_raw<T, VEC>(r, row, base, lane, D);
  to_float<T>(r, v);
}
template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* __restrict__ row, const float (&v)[8], int base, int lane, int D) {
  if constexpr (VEC) {
    const int p = base + lane * 8;
    if (p >= D) return;
    if constexpr (sizeof(T) == 4) {
      reinterpret_cast<float4*>(row + p)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(row + p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      *reinterpret_cast<uint4*>(row + p) = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]),
                                                      pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int p = base + j * 32 + lane;
      if (p < D) st(row + p, v[j]);
    }
  }
}

// ---- 8-bit integers -----------------------------------------------------------------------------
// A float of magnitude at most 127 plus 1.5 * 2^23 is that float rounded to the nearest integer (ties to
// even), whose two's complement is in the low byte of the sum's bits.
constexpr float kRound = 12582912.f;
__device__ __forceinline__ uint32_t code_of(float scaled) { return __float_as_uint(__fadd_rn(scaled, kRound)); }

// The low bytes of four words, the first lowest.
__device__ __forceinline__ uint32_t bytes4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// Eight codes to a row of bytes whose start is 16-byte aligned (every code array's pitch is a multiple of 16)
template <bool VEC>
__device__ __forceinline__ void store_codes(int8_t* __restrict__ row, const uint32_t (&q)[8], int base, int lane, int D) {
  if constexpr (VEC) {
    const int p = base + lane * 8;
    if (p < D) *reinterpret_cast<uint2*>(row + p) = make_uint2(bytes4(q[0], q[1], q[2], q[3]), bytes4(q[4], q[5], q[6], q[7]));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int p = base + j * 32 + lane;
      if (p < D) row[p] = (int8_t)(q[j] & 0xffu);
    }
  }
}
template <bool VEC>
__device__ __forceinline__ uint2 load_codes(const int8_t* __restrict__ row, int base, int lane, int D) {
  uint2 r = make_uint2(0, 0);
  if constexpr (VEC) {
    const int p = base + lane * 8;
    if (p < D) r = __ldg(reinterpret_cast<const uint2*>(row + p));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int p = base + j * 32 + lane;
      const uint32_t v = p < D ? (uint32_t)(uint8_t)__ldg(row + p) : 0u;
      if (j < 4) r.x |= v << (8 * j); else r.y |= v << (8 * (j - 4));
    }
  }
  return r;
}
// A signed byte b as a float: 2^23 + (b + 128) has b + 128 in its low byte.
__device__ __forceinline__ void codes_to_float(uint2 c, float (&v)[8]) {
  const uint32_t lo = c.x ^ 0x80808080u, hi = c.y ^ 0x80808080u;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[j] = __uint_as_float(__byte_perm(lo, 0x4B000000u, 0x7540 | j)) - 8388736.f;
    v[4 + j] = __uint_as_float(__byte_perm(hi, 0x4B000000u, 0x7540 | j)) - 8388736.f;
  }
}

// ---- the kept form --------------------------------------------------------------------------------
// A block of 128 consecutive elements is kept as codes c of magnitude at most 127 and one byte E:
// element = c * 2^(E - 127), E the smallest of at least 1 for which the block's largest magnitude a still
// rounds to at most 127 (a < 127.5 * 2^(E - 127)). A block with an infinity or NaN gets E = 255 and comes
// back as NaN. Powers of two because then scaling is exact: codes are the same for every order of
// computing them, an element of a 16-bit type times its inverse scale is exact in float32, and what comes
// back fits bfloat16 without a second rounding. With a unit of a / 127 instead, the rounding error would
// be smaller by up to a factor of two.
constexpr int kBlock = 128;
constexpr uint32_t kBadBlock = 255;

// E for the block whose largest magnitude has these bits: with a = 1.f * 2^(x - 127) (x the exponent
// field), 2^(x - 133) has a / 2^(x - 133) = 64 * 1.f, below 127.5 when 1.f < 1.9921875.
__device__ __forceinline__ uint32_t block_exp(uint32_t amax_bits) {
  const uint32_t x = amax_bits >> 23;
  if (x == 255) return kBadBlock;
  const uint32_t up = (amax_bits & 0x7fffffu) >= 0x7f0000u ? 1u : 0u;
  return x + up < 7u ? 1u : x + up - 6u;
}
__device__ __forceinline__ float scale_of(uint32_t e) {  // 2^(e - 127), NaN for a bad block
  return e == kBadBlock ? __uint_as_float(0x7fffffffu) : __uint_as_float(e << 23);
}
// Bits of the larger magnitude: integers of non-negative floats order as the floats do, and an infinity
// or NaN, whose exponent field is 255, is above every number.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// Keeps a lane's eight elements (chunk at `base`): codes to `crow`, the two blocks' E to `erow`.
// All 32 lanes take part; elements at or beyond D must be zero.
template <bool VEC>
__device__ __forceinline__ void keep8(const float (&v)[8], int8_t* __restrict__ crow, uint8_t* __restrict__ erow,
                                      int base, int lane, int D) {
  uint32_t q[8];
  auto code = [](float x, uint32_t e) {
    // 2^(127 - E) as (254 - E) in the exponent field. The largest E, 249, has 64 for a magnitude that
    // its own type holds and 64 * 2^122 exceeds float32: 63 then. A bad block's codes are not read.
    if (e >= 249u) x = fminf(fmaxf(x, -63.f * 5.316911983139664e36f), 63.f * 5.316911983139664e36f);
    return code_of(x * __uint_as_float((254u - (e > 249u ? 249u : e)) << 23));
  };
  if constexpr (VEC) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, abs_bits(v[j]));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const uint32_t e = block_exp(m);
#pragma unroll
    for (int j = 0; j < 8; ++j) q[j] = code(v[j], e);
    if ((lane & 15) == 0 && base + lane * 8 < D) erow[(base + lane * 8) / kBlock] = (uint8_t)e;
  } else {
    uint32_t m[2] = {0, 0}, e[2];
#pragma unroll
    for (int j = 0; j < 8; ++j) m[j / 4] = max(m[j / 4], abs_bits(v[j]));
#pragma unroll
    for (int h = 0; h < 2; ++h) e[h] = block_exp(__reduce_max_sync(0xffffffffu, m[h]));
#pragma unroll
    for (int j = 0; j < 8; ++j) q[j] = code(v[j], e[j / 4]);
    if (lane < 2 && base + lane * kBlock < D) erow[base / kBlock + lane] = (uint8_t)(lane ? e[1] : e[0]);
  }
  store_codes<VEC>(crow, q, base, lane, D);
}

// What a lane's eight kept elements stand for (zero at or beyond D).
struct Kept8 {
  uint2 c;
  uint32_t e;  // two bytes: the E of the lane's first four and last four elements
};
template <bool VEC>
__device__ __forceinline__ uint32_t load_exps(const uint8_t* __restrict__ erow, int base, int lane, int D) {
  if constexpr (VEC) return base + lane * 8 < D ? __ldg(erow + (base + lane * 8) / kBlock) : 1u;
  uint32_t e = base < D ? __ldg(erow + base / kBlock) : 1u;
  return e | (base + kBlock < D ? (uint32_t)__ldg(erow + base / kBlock + 1) : 1u) << 8;
}
template <bool VEC>
__device__ __forceinline__ Kept8 load_kept(const int8_t* __restrict__ crow, const uint8_t* __restrict__ erow,
                                           int base, int lane, int D) {
  return Kept8{load_codes<VEC>(crow, base, lane, D), load_exps<VEC>(erow, base, lane, D)};
}
template <bool VEC> __device__ __forceinline__ void kept_to_float(const Kept8& k, float (&v)[8]) {
  codes_to_float(k.c, v);
  const float s0 = scale_of(k.e & 0xffu), s1 = VEC ? s0 : scale_of(k.e >> 8);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] *= j < 4 ? s0 : s1;
}

// Where the codes of [.., D] rows lie: rows of this many bytes, and this many E bytes a row.
__host__ __device__ inline int64_t code_pitch(int64_t D) { return (D + 15) & ~(int64_t)15; }
__host__ __device__ inline int64_t blocks_of(int64_t D) { return (D + kBlock - 1) / kBlock; }

// ---- reductions over a row ------------------------------------------------------------------------
// Over one warp, or over the whole block through `slot` (32 words, not used for anything else until every
// thread has passed a later barrier). Every thread gets the result, summed in the same order each time.
template <bool WARP> __device__ __forceinline__ float row_sum(float v, float* slot) {
  v = warp_sum(v);
  if constexpr (!WARP) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = blockDim.x >> 5;
    if (lane == 0) slot[warp] = v;
    __syncthreads();
    v = warp_sum(lane < n ? slot[lane] : 0.f);
  }
  return v;
}
template <bool WARP> __device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t* slot) {
  v = __reduce_max_sync(0xffffffffu, v);
  if constexpr (!WARP) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = blockDim.x >> 5;
    if (lane == 0) slot[warp] = v;
    __syncthreads();
    v = __reduce_max_sync(0xffffffffu, lane < n ? slot[lane] : 0u);
  }
  return v;
}

}  // namespace rows

// ---- programmatic dependent launch ------------------------------------------------------------------
// A kernel launched with launch_dependent may start while its predecessor in the stream drains; it calls
// wait_predecessor before it touches anything the predecessor, or a kernel before that one, wrote or read.
__device__ __forceinline__ void wait_predecessor() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_successor_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename... KArgs, typename... Args>
cudaError_t launch_dependent(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t s,
                             Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

}  // namespace flb
