// Row kernels' shared parts: how the threads of a row divide its elements, vector access, reductions
// over a row, the 8-bit kept form and 8-bit integer codes, programmatic dependent launch.
#pragma once
#include <algorithm>
#include <type_traits>
#include "common.cuh"

namespace flb {
namespace rows {

constexpr int kBlock = 128;  // elements of the 8-bit kept form that share an exponent

// A row's threads (one warp, or a whole block) cover it in chunks of 256 consecutive elements per warp,
// eight elements a lane, in one of three layouts, such that each access of a warp is one contiguous run:
//   SCALARS  elements 32 apart, one access each (rows that do not start on 16 bytes, or not a multiple of 8 wide)
//   EIGHT    eight consecutive elements, one 16-byte access for 16-bit types
//   FOURS    two fours 128 apart, a 16-byte access each for float32
// Each way a warp's chunk is two blocks of 128 elements: lanes 0-15 and 16-31 (EIGHT), or a lane's first
// four and last four.
enum Layout { SCALARS, EIGHT, FOURS };
template <typename T, bool VEC> constexpr Layout kLayout = !VEC ? SCALARS : sizeof(T) == 4 ? FOURS : EIGHT;

template <Layout L> struct Chunk {
  // element j of the chunk that starts at `base`, and whether the row of D elements has it
  static __device__ __forceinline__ int at(int base, int lane, int j) {
    return L == EIGHT ? base + lane * 8 + j : L == FOURS ? base + (j >> 2) * kBlock + lane * 4 + (j & 3) : base + j * 32 + lane;
  }
  static __device__ __forceinline__ bool has(int base, int lane, int j, int D) {
    return at(base, lane, L == EIGHT ? 0 : L == FOURS ? j & 4 : j) < D;
  }
};

// Two float32 in one 64-bit register pair: Blackwell multiplies and adds both in one instruction, and the
// row kernels are near the rate at which instructions can be issued.
struct F2 {
  unsigned long long u;
};
__device__ __forceinline__ F2 f2(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.u) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ F2 f2(float v) { return f2(v, v); }
__device__ __forceinline__ float2 split(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.u));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.u) : "l"(a.u), "l"(b.u));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.u) : "l"(a.u), "l"(b.u));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.u) : "l"(a.u), "l"(b.u), "l"(c.u));
  return r;
}
__device__ __forceinline__ float sum2(F2 a) {
  const float2 v = split(a);
  return v.x + v.y;
}

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

template <typename T, Layout L>
__device__ __forceinline__ void load_raw(Raw8<T>& r, const T* __restrict__ row, int base, int lane, int D) {
  if constexpr (L != SCALARS) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
      const int p = Chunk<L>::at(base, lane, i * 16 / (int)sizeof(T));
      const uint4 v = p < D ? __ldg(reinterpret_cast<const uint4*>(row + p)) : make_uint4(0, 0, 0, 0);
      r.w[4 * i] = v.x, r.w[4 * i + 1] = v.y, r.w[4 * i + 2] = v.z, r.w[4 * i + 3] = v.w;
    }
  } else {
    // 16-bit values: one address and fixed distances from it (backward of 16384 x 4095 bf16 119 us, with an
    // address for each value 130). Float32 keeps an address for each: 16383 x 1001 forward 25 us, else 30.
    const T* const from = row + base + lane;
    const int left = D - base - lane;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (sizeof(T) == 4) {
        const int p = base + j * 32 + lane;
        r.w[j] = p < D ? __ldg(reinterpret_cast<const uint32_t*>(row) + p) : 0u;
      } else {
        const uint32_t v = j * 32 < left ? (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(from) + j * 32) : 0u;
        if (j & 1) r.w[j / 2] |= v << 16; else r.w[j / 2] = v;
      }
    }
  }
}
template <typename T> __device__ __forceinline__ void to_float(const Raw8<T>& r, F2 (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      v[i] = f2(__uint_as_float(r.w[2 * i]), __uint_as_float(r.w[2 * i + 1]));
    } else {
      const float2 f = unpack2<T>(r.w[i]);
      v[i] = f2(f.x, f.y);
    }
  }
}
__device__ __forceinline__ void to_scalars(const F2 (&v)[4], float (&s)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = split(v[i]);
    s[2 * i] = f.x, s[2 * i + 1] = f.y;
  }
}
template <typename T, Layout L>
__device__ __forceinline__ void load8(F2 (&v)[4], const T* __restrict__ row, int base, int lane, int D) {
  Raw8<T> r;
  load_raw<T, L>(r, row, base, lane, D);
  to_float<T>(r, v);
}
template <typename T, Layout L>
__device__ __forceinline__ void store8(T* __restrict__ row, const F2 (&f)[4], int base, int lane, int D) {
  float v[8];
  to_scalars(f, v);
  if constexpr (L != SCALARS) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
      const int p = Chunk<L>::at(base, lane, i * 16 / (int)sizeof(T));
      if (p >= D) return;
      if constexpr (sizeof(T) == 4)
        *reinterpret_cast<float4*>(row + p) = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
      else
        *reinterpret_cast<uint4*>(row + p) = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
    }
  } else {
    T* const from = row + base + lane;
    const int left = D - base - lane;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (sizeof(T) == 4) {
        const int p = base + j * 32 + lane;
        if (p < D) st(row + p, v[j]);
      } else {
        if (j * 32 < left) st(from + j * 32, v[j]);
      }
    }
  }
}

// Zeros in the place of a chunk's elements at or beyond D
template <Layout L> __device__ __forceinline__ void zero_beyond(F2 (&v)[4], int base, int lane, int D) {
  if (Chunk<L>::has(base, lane, 7, D)) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 r = split(v[i]);
    v[i] = f2(Chunk<L>::has(base, lane, 2 * i, D) ? r.x : 0.f, Chunk<L>::has(base, lane, 2 * i + 1, D) ? r.y : 0.f);
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
template <Layout L>
__device__ __forceinline__ void store_codes(int8_t* __restrict__ row, const uint32_t (&q)[8], int base, int lane, int D) {
  const uint32_t lo = bytes4(q[0], q[1], q[2], q[3]), hi = bytes4(q[4], q[5], q[6], q[7]);
  if constexpr (L == EIGHT) {
    const int p = base + lane * 8;
    if (p < D) *reinterpret_cast<uint2*>(row + p) = make_uint2(lo, hi);
  } else if constexpr (L == FOURS) {
    const int p = base + lane * 4;
    if (p < D) *reinterpret_cast<uint32_t*>(row + p) = lo;
    if (p + kBlock < D) *reinterpret_cast<uint32_t*>(row + p + kBlock) = hi;
  } else {
    int8_t* const from = row + base + lane;
    const int left = D - base - lane;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j * 32 < left) from[j * 32] = (int8_t)(q[j] & 0xffu);
  }
}
template <Layout L>
__device__ __forceinline__ uint2 load_codes(const int8_t* __restrict__ row, int base, int lane, int D) {
  uint2 r = make_uint2(0, 0);
  if constexpr (L == EIGHT) {
    const int p = base + lane * 8;
    if (p < D) r = __ldg(reinterpret_cast<const uint2*>(row + p));
  } else if constexpr (L == FOURS) {
    const int p = base + lane * 4;
    if (p < D) r.x = __ldg(reinterpret_cast<const uint32_t*>(row + p));
    if (p + kBlock < D) r.y = __ldg(reinterpret_cast<const uint32_t*>(row + p + kBlock));
  } else {
    const int8_t* const from = row + base + lane;
    const int left = D - base - lane;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t v = j * 32 < left ? (uint32_t)(uint8_t)from[j * 32] : 0u;
      if (j < 4) r.x |= v << (8 * j); else r.y |= v << (8 * (j - 4));
    }
  }
  return r;
}
// A signed byte b as a float: 2^23 + (b + 128) has b + 128 in its low byte.
__device__ __forceinline__ void codes_to_float(uint2 c, F2 (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t b = (i < 2 ? c.x : c.y) ^ 0x80808080u;
    const int j = 2 * (i & 1);
    v[i] = add2(f2(__uint_as_float(__byte_perm(b, 0x4B000000u, 0x7540 | j)), __uint_as_float(__byte_perm(b, 0x4B000000u, 0x7541 | j))),
                f2(-8388736.f));
  }
}

// A row in 8-bit integers, from the bits of its largest magnitude a: factor 127 / a, scale a / 127. An infinity or NaN in
// the row makes its scale, and so all that is computed with it, NaN. Below 2^-118 the factor would be
// infinite: such a row counts as zeros (factor 0).
__device__ __forceinline__ float int8_factor(uint32_t amax_bits) {
  const float a = __uint_as_float(amax_bits);
  return amax_bits >= 0x7f800000u || a < 3.0092655e-36f ? 0.f : 127.f / a;
}
__device__ __forceinline__ float int8_scale(uint32_t amax_bits) {
  return amax_bits >= 0x7f800000u ? __uint_as_float(0x7fffffffu) : __uint_as_float(amax_bits) / 127.f;
}
// Product and rounding apart, each rounded as written (as a packed pair they come out as one multiply-add,
// with another code now and then)
__device__ __forceinline__ void int8_codes(const F2 (&v)[4], float factor, uint32_t (&q)[8]) {
  float t[8];
  to_scalars(v, t);
#pragma unroll
  for (int j = 0; j < 8; ++j) q[j] = factor == 0.f ? 0u : code_of(__fmul_rn(t[j], factor));
}

// ---- the kept form --------------------------------------------------------------------------------
// A block of 128 consecutive elements is kept as codes c of magnitude at most 127 and one byte E:
// element = c * 2^(E - 127), E the smallest of at least 1 for which the block's largest magnitude a still
// rounds to at most 127 (a < 127.5 * 2^(E - 127)). A block with an infinity or NaN gets E = 255 and comes
// back as NaN. Powers of two because then scaling is exact: codes are the same for every order of
// computing them, an element of a 16-bit type times its inverse scale is exact in float32, and what comes
// back fits bfloat16 without a second rounding. With a unit of a / 127 instead, the rounding error would
// be smaller by up to a factor of two.
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

// The largest magnitude's bits among a lane's eight elements (EIGHT), or its first four and last four. 16-bit
// types: the packed halves' as 16-bit integers first, then as the float32 they are.
template <typename T> __device__ __forceinline__ uint32_t float_bits(uint32_t h) {
  if constexpr (std::is_same<T, __half>::value) return __float_as_uint(__half2float(__ushort_as_half((unsigned short)h)));
  else return h << 16;
}
__device__ __forceinline__ uint32_t max2_u16(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t max_halves(uint32_t v) { return max(v & 0xffffu, v >> 16); }
template <typename T, Layout L> __device__ __forceinline__ void max_bits(const Raw8<T>& r, uint32_t (&m)[L == EIGHT ? 1 : 2]) {
  if constexpr (sizeof(T) == 4) {
    constexpr uint32_t k = 0x7fffffffu;
    const uint32_t lo = max(__vimax3_u32(r.w[0] & k, r.w[1] & k, r.w[2] & k), r.w[3] & k);
    const uint32_t hi = max(__vimax3_u32(r.w[4] & k, r.w[5] & k, r.w[6] & k), r.w[7] & k);
    if constexpr (L == EIGHT) m[0] = max(lo, hi); else m[0] = lo, m[1] = hi;
  } else {
    constexpr uint32_t k = 0x7fff7fffu;
    const uint32_t lo = max2_u16(r.w[0] & k, r.w[1] & k), hi = max2_u16(r.w[2] & k, r.w[3] & k);
    if constexpr (L == EIGHT) m[0] = float_bits<T>(max_halves(max2_u16(lo, hi)));
    else m[0] = float_bits<T>(max_halves(lo)), m[1] = float_bits<T>(max_halves(hi));
  }
}
// The same of eight floats. A NaN among them gives a NaN's bits, also beside the zeros beyond a row's end.
__device__ __forceinline__ float max3_abs(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
template <Layout L> __device__ __forceinline__ void max_bits(const F2 (&f)[4], uint32_t (&m)[L == EIGHT ? 1 : 2]) {
  float v[8];
  to_scalars(f, v);
  const float lo = max3_abs(max3_abs(v[0], v[1], v[2]), v[3], 0.f);
  if constexpr (L == EIGHT) {
    m[0] = abs_bits(max3_abs(max3_abs(lo, v[4], v[5]), v[6], v[7]));
  } else {
    m[0] = abs_bits(lo);
    m[1] = abs_bits(max3_abs(max3_abs(v[4], v[5], v[6]), v[7], 0.f));
  }
}

// Keeps a lane's eight elements (chunk at `base`), whose largest magnitudes' bits are m: codes to `crow`,
// the two blocks' E to `erow`. All 32 lanes take part; elements at or beyond D must be zero.
template <Layout L>
__device__ __forceinline__ void keep8(const F2 (&v)[4], const uint32_t (&m)[L == EIGHT ? 1 : 2], int8_t* __restrict__ crow,
                                      uint8_t* __restrict__ erow, int base, int lane, int D) {
  uint32_t q[8], e[2];
  if constexpr (L == EIGHT) {
    e[0] = e[1] = block_exp(__reduce_max_sync(lane < 16 ? 0xffffu : 0xffff0000u, m[0]));
    if ((lane & 15) == 0 && base + lane * 8 < D) erow[(base + lane * 8) / kBlock] = (uint8_t)e[0];
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) e[h] = block_exp(__reduce_max_sync(0xffffffffu, m[h]));
    if (lane < 2 && base + lane * kBlock < D) erow[base / kBlock + lane] = (uint8_t)(lane ? e[1] : e[0]);
  }
  if (max(e[0], e[1]) < 249u) {
    // the unit's inverse, 2^(127 - E), has 254 - E in the exponent field; the product with it is exact, so the sum's
    // rounding is the only one
    const float f[2] = {__uint_as_float((254u - e[0]) << 23), __uint_as_float((254u - e[1]) << 23)};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 r = split(fma2(v[i], f2(f[L == EIGHT ? 0 : i / 2]), f2(kRound)));
      q[2 * i] = __float_as_uint(r.x), q[2 * i + 1] = __float_as_uint(r.y);
    }
  } else {
    // E = 249, the largest, has 64 for a magnitude that its own type holds and 64 * 2^122 exceeds float32: 63
    // then. A bad block's codes are not read.
    constexpr float top = 63.f * 5.316911983139664e36f;
    float s[8];
    to_scalars(v, s);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t ej = e[L == EIGHT ? 0 : j / 4];
      q[j] = code_of(fminf(fmaxf(s[j], -top), top) * __uint_as_float((254u - (ej > 249u ? 249u : ej)) << 23));
    }
  }
  store_codes<L>(crow, q, base, lane, D);
}

// What a lane's eight kept elements stand for (zero at or beyond D).
struct Kept8 {
  uint2 c;
  uint32_t e;  // two bytes: the E of the lane's first four and last four elements
};
template <Layout L>
__device__ __forceinline__ uint32_t load_exps(const uint8_t* __restrict__ erow, int base, int lane, int D) {
  if constexpr (L == EIGHT) return base + lane * 8 < D ? __ldg(erow + (base + lane * 8) / kBlock) : 1u;
  uint32_t e = base < D ? __ldg(erow + base / kBlock) : 1u;
  return e | (base + kBlock < D ? (uint32_t)__ldg(erow + base / kBlock + 1) : 1u) << 8;
}
template <Layout L>
__device__ __forceinline__ Kept8 load_kept(const int8_t* __restrict__ crow, const uint8_t* __restrict__ erow,
                                           int base, int lane, int D) {
  return Kept8{load_codes<L>(crow, base, lane, D), load_exps<L>(erow, base, lane, D)};
}
template <Layout L> __device__ __forceinline__ void kept_to_float(const Kept8& k, F2 (&v)[4]) {
  codes_to_float(k.c, v);
  const float s0 = scale_of(k.e & 0xffu), s1 = L == EIGHT ? s0 : scale_of(k.e >> 8);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = mul2(v[i], f2(i < 2 ? s0 : s1));
}

// Where the codes of [.., D] rows lie: rows of this many bytes, and this many E bytes a row.
__host__ __device__ inline int64_t code_pitch(int64_t D) { return (D + 15) & ~(int64_t)15; }
__host__ __device__ inline int64_t blocks_of(int64_t D) { return (D + kBlock - 1) / kBlock; }

// ---- rows ahead ------------------------------------------------------------------------------------
// Copies of the rows ahead, in shared memory, in pieces of 16 bytes. In the layouts of whole 16-byte accesses a
// thread copies, and later reads, only its own elements, so its own wait for its copies is all the
// synchronisation there is. Rows that do not start on 16 bytes (SCALARS) are copied from the 16 bytes that their
// chunk starts in to those that it ends in, by the warp that reads them: it meets after the wait, and
// before the place is copied to again. (A norm's forward over 16383 x 1001 float32 takes 26 us so, 30 with copies
// of 4 bytes; over 16384 x 4095 bfloat16 79 us, 100 with the row loaded when its turn comes.)
__device__ __forceinline__ uint32_t shared_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
template <int BYTES> __device__ __forceinline__ void copy_async(uint32_t dst, const void* src, bool there) {
  // with no source bytes the destination is filled with zeros
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(there ? BYTES : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Bytes of a chunk of each of a block's warps. In the layouts of whole accesses: [word group][thread], so that a
// warp's accesses are contiguous.
template <typename T, Layout L> __host__ __device__ constexpr int copy_bytes(int threads) {
  return L != SCALARS ? 8 * (int)sizeof(T) * threads : (256 * (int)sizeof(T) + 16) * (threads / 32);
}
template <typename T, Layout L>
__device__ __forceinline__ void copy8(uint8_t* slot, const T* row, int base, int lane, int D) {
  if constexpr (L != SCALARS) {
    const uint32_t at = shared_addr(slot);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
      const int p = Chunk<L>::at(base, lane, i * 16 / (int)sizeof(T));
      copy_async<16>(at + (i * blockDim.x + threadIdx.x) * 16, row + (p < D ? p : 0), p < D);
    }
  } else {
    constexpr int kPieces = 256 * (int)sizeof(T) / 16 + 1;
    const uint32_t at = shared_addr(slot) + (threadIdx.x >> 5) * (256 * (int)sizeof(T) + 16);
    const uintptr_t from = reinterpret_cast<uintptr_t>(row + base) & ~(uintptr_t)15, end = reinterpret_cast<uintptr_t>(row + D);
    if (base < D) {
#pragma unroll
      for (int i = 0; i < (kPieces + 31) / 32; ++i) {
        // a piece that holds an element of the row; what else it holds is not read
        const int n = i * 32 + lane;
        const uintptr_t src = from + 16 * (uintptr_t)n;
        if (n < kPieces && src < end) copy_async<16>(at + 16 * n, reinterpret_cast<const void*>(src), true);
      }
    }
  }
}
template <typename T, Layout L>
__device__ __forceinline__ void copied_raw(const uint8_t* slot, Raw8<T>& r, const T* row, int base, int lane, int D) {
  if constexpr (L != SCALARS) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
      const uint4 u = reinterpret_cast<const uint4*>(slot)[i * blockDim.x + threadIdx.x];
      r.w[4 * i] = u.x, r.w[4 * i + 1] = u.y, r.w[4 * i + 2] = u.z, r.w[4 * i + 3] = u.w;
    }
  } else {
    const uint8_t* mine = slot + (threadIdx.x >> 5) * (256 * (int)sizeof(T) + 16) + (reinterpret_cast<uintptr_t>(row + base) & 15u);
    const int left = D - base - lane;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const bool has = j * 32 < left;
      if constexpr (sizeof(T) == 4) {
        r.w[j] = has ? reinterpret_cast<const uint32_t*>(mine)[j * 32 + lane] : 0u;
      } else {
        const uint32_t v = has ? (uint32_t)reinterpret_cast<const uint16_t*>(mine)[j * 32 + lane] : 0u;
        if (j & 1) r.w[j / 2] |= v << 16; else r.w[j / 2] = v;
      }
    }
  }
}
template <typename T, Layout L>
__device__ __forceinline__ void copied8(const uint8_t* slot, F2 (&v)[4], const T* row, int base, int lane, int D) {
  Raw8<T> r;
  copied_raw<T, L>(slot, r, row, base, lane, D);
  to_float<T>(r, v);
}
// The same for codes, 8 bytes a thread; their rows start on 16 bytes in every layout.
template <Layout L>
__device__ __forceinline__ void copy_codes(uint8_t* slot, const int8_t* row, int base, int lane, int D) {
  const uint32_t at = shared_addr(slot);
  if constexpr (L == SCALARS) {
    const int p = base + lane * 16;
    if (lane < 16 && p < D) copy_async<16>(at + (threadIdx.x >> 5) * 256 + lane * 16, row + p, true);
  } else {
#pragma unroll
    for (int i = 0; i < (L == FOURS ? 2 : 1); ++i) {
      const int p = Chunk<L>::at(base, lane, 4 * i);
      copy_async<L == FOURS ? 4 : 8>(at + threadIdx.x * 8 + 4 * i, row + (p < D ? p : 0), p < D);
    }
  }
}
template <Layout L> __device__ __forceinline__ uint2 copied_codes(const uint8_t* slot, int base, int lane, int D) {
  if constexpr (L != SCALARS) return reinterpret_cast<const uint2*>(slot)[threadIdx.x];
  return load_codes<L>(reinterpret_cast<const int8_t*>(slot) + (threadIdx.x >> 5) * 256 - base, base, lane, D);
}
// Where a warp reads what all of its lanes have copied
template <Layout L> __device__ __forceinline__ void meet_copies() {
  if constexpr (L == SCALARS) __syncwarp();
}

// ---- reductions over a row ------------------------------------------------------------------------
// Over one warp, or over the whole block through `slot` (32 words, not used for anything else until every
// thread has passed a later barrier). Every thread gets the result, summed in the same order each time.
// The slots of warps that the block does not have hold zeros.
template <bool WARP> __device__ __forceinline__ float row_sum(float v, float* slot) {
  v = warp_sum(v);
  if constexpr (!WARP) {
    if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.f;
    for (int i = 0; i < (int)(blockDim.x >> 5); i += 4) {
      const float4 t = *reinterpret_cast<const float4*>(slot + i);
      v += (t.x + t.y) + (t.z + t.w);
    }
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
