// One AdamW step over many tensors, and its moments read out in 32 bits.
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,
//   p = p (1 - lr decay) - lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps)
//
// in float32, the sums of m and v as products and sums rounded one by one, so that what is rounded to 8 bits below does not
// depend on how a compiler contracts them. Bound by memory: 28 bytes an element with float32 parameters and moments,
// 16 with moments in 8 bits.
//
// 8-bit moments: blocks of 128 elements, with the biased float32 exponent E of the block's largest magnitude in a byte.
// A code is the float32's exponent relative to E and its first three bits of mantissa: for m a sign and 4 + 3 bits, the
// binades from 2^-14 of E's up to twice E's; v (never negative) 5 + 3 bits, from 2^-30. Code 0 is zero. Rounding adds 16
// random bits under the third bit of mantissa and cuts: up or down with the probability that keeps the mean, without
// which v, which loses a thousandth of itself a step where no gradient comes, would never move. (Its unit is an eighth
// to a sixteenth.) What is below the smallest code becomes zero for m, and the smallest for v, so that no m is divided by a v
// that is zero for its rounding alone. The random bits are a mix of the element's index, the step and a seed: the same
// every time. A block with an infinity or NaN is marked by E = 255 and comes back as NaN.
#include "rows.cuh"

namespace flb {

namespace {

constexpr int kThreads = 256;
constexpr int kBlockElems = 128;                    // a block of 8-bit moments: a warp's four elements a lane
constexpr int kUnroll = 4;                          // such blocks a warp has in flight
constexpr int kChunk = kThreads / 32 * kUnroll * kBlockElems;
constexpr int kBelowM = 14, kBitsM = 7, kBelowV = 30, kBitsV = 8;

struct Tensor {
  void* p;
  const void* g;
  void* m;        // float32, or codes
  void* v;
  uint8_t* me;    // null, or a byte a block
  uint8_t* ve;
  int64_t* step;  // steps taken before this one
  int64_t n;      // elements; negative: -n of them, not all of whose arrays allow vector access
};

// The tensors of one launch, in the kernel's parameters: no table to copy to the device, and none that a captured
// graph would have to keep.
template <int CAP> struct Table {
  Tensor t[CAP];
  uint32_t first[CAP + 1];  // chunks before each tensor
  int count;
};

struct Args {
  float b1, c1, b2, c2;     // c = 1 - b
  double log_b1, log_b2;
  double lr, decay;
  const float* lr_device;   // null, or in lr's place
  float eps;
  uint32_t seed;
  uint32_t* counter;        // blocks done; zero between launches
};

// Four consecutive elements from i on of n, zeros beyond.
template <typename T> __device__ __forceinline__ void load4(float (&x)[4], const T* p, int64_t i, int64_t n, bool vec) {
  if (vec && i + 4 <= n) {
    if constexpr (sizeof(T) == 4) {
      const float4 a = *reinterpret_cast<const float4*>(p + i);
      x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
    } else {
      const uint2 a = *reinterpret_cast<const uint2*>(p + i);
      const float2 lo = rows::unpack2<T>(a.x), hi = rows::unpack2<T>(a.y);
      x[0] = lo.x, x[1] = lo.y, x[2] = hi.x, x[3] = hi.y;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = i + j < n ? ld(p + i + j) : 0.f;
  }
}
template <typename T> __device__ __forceinline__ void store4(T* p, const float (&x)[4], int64_t i, int64_t n, bool vec) {
  if (vec && i + 4 <= n) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(p + i) = make_float4(x[0], x[1], x[2], x[3]);
    else *reinterpret_cast<uint2*>(p + i) = make_uint2(rows::pack2<T>(x[0], x[1]), rows::pack2<T>(x[2], x[3]));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j < n) st(p + i + j, x[j]);
  }
}

// A code's float32 bits, without a sign: base = (E - below) * 8. Not for a block marked as NaN.
template <int BITS> __device__ __forceinline__ float decode(uint32_t code, int base) {
  const uint32_t low = code & ((1u << BITS) - 1);
  uint32_t u = low ? (low + base) << 20 : 0u;
  if (BITS == 7) u |= (code >> 7) << 31;
  return __uint_as_float(u);
}
// size: a magnitude's bits. noise: 16 random bits, from bit 4 on.
template <bool UNSIGNED> __device__ __forceinline__ uint32_t encode(uint32_t size, uint32_t noise, int base) {
  // (up to the largest finite exponent)
  const int key = (int)min((size + noise) >> 20, 254u * 8 + 7) - base;
  if (UNSIGNED) return size ? (uint32_t)max(key, 1) : 0u;
  return (uint32_t)max(key, 0);
}
// E of a block whose largest magnitude has these bits, not below the least for which every code is a normal number
__device__ __forceinline__ int block_exponent(uint32_t top, int below) { return max((int)(top >> 23), below + 1); }

__device__ __forceinline__ uint32_t mix(uint32_t i, uint32_t step_and_seed) {
  uint32_t x = i * 0x9E3779B9u + step_and_seed;  // the golden ratio's and the roots' of 2 and 3 first digits
  x = (x ^ (x >> 16)) * 0xBB67AE85u;
  return x ^ (x >> 16);
}

template <typename T, int BITS, int CAP>
__global__ void __launch_bounds__(kThreads) adamw_kernel(const __grid_constant__ Table<CAP> tb, const Args a) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t chunks = tb.first[tb.count];
  int64_t known = -1;  // the step whose factors these are
  float keep = 0, rate = 0, root = 0;
  for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) {
    int lo = 0, hi = tb.count - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (tb.first[mid] <= c) lo = mid; else hi = mid - 1;
    }
    const Tensor& t = tb.t[lo];
    const bool vec = t.n >= 0;
    const int64_t n = vec ? t.n : -t.n;
    const int64_t from = (int64_t)(c - tb.first[lo]) * kChunk + warp * (kUnroll * kBlockElems) + lane * 4;
    float p[kUnroll][4], g[kUnroll][4], m[kUnroll][4], v[kUnroll][4];
    uint32_t cm[kUnroll], cv[kUnroll], exps = 0;
    const int64_t block0 = (from - lane * 4) / kBlockElems, blocks = (n + kBlockElems - 1) / kBlockElems;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t i = from + u * kBlockElems;
      load4(p[u], static_cast<const T*>(t.p), i, n, vec);
      load4(g[u], static_cast<const T*>(t.g), i, n, vec);
      if constexpr (BITS == 32) {
        load4(m[u], static_cast<const float*>(t.m), i, n, vec);
        load4(v[u], static_cast<const float*>(t.v), i, n, vec);
      } else {
        const bool there = block0 + u < blocks;
        cm[u] = there ? static_cast<const uint32_t*>(t.m)[i / 4] : 0u;
        cv[u] = there ? static_cast<const uint32_t*>(t.v)[i / 4] : 0u;
      }
    }
    // lanes 0 to 3 have the four blocks' bytes of m, 4 to 7 those of v
    const bool has_byte = BITS == 8 && lane < 2 * kUnroll && block0 + lane % kUnroll < blocks;
    uint8_t* const byte = (lane < kUnroll ? t.me : t.ve) + block0 + lane % kUnroll;
    if (has_byte) exps = *byte;
    const int64_t step = *t.step + 1;
    if (step != known) {
      known = step;
      const double lr = a.lr_device ? (double)*a.lr_device : a.lr;
      keep = (float)(1.0 - lr * a.decay);
      rate = (float)(lr / -expm1((double)step * a.log_b1));
      root = (float)rsqrt(-expm1((double)step * a.log_b2));
    }
    const uint32_t salt = (uint32_t)step * 0x6A09E667u + a.seed;
    uint32_t kept_exps = 0;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t i = from + u * kBlockElems;
      if constexpr (BITS == 8) {
        const int em = __shfl_sync(0xffffffffu, exps, u), ev = __shfl_sync(0xffffffffu, exps, kUnroll + u);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          m[u][j] = decode<kBitsM>(cm[u] >> (8 * j) & 255, (em - kBelowM) * 8);
          v[u][j] = decode<kBitsV>(cv[u] >> (8 * j) & 255, (ev - kBelowV) * 8);
          if (em == 255) m[u][j] = __uint_as_float(0x7fffffffu);
          if (ev == 255) v[u][j] = __uint_as_float(0x7fffffffu);
        }
      }
      uint32_t top_m = 0, top_v = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float gj = g[u][j];
        m[u][j] = __fadd_rn(__fmul_rn(m[u][j], a.b1), __fmul_rn(gj, a.c1));
        v[u][j] = __fadd_rn(__fmul_rn(v[u][j], a.b2), __fmul_rn(__fmul_rn(gj, gj), a.c2));
        const float q = __fdividef(m[u][j], fmaf(sqrtf(v[u][j]), root, a.eps));
        p[u][j] = fmaf(p[u][j], keep, -rate * q);
        if constexpr (BITS == 8) {
          // places beyond the last element hold zeros, and stay zeros
          top_m = max(top_m, __float_as_uint(m[u][j]) & 0x7fffffffu);
          top_v = max(top_v, __float_as_uint(v[u][j]) & 0x7fffffffu);
        }
      }
      store4(static_cast<T*>(t.p), p[u], i, n, vec);
      if constexpr (BITS == 32) {
        store4(static_cast<float*>(t.m), m[u], i, n, vec);
        store4(static_cast<float*>(t.v), v[u], i, n, vec);
      } else {
        top_m = __reduce_max_sync(0xffffffffu, top_m);
        top_v = __reduce_max_sync(0xffffffffu, top_v);
        const int em = block_exponent(top_m, kBelowM), ev = block_exponent(top_v, kBelowV);
        uint32_t wm = 0, wv = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t r = mix((uint32_t)i + j, salt);
          const uint32_t bits_m = __float_as_uint(m[u][j]);
          const uint32_t km = encode<false>(bits_m & 0x7fffffffu, r >> 16 << 4, (em - kBelowM) * 8);
          wm |= (km | (bits_m >> 31 && km ? 128u : 0u)) << (8 * j);
          wv |= encode<true>(__float_as_uint(v[u][j]), (r & 0xffffu) << 4, (ev - kBelowV) * 8) << (8 * j);
        }
        if (block0 + u < blocks) {
          static_cast<uint32_t*>(t.m)[i / 4] = wm;
          static_cast<uint32_t*>(t.v)[i / 4] = wv;
        }
        if (lane == u) kept_exps = em;
        if (lane == kUnroll + u) kept_exps = ev;
      }
    }
    if (has_byte) *byte = (uint8_t)kept_exps;
  }
  // The steps count up once every block has read them: by the last block to end.
  __shared__ bool last;
  __syncthreads();
  if (threadIdx.x == 0) last = atomicInc(a.counter, gridDim.x - 1) == gridDim.x - 1;
  __syncthreads();
  if (last)
    for (int i = threadIdx.x; i < tb.count; i += kThreads) ++*tb.t[i].step;
}

// Codes into float32: p and g are where m and v go (either may be null).
template <int CAP> __global__ void __launch_bounds__(kThreads) moments_kernel(const __grid_constant__ Table<CAP> tb) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t chunks = tb.first[tb.count];
  for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) {
    int lo = 0, hi = tb.count - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (tb.first[mid] <= c) lo = mid; else hi = mid - 1;
    }
    const Tensor& t = tb.t[lo];
    const bool vec = t.n >= 0;
    const int64_t n = vec ? t.n : -t.n, blocks = (n + kBlockElems - 1) / kBlockElems;
    const int64_t from = (int64_t)(c - tb.first[lo]) * kChunk + warp * (kUnroll * kBlockElems) + lane * 4;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t i = from + u * kBlockElems, block = i / kBlockElems;
      if (block >= blocks) break;
      const uint32_t cm = static_cast<const uint32_t*>(t.m)[i / 4], cv = static_cast<const uint32_t*>(t.v)[i / 4];
      const int em = t.me[block], ev = t.ve[block];
      float m[4], v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        m[j] = em == 255 ? __uint_as_float(0x7fffffffu) : decode<kBitsM>(cm >> (8 * j) & 255, (em - kBelowM) * 8);
        v[j] = ev == 255 ? __uint_as_float(0x7fffffffu) : decode<kBitsV>(cv >> (8 * j) & 255, (ev - kBelowV) * 8);
      }
      store4(static_cast<float*>(t.p), m, i, n, vec);
      store4(static_cast<float*>(const_cast<void*>(t.g)), v, i, n, vec);
    }
  }
}

// Fills tables of up to CAP tensors and launches for each.
template <int CAP, typename Launch>
int in_tables(const flb_adamw_tensor* t, int64_t count, int elem, int state_bits, Launch&& launch) {
  static_assert(sizeof(Table<CAP>) <= 32 * 1024, "a launch's parameters");
  Table<CAP> tb;
  auto off = [](const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) != 0; };
  for (int64_t from = 0; from < count;) {
    tb.count = 0;
    tb.first[0] = 0;
    while (from < count && tb.count < CAP) {
      const flb_adamw_tensor& s = t[from];
      const int64_t chunks = (s.n + kChunk - 1) / kChunk;
      if (chunks > 0 && chunks + tb.first[tb.count] > INT32_MAX) break;
      ++from;
      if (chunks == 0 && !s.step) continue;
      const bool vec = !off(s.p, 4 * elem) && !off(s.g, 4 * elem) && (state_bits == 8 || (!off(s.m, 16) && !off(s.v, 16)));
      tb.t[tb.count] = Tensor{s.p, s.g, s.m, s.v, s.m_exps, s.v_exps, s.step, vec ? s.n : -s.n};
      tb.first[tb.count + 1] = tb.first[tb.count] + (uint32_t)chunks;
      ++tb.count;
    }
    if (tb.count == 0) continue;
    const int st = launch(tb);
    if (st != FLB_OK) return st;
  }
  return FLB_OK;
}

unsigned grid_of(uint32_t chunks, int per_sm) { return (unsigned)std::max<int64_t>(1, std::min<int64_t>(chunks, (int64_t)num_sms() * per_sm)); }

template <typename T, int BITS, int CAP> int step_tables(const flb_adamw_tensor* t, int64_t count, const Args& a, cudaStream_t s) {
  return in_tables<CAP>(t, count, sizeof(T), BITS, [&](const Table<CAP>& tb) {
    adamw_kernel<T, BITS, CAP><<<grid_of(tb.first[tb.count], 4), kThreads, 0, s>>>(tb, a);
    count_launches(1);
    return check_cuda(cudaGetLastError(), "adamw launch");
  });
}
// a launch's parameters are copied whole: a small table for few tensors
template <typename T, int BITS> int step_t(const flb_adamw_tensor* t, int64_t count, const Args& a, cudaStream_t s) {
  return count <= 48 ? step_tables<T, BITS, 48>(t, count, a, s) : step_tables<T, BITS, 440>(t, count, a, s);
}
template <typename T> int step_b(const flb_adamw_tensor* t, int64_t count, int bits, const Args& a, cudaStream_t s) {
  return bits == 8 ? step_t<T, 8>(t, count, a, s) : step_t<T, 32>(t, count, a, s);
}

}  // namespace

int adamw(const flb_adamw_tensor* t, int64_t count, int dtype, int state_bits, double lr, const float* lr_device, double b1, double b2,
          double eps, double decay, uint32_t seed, uint32_t* counter, cudaStream_t s) {
  Args a = {};
  a.b1 = (float)b1, a.c1 = (float)(1 - b1), a.b2 = (float)b2, a.c2 = (float)(1 - b2);
  a.log_b1 = log(b1), a.log_b2 = log(b2);
  a.lr = lr, a.lr_device = lr_device, a.decay = decay, a.eps = (float)eps, a.seed = seed, a.counter = counter;
  switch (dtype) {
    case FLB_F32: return step_b<float>(t, count, state_bits, a, s);
    case FLB_F16: return step_b<__half>(t, count, state_bits, a, s);
    default: return step_b<__nv_bfloat16>(t, count, state_bits, a, s);
  }
}

int adamw_moments(const flb_adamw_tensor* t, int64_t count, cudaStream_t s) {
  return in_tables<440>(t, count, 4, 8, [&](const Table<440>& tb) {
    if (tb.first[tb.count] == 0) return (int)FLB_OK;
    moments_kernel<440><<<grid_of(tb.first[tb.count], 8), kThreads, 0, s>>>(tb);
    count_launches(1);
    return check_cuda(cudaGetLastError(), "adamw_moments launch");
  });
}

}  // namespace flb
