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
// every time, and the same in every tensor. Over thousands of steps v stands off its float64 value by 21% (root of the mean square; from 0.4 to
// 2.2 of it over 16384 elements, beta2 = 0.999), by 26% where one gradient in ten is not zero, with its mean kept to 0.2%.
// A block with an infinity or NaN is marked by E = 255 and comes back as NaN.
#include "rows.cuh"

namespace flb {

namespace {

constexpr int kThreads = 256;
constexpr int kBlockElems = 128;                    // a block of 8-bit moments: a warp's four elements a lane
// Such blocks a warp has in flight, thread blocks an SM, and elements of a tensor that a thread block takes at a time. (Moments in 8 bits with two
// blocks in flight and four thread blocks: 391 us for 106 million float32, with four and three 365, before a chunk was several such steps.)
constexpr int kUnroll = 4;
template <int BITS> constexpr int kPerSm = BITS == 32 ? 2 : 3;
constexpr int kStep = kThreads / 32 * kUnroll * kBlockElems;
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
  int chunk;                // elements, a multiple of kStep
};

struct Args {
  float b1, c1, b2, c2;     // c = 1 - b
  double log_b1, log_b2;
  double lr, decay;
  const float* lr_device;   // null, or in lr's place
  float eps;
  bool flush;               // see quotient()
  uint32_t seed;
  uint32_t* counter;        // blocks done; zero between launches
  uint32_t place;           // 2^20
};

// Four consecutive elements from i on of n, zeros beyond. FULL: all are there, on 16 bytes (8 of 16-bit types).
template <bool FULL, typename T> __device__ __forceinline__ void load4(float (&x)[4], const T* p, int i, int n, bool vec) {
  if (FULL || (vec && i + 4 <= n)) {
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
template <bool FULL, typename T> __device__ __forceinline__ void store4(T* p, const float (&x)[4], int i, int n, bool vec) {
  if (FULL || (vec && i + 4 <= n)) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(p + i) = make_float4(x[0], x[1], x[2], x[3]);
    else *reinterpret_cast<uint2*>(p + i) = make_uint2(rows::pack2<T>(x[0], x[1]), rows::pack2<T>(x[2], x[3]));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j < n) st(p + i + j, x[j]);
  }
}

// Four codes of a block. base: (E - below) * 8 << 20, what a code's bits at their place in a float32 are short of that float32's. The 8-bit
// forms are bound by the integer units as much as by memory, so shifts here are multiplications by arguments (place: 2^20), which run
// beside those, and what is rare (zeros, marked blocks) is looked for four codes at a time.
template <int BITS> __device__ __forceinline__ void decode(float (&x)[4], uint32_t codes, int e, uint32_t base, uint32_t place) {
  const uint32_t low = BITS == 7 ? codes & 0x7f7f7f7fu : codes;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t u = __byte_perm(low, 0, 0x4440 + j) * place + base;
    if (BITS == 7) u |= codes << (24 - 8 * j) & 0x80000000u;
    x[j] = __uint_as_float(u);
  }
  if ((low - 0x01010101u) & ~low & 0x80808080u) {  // a zero among them
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (!(low >> (8 * j) & 255)) x[j] = 0.f;
  }
  if (e == 255) {  // the block's own, so of the whole warp
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = __uint_as_float(0x7fffffffu);
  }
}
// E of a block whose largest magnitude has these bits, not below the least for which every code is a normal number
__device__ __forceinline__ int block_exponent(uint32_t top, int below) { return max((int)(top >> 23), below + 1); }
__device__ __forceinline__ uint32_t base_of(int e, int below) { return (uint32_t)(e - below) << 23; }

// 32 random bits for element i: products with the first digits of the golden ratio and of the root of 3. Of the result x ^ x >> 16 the
// upper half is m's noise and the lower v's, both at bits 4 to 19.
__device__ __forceinline__ void noise_of(uint32_t i_and_salt, uint32_t& m, uint32_t& v) {
  const uint32_t x = (i_and_salt ^ (i_and_salt >> 16)) * 0xBB67AE85u, high = x >> 12;
  m = high & 0xffff0u;
  v = ((x << 4) ^ high) & 0xffff0u;
}
__device__ __forceinline__ uint32_t bytes_of(const uint32_t (&k)[4], int from) {
  return __byte_perm(__byte_perm(k[0], k[1], from | (4 + from) << 4), __byte_perm(k[2], k[3], from | (4 + from) << 4), 0x5410);
}
constexpr uint32_t kMix = 0x9E3779B9u;

// The tensor that a chunk belongs to, and its place there: from element `at` on, `left` of them.
template <int CAP> __device__ __forceinline__ const Tensor& tensor_of(const Table<CAP>& tb, uint32_t c, int64_t& at, int& left) {
  int lo = 0, hi = tb.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tb.first[mid] <= c) lo = mid; else hi = mid - 1;
  }
  const Tensor& t = tb.t[lo];
  at = (int64_t)(c - tb.first[lo]) * tb.chunk;
  left = (int)min((t.n >= 0 ? t.n : -t.n) - at, (int64_t)tb.chunk);
  return t;
}

// m / (sqrt(v) root + eps), root and quotient each within 2^-22. flush: eps is so large that it makes no difference whether v and m below float32's
// normal numbers count as zero, which saves the operations that scale them.
__device__ __forceinline__ float quotient(float m, float v, float root, float eps, bool flush) {
  float s, q;
  if (flush) {
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(v));
    asm("div.approx.ftz.f32 %0, %1, %2;" : "=f"(q) : "f"(m), "f"(fmaf(s, root, eps)));
  } else {
    asm("sqrt.approx.f32 %0, %1;" : "=f"(s) : "f"(v));
    asm("div.approx.f32 %0, %1, %2;" : "=f"(q) : "f"(m), "f"(fmaf(s, root, eps)));
  }
  return q;
}

template <typename T, int BITS, int CAP>
__global__ void __launch_bounds__(kThreads, kPerSm<BITS>) adamw_kernel(const __grid_constant__ Table<CAP> tb, const Args a) {
  constexpr int U = kUnroll;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t chunks = tb.first[tb.count];
  int64_t known = -1;  // the step whose factors these are
  float keep = 0, rate = 0, root = 0;
  for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) {
    int64_t at;
    int left;
    const Tensor& t = tensor_of(tb, c, at, left);
    const bool vec = t.n >= 0;
    T* const pp = static_cast<T*>(t.p) + at;
    const T* const pg = static_cast<const T*>(t.g) + at;
    using State = std::conditional_t<BITS == 32, float, uint8_t>;
    State* const pm = static_cast<State*>(t.m) + at;
    State* const pv = static_cast<State*>(t.v) + at;
    const int blocks = (left + kBlockElems - 1) / kBlockElems;
    // the first U lanes have the bytes of a step's blocks of m, the next those of v
    uint8_t* const bytes = BITS == 8 ? (lane < U ? t.me : t.ve) + at / kBlockElems + lane % U : nullptr;
    const int64_t step = *t.step + 1;
    auto step_at = [&](int o, auto full) {
      constexpr bool FULL = decltype(full)::value;
      float p[U][4], g[U][4], m[U][4], v[U][4];
      [[maybe_unused]] uint32_t cm[U], cv[U], exps = 0;
      const int block0 = o / kBlockElems;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = o + u * kBlockElems + lane * 4;
        load4<FULL>(p[u], pp, i, left, vec);
        load4<FULL>(g[u], pg, i, left, vec);
        if constexpr (BITS == 32) {
          load4<FULL>(m[u], pm, i, left, vec);
          load4<FULL>(v[u], pv, i, left, vec);
        } else {
          const bool there = FULL || block0 + u < blocks;
          cm[u] = there ? *reinterpret_cast<const uint32_t*>(pm + i) : 0u;
          cv[u] = there ? *reinterpret_cast<const uint32_t*>(pv + i) : 0u;
        }
      }
      const bool has_byte = BITS == 8 && lane < 2 * U && (FULL || block0 + lane % U < blocks);
      if (has_byte) exps = bytes[block0];
      if (step != known) {
        known = step;
        const double lr = a.lr_device ? (double)*a.lr_device : a.lr;
        keep = (float)(1.0 - lr * a.decay);
        rate = (float)(lr / expm1((double)step * a.log_b1));  // (negative)
        root = (float)rsqrt(-expm1((double)step * a.log_b2));
      }
      // (the root of 2's digits)
      [[maybe_unused]] const uint32_t salt = ((uint32_t)at + o + lane * 4) * kMix + (uint32_t)step * 0x6A09E667u + a.seed;
      [[maybe_unused]] uint32_t kept_exps = 0;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = o + u * kBlockElems + lane * 4;
        if constexpr (BITS == 8) {
          const int em = __shfl_sync(0xffffffffu, exps, u), ev = __shfl_sync(0xffffffffu, exps, U + u);
          decode<kBitsM>(m[u], cm[u], em, base_of(em, kBelowM), a.place);
          decode<kBitsV>(v[u], cv[u], ev, base_of(ev, kBelowV), a.place);
        }
        [[maybe_unused]] uint32_t top_m = 0, top_v = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float gj = g[u][j];
          m[u][j] = __fadd_rn(__fmul_rn(m[u][j], a.b1), __fmul_rn(gj, a.c1));
          v[u][j] = __fadd_rn(__fmul_rn(v[u][j], a.b2), __fmul_rn(__fmul_rn(gj, gj), a.c2));
          p[u][j] = fmaf(p[u][j], keep, rate * quotient(m[u][j], v[u][j], root, a.eps, a.flush));
          if constexpr (BITS == 8) {
            // places beyond the last element hold zeros, and stay zeros
            top_m = max(top_m, __float_as_uint(m[u][j]) & 0x7fffffffu);
            top_v = max(top_v, __float_as_uint(v[u][j]) & 0x7fffffffu);
          }
        }
        store4<FULL>(pp, p[u], i, left, vec);
        if constexpr (BITS == 32) {
          store4<FULL>(pm, m[u], i, left, vec);
          store4<FULL>(pv, v[u], i, left, vec);
        } else {
          top_m = __reduce_max_sync(0xffffffffu, top_m);
          top_v = __reduce_max_sync(0xffffffffu, top_v);
          const int em = block_exponent(top_m, kBelowM), ev = block_exponent(top_v, kBelowV);
          const uint32_t base_m = base_of(em, kBelowM), base_v = base_of(ev, kBelowV);
          uint32_t km[4], kv[4], bits_m[4];
          bool zero = false;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t noise_m, noise_v;
            noise_of(salt + (uint32_t)(u * kBlockElems + j) * kMix, noise_m, noise_v);
            bits_m[j] = __float_as_uint(m[u][j]);
            const uint32_t size_m = bits_m[j] & 0x7fffffffu, size_v = __float_as_uint(v[u][j]);
            km[j] = (uint32_t)max((int)(size_m + noise_m - base_m) >> 20, 0);
            kv[j] = (uint32_t)max((int)(size_v + noise_v - base_v) >> 20, 1);
            zero |= size_v == 0;
          }
          if (zero) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (v[u][j] == 0) kv[j] = 0;
          }
          if (max(em, ev) >= 254) {  // up to the largest finite exponent (of the whole warp)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              km[j] = min(km[j], (254u * 8 + 7) - (base_m >> 20));
              kv[j] = min(kv[j], (254u * 8 + 7) - (base_v >> 20));
            }
          }
          if (FULL || block0 + u < blocks) {
            *reinterpret_cast<uint32_t*>(pm + i) = bytes_of(km, 0) | (bytes_of(bits_m, 3) & 0x80808080u);
            *reinterpret_cast<uint32_t*>(pv + i) = bytes_of(kv, 0);
          }
          if (lane == u) kept_exps = em;
          if (lane == U + u) kept_exps = ev;
        }
      }
      if (has_byte) bytes[block0] = (uint8_t)kept_exps;
    };
#pragma unroll 1
    for (int o = warp * U * kBlockElems; o < left; o += kStep) {
      if (vec && o + U * kBlockElems <= left) step_at(o, std::true_type());
      else step_at(o, std::false_type());
    }
  }
  // The steps count up once every block has read them: by the last block to end.
  __shared__ bool last;
  __syncthreads();
  if (threadIdx.x == 0) last = atomicInc(a.counter, gridDim.x - 1) == gridDim.x - 1;
  __syncthreads();
  if (last)
    for (int i = threadIdx.x; i < tb.count; i += kThreads) ++*tb.t[i].step;
}

// Codes into float32: p and g are where m and v go.
template <int CAP> __global__ void __launch_bounds__(kThreads) moments_kernel(const __grid_constant__ Table<CAP> tb) {
  constexpr int U = kUnroll;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t chunks = tb.first[tb.count];
  for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) {
    int64_t at;
    int left;
    const Tensor& t = tensor_of(tb, c, at, left);
    const bool vec = t.n >= 0;
    float* const to_m = static_cast<float*>(t.p) + at;
    float* const to_v = static_cast<float*>(const_cast<void*>(t.g)) + at;
    const uint8_t* const pm = static_cast<const uint8_t*>(t.m) + at;
    const uint8_t* const pv = static_cast<const uint8_t*>(t.v) + at;
    const uint8_t* const pe = (lane < U ? t.me : t.ve) + at / kBlockElems + lane % U;
    const int blocks = (left + kBlockElems - 1) / kBlockElems;
#pragma unroll 1
    for (int o = warp * U * kBlockElems; o < left; o += kStep) {
      uint32_t cm[U], cv[U], exps = 0;
      const int block0 = o / kBlockElems;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = o + u * kBlockElems + lane * 4;
        const bool there = block0 + u < blocks;
        cm[u] = there ? *reinterpret_cast<const uint32_t*>(pm + i) : 0u;
        cv[u] = there ? *reinterpret_cast<const uint32_t*>(pv + i) : 0u;
      }
      if (lane < 2 * U && block0 + lane % U < blocks) exps = pe[block0];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = o + u * kBlockElems + lane * 4, em = __shfl_sync(0xffffffffu, exps, u), ev = __shfl_sync(0xffffffffu, exps, U + u);
        float m[4], v[4];
        decode<kBitsM>(m, cm[u], em, base_of(em, kBelowM), 1u << 20);
        decode<kBitsV>(v, cv[u], ev, base_of(ev, kBelowV), 1u << 20);
        store4<false>(to_m, m, i, left, vec);
        store4<false>(to_v, v, i, left, vec);
      }
    }
  }
}

// Fills tables of up to CAP tensors and launches for each, a thread block a chunk: in the order of the addresses memory gives 6.7 TB/s (106 million
// float32 with moments in 32 bits in 440 us; 495 by 296 blocks that go on to further chunks). A chunk is a step of a block, or with `steps` up to so
// many where there are enough for all SMs a few times over (moments in 8 bits, bound by operations: 338 us with eight, 370 with one).
template <int CAP, typename Launch>
int in_tables(const flb_adamw_tensor* t, int64_t count, int elem, int state_bits, int steps, Launch&& launch) {
  static_assert(sizeof(Table<CAP>) + sizeof(Args) <= 32 * 1024 - 4, "a launch's parameters");
  Table<CAP> tb;
  auto off = [](const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) != 0; };
  int64_t total = 0;
  for (int64_t i = 0; i < count; ++i) total += t[i].n;
  tb.chunk = kStep;
  while (tb.chunk < steps * kStep && total / tb.chunk > 24 * (int64_t)num_sms()) tb.chunk *= 2;
  for (int64_t from = 0; from < count;) {
    tb.count = 0;
    tb.first[0] = 0;
    while (from < count && tb.count < CAP) {
      const flb_adamw_tensor& s = t[from];
      const int64_t chunks = (s.n + tb.chunk - 1) / tb.chunk;
      if (chunks > 0 && chunks + tb.first[tb.count] > INT32_MAX) break;
      ++from;
      if (chunks == 0 && !s.step) continue;
      const bool vec = !off(s.p, 4 * elem) && !off(s.g, 4 * elem) && (state_bits == 8 || (!off(s.m, 16) && !off(s.v, 16)));
      tb.t[tb.count] = Tensor{s.p, s.g, s.m, s.v, s.m_exps, s.v_exps, s.step, vec ? s.n : -s.n};
      tb.first[tb.count + 1] = tb.first[tb.count] + (uint32_t)chunks;
      ++tb.count;
    }
    if (tb.count == 0) continue;
    const int st = launch(tb, std::max(1u, tb.first[tb.count]));
    if (st != FLB_OK) return st;
  }
  return FLB_OK;
}

template <typename T, int BITS, int CAP> int step_tables(const flb_adamw_tensor* t, int64_t count, const Args& a, cudaStream_t s) {
  return in_tables<CAP>(t, count, sizeof(T), BITS, BITS == 8 ? 8 : 1, [&](const Table<CAP>& tb, unsigned grid) {
    adamw_kernel<T, BITS, CAP><<<grid, kThreads, 0, s>>>(tb, a);
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
  a.lr = lr, a.lr_device = lr_device, a.decay = decay, a.eps = (float)eps, a.flush = eps >= 1e-11, a.seed = seed, a.counter = counter, a.place = 1u << 20;
  switch (dtype) {
    case FLB_F32: return step_b<float>(t, count, state_bits, a, s);
    case FLB_F16: return step_b<__half>(t, count, state_bits, a, s);
    default: return step_b<__nv_bfloat16>(t, count, state_bits, a, s);
  }
}

int adamw_moments(const flb_adamw_tensor* t, int64_t count, cudaStream_t s) {
  return in_tables<440>(t, count, 4, 8, 1, [&](const Table<440>& tb, unsigned grid) {
    if (tb.first[tb.count] == 0) return (int)FLB_OK;
    moments_kernel<440><<<grid, kThreads, 0, s>>>(tb);
    count_launches(1);
    return check_cuda(cudaGetLastError(), "adamw_moments launch");
  });
}

}  // namespace flb
