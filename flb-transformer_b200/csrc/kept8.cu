// The 8-bit kept form on its own (a tensor into it and back), and the sigmoid gate that keeps its inputs so:
//
//   y = x g,  g = 1 / (1 + exp(-z));   dx = dy g,   dz = dy x g (1 - g), with x and z of the kept form
//
// Bound by memory: every element is read and written once. A warp takes 256 consecutive elements of a row at
// a time, two blocks of the kept form, whose largest magnitudes are a reduction over 16 lanes (32 where rows
// do not start on 16 bytes).
#include <type_traits>
#include "rows.cuh"

namespace flb {

using namespace rows;

namespace {

constexpr int kThreads = 256;

struct KeptArgs {
  const void *x, *z;   // inputs, contiguous [rows, D]
  void *y, *y2;        // outputs
  int8_t *cx, *cz;     // codes
  uint8_t *ex, *ez;
  int64_t chunks;      // rows * chunks a row
  int64_t per_row;     // chunks a row
  int D;
};

// g = sigmoid(z) and 1 - g, from exp(-|z|) so that neither overflows nor cancels. 16-bit outputs hold 11
// bits at most: the fast exponential and division (errors near 2^-21) do for them.
template <typename T> __device__ __forceinline__ float2 gate_of(float z) {
  const float e = sizeof(T) == 4 ? expf(-fabsf(z)) : __expf(-fabsf(z));
  const float r = sizeof(T) == 4 ? 1.f / (1.f + e) : __fdividef(1.f, 1.f + e);
  return z >= 0.f ? make_float2(r, e * r) : make_float2(e * r, r);
}

// The warp's chunks, one after the other; the body gets the row, the chunk's first element and the lane.
template <typename F> __device__ __forceinline__ void for_chunks(const KeptArgs& a, F&& body) {
  const int lane = threadIdx.x & 31;
  const int64_t n = (int64_t)gridDim.x * (kThreads / 32);
  for (int64_t i = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); i < a.chunks; i += n) {
    const int64_t row = a.per_row == 1 ? i : a.chunks <= 0xffffffffll ? (uint32_t)i / (uint32_t)a.per_row : i / a.per_row;
    body(row, (int)(i - row * a.per_row) * 256, lane);
  }
}

template <typename T, bool VEC> __global__ void __launch_bounds__(kThreads) pack_kernel(const KeptArgs a) {
  const int D = a.D;
  for_chunks(a, [&](int64_t row, int base, int lane) {
    float v[8];
    load8<T, VEC>(v, reinterpret_cast<const T*>(a.x) + row * D, base, lane, D);
    keep8<VEC>(v, a.cx + row * code_pitch(D), a.ex + row * blocks_of(D), base, lane, D);
  });
}

template <typename T, bool VEC> __global__ void __launch_bounds__(kThreads) unpack_kernel(const KeptArgs a) {
  const int D = a.D;
  for_chunks(a, [&](int64_t row, int base, int lane) {
    float v[8];
    kept_to_float<VEC>(load_kept<VEC>(a.cx + row * code_pitch(D), a.ex + row * blocks_of(D), base, lane, D), v);
    if constexpr (std::is_same<T, __half>::value) {
      // a magnitude near the type's largest can be kept as 65536: back to the largest (a NaN stays one)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = fabsf(v[j]) > 65504.f ? copysignf(65504.f, v[j]) : v[j];
    }
    store8<T, VEC>(reinterpret_cast<T*>(a.y) + row * D, v, base, lane, D);
  });
}

template <typename T, bool VEC, bool KEEP> __global__ void __launch_bounds__(kThreads) gate_fwd_kernel(const KeptArgs a) {
  const int D = a.D;
  for_chunks(a, [&](int64_t row, int base, int lane) {
    float x[8], z[8];
    load8<T, VEC>(x, reinterpret_cast<const T*>(a.x) + row * D, base, lane, D);
    load8<T, VEC>(z, reinterpret_cast<const T*>(a.z) + row * D, base, lane, D);
    if constexpr (KEEP) {
      keep8<VEC>(x, a.cx + row * code_pitch(D), a.ex + row * blocks_of(D), base, lane, D);
      keep8<VEC>(z, a.cz + row * code_pitch(D), a.ez + row * blocks_of(D), base, lane, D);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] *= gate_of<T>(z[j]).x;
    store8<T, VEC>(reinterpret_cast<T*>(a.y) + row * D, x, base, lane, D);
  });
}

// x, z as in the forward, or their kept form; y takes dx, y2 takes dz
template <typename T, bool VEC, bool KEEP>
__global__ void __launch_bounds__(kThreads) gate_bwd_kernel(const KeptArgs a, const void* dy_) {
  const int D = a.D;
  for_chunks(a, [&](int64_t row, int base, int lane) {
    float x[8], z[8], dy[8], dz[8];
    load8<T, VEC>(dy, reinterpret_cast<const T*>(dy_) + row * D, base, lane, D);
    if constexpr (KEEP) {
      const Kept8 kx = load_kept<VEC>(a.cx + row * code_pitch(D), a.ex + row * blocks_of(D), base, lane, D);
      const Kept8 kz = load_kept<VEC>(a.cz + row * code_pitch(D), a.ez + row * blocks_of(D), base, lane, D);
      kept_to_float<VEC>(kx, x);
      kept_to_float<VEC>(kz, z);
    } else {
      load8<T, VEC>(x, reinterpret_cast<const T*>(a.x) + row * D, base, lane, D);
      load8<T, VEC>(z, reinterpret_cast<const T*>(a.z) + row * D, base, lane, D);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 g = gate_of<T>(z[j]);
      const float dx = dy[j] * g.x;
      dz[j] = dx * x[j] * g.y;
      x[j] = dx;
    }
    store8<T, VEC>(reinterpret_cast<T*>(a.y) + row * D, x, base, lane, D);
    store8<T, VEC>(reinterpret_cast<T*>(a.y2) + row * D, dz, base, lane, D);
  });
}

bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Blocks for all chunks at once, up to 16 a SM; they stride beyond that
unsigned grid_of(int64_t chunks) {
  const int64_t per = kThreads / 32;
  return (unsigned)std::max<int64_t>(1, std::min<int64_t>((chunks + per - 1) / per, (int64_t)num_sms() * 16));
}

template <template <typename, bool> class Launch, typename... A>
int by_type(int dtype, bool vec, const A&... args) {
  switch (dtype) {
    case FLB_F32: vec ? Launch<float, true>::run(args...) : Launch<float, false>::run(args...); break;
    case FLB_F16: vec ? Launch<__half, true>::run(args...) : Launch<__half, false>::run(args...); break;
    default: vec ? Launch<__nv_bfloat16, true>::run(args...) : Launch<__nv_bfloat16, false>::run(args...); break;
  }
  count_launches(1);
  return check_cuda(cudaGetLastError(), "8-bit kept form launch");
}

template <typename T, bool VEC> struct Pack {
  static void run(const KeptArgs& a, cudaStream_t s) { pack_kernel<T, VEC><<<grid_of(a.chunks), kThreads, 0, s>>>(a); }
};
template <typename T, bool VEC> struct Unpack {
  static void run(const KeptArgs& a, cudaStream_t s) { unpack_kernel<T, VEC><<<grid_of(a.chunks), kThreads, 0, s>>>(a); }
};
template <typename T, bool VEC> struct GateFwd {
  static void run(const KeptArgs& a, cudaStream_t s) {
    if (a.cx) gate_fwd_kernel<T, VEC, true><<<grid_of(a.chunks), kThreads, 0, s>>>(a);
    else gate_fwd_kernel<T, VEC, false><<<grid_of(a.chunks), kThreads, 0, s>>>(a);
  }
};
template <typename T, bool VEC> struct GateBwd {
  static void run(const KeptArgs& a, const void* dy, cudaStream_t s) {
    if (a.cx) gate_bwd_kernel<T, VEC, true><<<grid_of(a.chunks), kThreads, 0, s>>>(a, dy);
    else gate_bwd_kernel<T, VEC, false><<<grid_of(a.chunks), kThreads, 0, s>>>(a, dy);
  }
};

KeptArgs kept_args(int64_t R, int64_t D) {
  KeptArgs a = {};
  a.per_row = (D + 255) / 256;
  a.chunks = R * a.per_row;
  a.D = (int)D;
  return a;
}

}  // namespace

int pack8(const void* x, int8_t* codes, uint8_t* exps, int64_t R, int64_t D, int dtype, cudaStream_t s) {
  KeptArgs a = kept_args(R, D);
  a.x = x, a.cx = codes, a.ex = exps;
  return by_type<Pack>(dtype, D % 8 == 0 && on16(x) && on16(codes), a, s);
}

int unpack8(const int8_t* codes, const uint8_t* exps, void* out, int64_t R, int64_t D, int dtype, cudaStream_t s) {
  KeptArgs a = kept_args(R, D);
  a.cx = const_cast<int8_t*>(codes), a.ex = const_cast<uint8_t*>(exps), a.y = out;
  return by_type<Unpack>(dtype, D % 8 == 0 && on16(out) && on16(codes), a, s);
}

int gate_fwd(const void* x, const void* z, void* y, int8_t* cx, uint8_t* ex, int8_t* cz, uint8_t* ez, int64_t R,
             int64_t D, int dtype, cudaStream_t s) {
  KeptArgs a = kept_args(R, D);
  a.x = x, a.z = z, a.y = y, a.cx = cx, a.ex = ex, a.cz = cz, a.ez = ez;
  return by_type<GateFwd>(dtype, D % 8 == 0 && on16(x) && on16(z) && on16(y) && on16(cx) && on16(cz), a, s);
}

int gate_bwd(const void* x, const void* z, const int8_t* cx, const uint8_t* ex, const int8_t* cz, const uint8_t* ez,
             const void* dy, void* dx, void* dz, int64_t R, int64_t D, int dtype, cudaStream_t s) {
  KeptArgs a = kept_args(R, D);
  a.x = x, a.z = z, a.y = dx, a.y2 = dz;
  a.cx = const_cast<int8_t*>(cx), a.ex = const_cast<uint8_t*>(ex);
  a.cz = const_cast<int8_t*>(cz), a.ez = const_cast<uint8_t*>(ez);
  return by_type<GateBwd>(dtype, D % 8 == 0 && on16(x) && on16(z) && on16(cx) && on16(cz) && on16(dy) && on16(dx) && on16(dz),
                          a, dy, s);
}

}  // namespace flb
