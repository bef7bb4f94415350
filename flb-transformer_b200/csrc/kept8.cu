// The 8-bit kept form on its own (a tensor into it and back), and the sigmoid gate that keeps its inputs so:
//
//   y = x g,  g = 1 / (1 + exp(-z));   dx = dy g,   dz = dy x g (1 - g), with x and z of the kept form
//
// Bound by memory: every element is read and written once. A warp takes 256 consecutive elements of a row at
// a time, two blocks of the kept form, whose largest magnitudes are a reduction over 16 or 32 lanes. Rows of a
// multiple of 128 elements are whole blocks on end, in every array: they are taken as rows of 256, one chunk
// each, with all sizes known when the kernel is compiled (FLAT). bfloat16 on a B200: 49152 x 2304 kept in 60 us
// and back in 56 (5.6 and 6.1 TB/s), gates of 65536 x 1024 in 91 us forward and 84 backward (5.9 and 6.4 TB/s).
#include <initializer_list>
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

// The warp's chunks, two at a time so that twice the loads are under way; load(row, base, lane) gives what
// finish(row, base, lane, loaded) goes on with, base the chunk's first element in the row.
template <bool FLAT, typename L, typename F> __device__ __forceinline__ void for_chunks(const KeptArgs& a, L&& load, F&& finish) {
  const int lane = threadIdx.x & 31;
  const int64_t n = (int64_t)gridDim.x * (kThreads / 32);
  auto place = [&](int64_t i, int64_t& row, int& base) {
    row = i, base = 0;
    if constexpr (!FLAT) {
      row = a.chunks <= 0xffffffffll ? (uint32_t)i / (uint32_t)a.per_row : i / a.per_row;
      base = (int)(i - row * a.per_row) * 256;
    }
  };
  for (int64_t i = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); i < a.chunks; i += 2 * n) {
    int64_t r0, r1;
    int b0, b1;
    place(i, r0, b0);
    place(i + n, r1, b1);
    const bool two = i + n < a.chunks;
    auto x0 = load(r0, b0, lane);
    decltype(x0) x1;
    if (two) x1 = load(r1, b1, lane);
    finish(r0, b0, lane, x0);
    if (two) finish(r1, b1, lane, x1);
  }
}

template <typename T, Layout L>
__device__ __forceinline__ void keep_raw(const Raw8<T>& r, const F2 (&v)[4], int8_t* codes, uint8_t* exps, int64_t row, int base,
                                         int lane, int D) {
  uint32_t m[L == EIGHT ? 1 : 2];
  max_bits<T, L>(r, m);
  keep8<L>(v, m, codes + row * code_pitch(D), exps + row * blocks_of(D), base, lane, D);
}

// FORM 0: rows that start on 16 bytes, a multiple of 8 wide; 1: others; 2: FLAT
template <typename T, int FORM> constexpr Layout kForm = kLayout<T, FORM != 1>;

template <typename T, int FORM> __global__ void __launch_bounds__(kThreads) pack_kernel(const KeptArgs a) {
  constexpr Layout L = kForm<T, FORM>;
  const int D = FORM == 2 ? 256 : a.D;
  auto load = [&](int64_t row, int base, int lane) {
    Raw8<T> r;
    load_raw<T, L>(r, reinterpret_cast<const T*>(a.x) + row * D, base, lane, D);
    return r;
  };
  for_chunks<FORM == 2>(a, load, [&](int64_t row, int base, int lane, const Raw8<T>& r) {
    F2 v[4];
    to_float<T>(r, v);
    keep_raw<T, L>(r, v, a.cx, a.ex, row, base, lane, D);
  });
}

template <typename T, int FORM> __global__ void __launch_bounds__(kThreads) unpack_kernel(const KeptArgs a) {
  constexpr Layout L = kForm<T, FORM>;
  const int D = FORM == 2 ? 256 : a.D;
  auto load = [&](int64_t row, int base, int lane) {
    return load_kept<L>(a.cx + row * code_pitch(D), a.ex + row * blocks_of(D), base, lane, D);
  };
  for_chunks<FORM == 2>(a, load, [&](int64_t row, int base, int lane, const Kept8& k) {
    F2 v[4];
    kept_to_float<L>(k, v);
    if constexpr (std::is_same<T, __half>::value) {
      // a magnitude near the type's largest can be kept as 65536: back to the largest (a NaN stays one)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = split(v[i]);
        v[i] = f2(fabsf(f.x) > 65504.f ? copysignf(65504.f, f.x) : f.x, fabsf(f.y) > 65504.f ? copysignf(65504.f, f.y) : f.y);
      }
    }
    store8<T, L>(reinterpret_cast<T*>(a.y) + row * D, v, base, lane, D);
  });
}

template <typename T, int FORM, bool KEEP> __global__ void __launch_bounds__(kThreads) gate_fwd_kernel(const KeptArgs a) {
  constexpr Layout L = kForm<T, FORM>;
  const int D = FORM == 2 ? 256 : a.D;
  struct Both {
    Raw8<T> x, z;
  };
  auto load = [&](int64_t row, int base, int lane) {
    Both r;
    load_raw<T, L>(r.x, reinterpret_cast<const T*>(a.x) + row * D, base, lane, D);
    load_raw<T, L>(r.z, reinterpret_cast<const T*>(a.z) + row * D, base, lane, D);
    return r;
  };
  for_chunks<FORM == 2>(a, load, [&](int64_t row, int base, int lane, const Both& r) {
    F2 x[4], z[4];
    to_float<T>(r.x, x);
    to_float<T>(r.z, z);
    if constexpr (KEEP) {
      keep_raw<T, L>(r.x, x, a.cx, a.ex, row, base, lane, D);
      keep_raw<T, L>(r.z, z, a.cz, a.ez, row, base, lane, D);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = split(z[i]);
      x[i] = mul2(x[i], f2(gate_of<T>(f.x).x, gate_of<T>(f.y).x));
    }
    store8<T, L>(reinterpret_cast<T*>(a.y) + row * D, x, base, lane, D);
  });
}

// x, z as in the forward, or their kept form; y takes dx, y2 takes dz
template <typename T, int FORM, bool KEEP>
__global__ void __launch_bounds__(kThreads) gate_bwd_kernel(const KeptArgs a, const void* dy_) {
  constexpr Layout L = kForm<T, FORM>;
  const int D = FORM == 2 ? 256 : a.D;
  struct All {
    Raw8<T> dy, x, z;
    Kept8 kx, kz;
  };
  auto load = [&](int64_t row, int base, int lane) {
    All r;
    load_raw<T, L>(r.dy, reinterpret_cast<const T*>(dy_) + row * D, base, lane, D);
    if constexpr (KEEP) {
      r.kx = load_kept<L>(a.cx + row * code_pitch(D), a.ex + row * blocks_of(D), base, lane, D);
      r.kz = load_kept<L>(a.cz + row * code_pitch(D), a.ez + row * blocks_of(D), base, lane, D);
    } else {
      load_raw<T, L>(r.x, reinterpret_cast<const T*>(a.x) + row * D, base, lane, D);
      load_raw<T, L>(r.z, reinterpret_cast<const T*>(a.z) + row * D, base, lane, D);
    }
    return r;
  };
  for_chunks<FORM == 2>(a, load, [&](int64_t row, int base, int lane, const All& r) {
    F2 x[4], z[4], dy[4], dz[4];
    to_float<T>(r.dy, dy);
    if constexpr (KEEP) {
      kept_to_float<L>(r.kx, x);
      kept_to_float<L>(r.kz, z);
    } else {
      to_float<T>(r.x, x);
      to_float<T>(r.z, z);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = split(z[i]), g = gate_of<T>(f.x), h = gate_of<T>(f.y);
      const F2 dx = mul2(dy[i], f2(g.x, h.x));
      dz[i] = mul2(mul2(dx, x[i]), f2(g.y, h.y));
      x[i] = dx;
    }
    store8<T, L>(reinterpret_cast<T*>(a.y) + row * D, x, base, lane, D);
    store8<T, L>(reinterpret_cast<T*>(a.y2) + row * D, dz, base, lane, D);
  });
}

bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Blocks for all chunks at once, up to 16 a SM; they stride beyond that
unsigned grid_of(int64_t chunks) {
  const int64_t per = kThreads / 32;
  return (unsigned)std::max<int64_t>(1, std::min<int64_t>((chunks + per - 1) / per, (int64_t)num_sms() * 16));
}

template <template <typename, int> class Launch, typename T, typename... A> void by_form(int form, const A&... args) {
  if (form == 2) Launch<T, 2>::run(args...);
  else if (form == 1) Launch<T, 1>::run(args...);
  else Launch<T, 0>::run(args...);
}
template <template <typename, int> class Launch, typename... A> int by_type(int dtype, int form, const A&... args) {
  switch (dtype) {
    case FLB_F32: by_form<Launch, float>(form, args...); break;
    case FLB_F16: by_form<Launch, __half>(form, args...); break;
    default: by_form<Launch, __nv_bfloat16>(form, args...); break;
  }
  count_launches(1);
  return check_cuda(cudaGetLastError(), "8-bit kept form launch");
}

template <typename T, int FORM> struct Pack {
  static void run(const KeptArgs& a, cudaStream_t s) { pack_kernel<T, FORM><<<grid_of(a.chunks), kThreads, 0, s>>>(a); }
};
template <typename T, int FORM> struct Unpack {
  static void run(const KeptArgs& a, cudaStream_t s) { unpack_kernel<T, FORM><<<grid_of(a.chunks), kThreads, 0, s>>>(a); }
};
template <typename T, int FORM> struct GateFwd {
  static void run(const KeptArgs& a, cudaStream_t s) {
    if (a.cx) gate_fwd_kernel<T, FORM, true><<<grid_of(a.chunks), kThreads, 0, s>>>(a);
    else gate_fwd_kernel<T, FORM, false><<<grid_of(a.chunks), kThreads, 0, s>>>(a);
  }
};
template <typename T, int FORM> struct GateBwd {
  static void run(const KeptArgs& a, const void* dy, cudaStream_t s) {
    if (a.cx) gate_bwd_kernel<T, FORM, true><<<grid_of(a.chunks), kThreads, 0, s>>>(a, dy);
    else gate_bwd_kernel<T, FORM, false><<<grid_of(a.chunks), kThreads, 0, s>>>(a, dy);
  }
};

// The chunks of [R, D], and the form that every pointer and the width allow
KeptArgs kept_args(int64_t R, int64_t D, std::initializer_list<const void*> pointers, int* form) {
  KeptArgs a = {};
  *form = D % 8 == 0 ? 0 : 1;
  for (const void* p : pointers)
    if (!on16(p)) *form = 1;
  if (*form == 0 && D % kBlock == 0 && R * D % 256 == 0) {
    *form = 2;
    R = R * D / 256;
    D = 256;
  }
  a.per_row = (D + 255) / 256;
  a.chunks = R * a.per_row;
  a.D = (int)D;
  return a;
}

}  // namespace

int pack8(const void* x, int8_t* codes, uint8_t* exps, int64_t R, int64_t D, int dtype, cudaStream_t s) {
  int form;
  KeptArgs a = kept_args(R, D, {x, codes}, &form);
  a.x = x, a.cx = codes, a.ex = exps;
  return by_type<Pack>(dtype, form, a, s);
}

int unpack8(const int8_t* codes, const uint8_t* exps, void* out, int64_t R, int64_t D, int dtype, cudaStream_t s) {
  int form;
  KeptArgs a = kept_args(R, D, {codes, out}, &form);
  a.cx = const_cast<int8_t*>(codes), a.ex = const_cast<uint8_t*>(exps), a.y = out;
  return by_type<Unpack>(dtype, form, a, s);
}

int gate_fwd(const void* x, const void* z, void* y, int8_t* cx, uint8_t* ex, int8_t* cz, uint8_t* ez, int64_t R,
             int64_t D, int dtype, cudaStream_t s) {
  int form;
  KeptArgs a = kept_args(R, D, {x, z, y, cx, cz}, &form);
  a.x = x, a.z = z, a.y = y, a.cx = cx, a.ex = ex, a.cz = cz, a.ez = ez;
  return by_type<GateFwd>(dtype, form, a, s);
}

int gate_bwd(const void* x, const void* z, const int8_t* cx, const uint8_t* ex, const int8_t* cz, const uint8_t* ez,
             const void* dy, void* dx, void* dz, int64_t R, int64_t D, int dtype, cudaStream_t s) {
  int form;
  KeptArgs a = kept_args(R, D, {x, z, cx, cz, dy, dx, dz}, &form);
  a.x = x, a.z = z, a.y = dx, a.y2 = dz;
  a.cx = const_cast<int8_t*>(cx), a.ex = const_cast<uint8_t*>(ex);
  a.cz = const_cast<int8_t*>(cz), a.ez = const_cast<uint8_t*>(ez);
  return by_type<GateBwd>(dtype, form, a, dy, s);
}

}  // namespace flb
