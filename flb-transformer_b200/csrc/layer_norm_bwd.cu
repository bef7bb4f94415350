// LayerNorm backward. With h the normalised row (from x and the forward's mean and 1/sigma, or from its
// 8-bit kept form), gw = dy w:
//
//   dx = (gw - mean(gw) - h mean(gw h)) / sigma,   dw = sum over rows of dy h,   db = sum over rows of dy
//
// Bound by memory: dy and h are read once, dx is written once. A warp (D <= 512) or block walks over rows
// a fixed distance apart, the next rows on their way to shared memory meanwhile, and adds up dw and db of
// the columns that its threads own in float32 registers. A block's sums go to its own row of a
// workspace, which a second kernel adds up in a fixed order: no atomics, the same bits every time. With
// one block a group (few rows) the block writes dw and db itself. 32768 x 4096 bfloat16: 151 us, 5.3 TB/s, of which
// the second kernel takes 5; what is left is the warps' waits for one another once a row.
#include "rows.cuh"

namespace flb {

using namespace rows;

namespace {

// Floats between two rows of the workspace: each starts on 16 bytes
__host__ __device__ inline int part_pitch(int D) { return (D + 3) & ~3; }

struct BwdArgs {
  const void* x;
  int64_t ldx;
  const int8_t* codes;  // the kept form of h instead of x and mean
  const uint8_t* exps;
  const float *mean, *rstd;
  const void* w;
  bool w32;
  const void* dy;
  void* dx;
  void *dw, *db;  // final gradients (one block a group), w's type
  float* part;    // [G][blocks][2][part_pitch(D)] otherwise
  int64_t R;
  int D;
};

template <typename T> __device__ __forceinline__ void store_param(void* p, bool f32, int64_t i, float v) {
  if (!p) return;
  if (f32) reinterpret_cast<float*>(p)[i] = v; else st(reinterpret_cast<T*>(p) + i, v);
}

// Rows held at a time: three with 16-bit elements, two with float32; in the widest form, whose block is a
// whole SM's, two and one.
template <typename T, bool WIDE> constexpr int kStages = (sizeof(T) == 4 ? 2 : 3) - (WIDE ? 1 : 0);
constexpr int kWarps = 4;  // of a block whose warps have a row each
constexpr int kBlocksPerSm = 4;  // such blocks on an SM

// Bytes a chunk of each of a block's warps takes in the ring: x or codes, then dy
template <typename T, Layout L, bool KEPT> __host__ __device__ constexpr int chunk_bytes(int threads) {
  return copy_bytes<T, L>(threads) + (KEPT ? 8 * threads : copy_bytes<T, L>(threads));
}

// MODE 0: a warp a row (D <= 512), 1: a block a row (D <= 8192), 2: a block of up to 1024 threads (D <= 16384)
template <typename T, bool VEC, int MODE, int CH, bool KEPT>
__global__ void __launch_bounds__(MODE == 0 ? 32 * kWarps : MODE == 1 ? 512 : 1024, MODE == 0 ? kBlocksPerSm : 1)
    ln_bwd_kernel(const BwdArgs a) {
  constexpr Layout L = kLayout<T, VEC>;
  constexpr bool WARP = MODE == 0;
  constexpr int S = kStages<T, MODE == 2>;
  extern __shared__ __align__(16) uint8_t ring[];  // [S][CH][x or codes | dy]; at the end [2][D] floats
  __shared__ __align__(16) float2 slot[WARP ? 1 : 2][32];  // zero for warps that the block does not have
  let_successor_start();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if constexpr (!WARP) {
    if (warp == 0) slot[0][lane] = slot[1][lane] = make_float2(0.f, 0.f);
    __syncthreads();
  }
  const int64_t group = blockIdx.y;
  const int D = a.D;
  const int first = WARP ? 0 : warp * 256 * CH;
  const int64_t stride = WARP ? (int64_t)gridDim.x * kWarps : gridDim.x;
  const int64_t row0 = WARP ? (int64_t)blockIdx.x * kWarps + warp : blockIdx.x;
  const float inv_d = 1.f / D;
  auto part_of = [&](int stage, int c, bool dy) {
    return ring + (size_t)(stage * CH + c) * chunk_bytes<T, L, KEPT>(blockDim.x) +
           (dy ? (KEPT ? 8 * blockDim.x : copy_bytes<T, L>(blockDim.x)) : 0);
  };
  auto dy_row = [&](int64_t r) { return reinterpret_cast<const T*>(a.dy) + (group * a.R + r) * D; };
  auto x_row = [&](int64_t r) { return reinterpret_cast<const T*>(a.x) + (group * a.R + r) * a.ldx; };
  auto code_row = [&](int64_t r) { return a.codes + (group * a.R + r) * code_pitch(D); };
  auto issue = [&](int64_t r, int stage) {
    if (r < a.R) {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int base = first + c * 256;
        copy8<T, L>(part_of(stage, c, true), dy_row(r), base, lane, D);
        if constexpr (KEPT) copy_codes<L>(part_of(stage, c, false), code_row(r), base, lane, D);
        else copy8<T, L>(part_of(stage, c, false), x_row(r), base, lane, D);
      }
    }
    copies_commit();
  };

  F2 dw[CH][4], db[CH][4];
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i) dw[c][i] = db[c][i] = f2(0.f);

  F2 w[CH][4];  // the group's weight
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    if (!a.w) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[c][i] = f2(1.f);
    } else if (a.w32) {
      load8<float, L>(w[c], reinterpret_cast<const float*>(a.w) + group * D, first + c * 256, lane, D);
    } else {
      load8<T, L>(w[c], reinterpret_cast<const T*>(a.w) + group * D, first + c * 256, lane, D);
    }
  }

  // what is not copied: the row's statistics and its blocks' exponents
  float mean = 0.f, rstd = 0.f;
  uint32_t exps[CH];
  auto fetch_small = [&](int64_t r) {
    const int64_t rr = group * a.R + r;
    if constexpr (!KEPT) mean = __ldg(a.mean + rr);
    rstd = __ldg(a.rstd + rr);
    if constexpr (KEPT) {
#pragma unroll
      for (int c = 0; c < CH; ++c) exps[c] = load_exps<L>(a.exps + rr * blocks_of(D), first + c * 256, lane, D);
    }
  };

#pragma unroll
  for (int k = 0; k < S - 1; ++k) issue(row0 + k * stride, k);
  if (row0 < a.R) fetch_small(row0);
  int stage = 0, turn = 0;
  for (int64_t row = row0; row < a.R; row += stride) {
    meet_copies<L>();
    issue(row + (S - 1) * stride, stage == 0 ? S - 1 : stage - 1);  // where the row before this one was
    const float m = mean, rs = rstd;
    uint32_t e[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c)
      if constexpr (KEPT) e[c] = exps[c];
    if (row + stride < a.R) fetch_small(row + stride);
    copies_wait<S - 1>();
    meet_copies<L>();
    // chunk c of x (or the kept h) and dy; read again after the sums, which costs less than the
    // registers to hold them
    auto values = [&](int c, F2 (&x)[4], F2 (&dy)[4]) {
      const int base = first + c * 256;
      copied8<T, L>(part_of(stage, c, true), dy, dy_row(row), base, lane, D);
      if constexpr (KEPT) kept_to_float<L>(Kept8{copied_codes<L>(part_of(stage, c, false), base, lane, D), e[c]}, x);
      else copied8<T, L>(part_of(stage, c, false), x, x_row(row), base, lane, D);
    };
    // h = (x - m) h1, the difference first, as in the forward: exact where x is near the mean. Beyond D, dy and x are zero, and the
    // mean counts as zero too: over a small sigma it can be infinite (a row of 2^110 throughout, eps 1e-12), and 0 h NaN then.
    const float h1 = KEPT ? 1.f : rs;
    F2 t1 = f2(0.f), t2 = f2(0.f);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      F2 x[4], dy[4];
      values(c, x, dy);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const F2 minus = f2(L == SCALARS || Chunk<L>::has(first + c * 256, lane, 2 * i, D) ? -m : 0.f);
        const F2 h = KEPT ? x[i] : mul2(add2(x[i], minus), f2(h1)), gw = mul2(dy[i], w[c][i]);
        dw[c][i] = fma2(dy[i], h, dw[c][i]);
        db[c][i] = add2(db[c][i], dy[i]);
        t1 = add2(t1, gw);
        t2 = fma2(gw, h, t2);
      }
    }
    if constexpr (!KEPT && L == SCALARS) {
      // Scalars have that place element by element, and a choice at each in every row took 45.6 us instead of 41.7 for 16383 x 1001
      // float32 and 139 instead of 118 for 16384 x 4095 bfloat16: the sum again, without those places, where it matters.
      if (isinf(m * h1)) {
        t2 = f2(0.f);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          F2 x[4], dy[4];
          values(c, x, dy);
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = add2(x[i], f2(-m));
          zero_beyond<L>(x, first + c * 256, lane, D);
#pragma unroll
          for (int i = 0; i < 4; ++i) t2 = fma2(mul2(dy[i], w[c][i]), mul2(x[i], f2(h1)), t2);
        }
      }
    }
    float s1 = warp_sum(sum2(t1)), s2 = warp_sum(sum2(t2));
    if constexpr (!WARP) {
      // the slots alternate: a warp that is a row ahead writes the other ones, and is not two ahead
      // before every warp has passed the barrier of the row between, after reading this one's
      if (lane == 0) slot[turn][warp] = make_float2(s1, s2);
      __syncthreads();
      s1 = s2 = 0.f;
      for (int i = 0; i < (int)(blockDim.x >> 5); i += 2) {
        const float4 t = *reinterpret_cast<const float4*>(&slot[turn][i]);
        s1 += t.x + t.z;
        s2 += t.y + t.w;
      }
      turn ^= 1;
    }
    // dx = rs (dy w - s1 - h s2) = rs w dy + (x - m) c1 + c0
    s1 *= inv_d;
    s2 *= inv_d;
    const float c1 = -rs * s2 * h1, c0 = -rs * s1;
    T* dx = reinterpret_cast<T*>(a.dx) + (group * a.R + row) * D;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      F2 x[4], dy[4];
      values(c, x, dy);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        x[i] = fma2(mul2(f2(rs), w[c][i]), dy[i], fma2(KEPT ? x[i] : add2(x[i], f2(-m)), f2(c1), f2(c0)));
      store8<T, L>(dx, x, first + c * 256, lane, D);
    }
    stage = stage + 1 == S ? 0 : stage + 1;
  }

  if (!a.dw && !a.db) return;  // uniform over the grid
  const bool alone = gridDim.x == 1;
  const int pitch = part_pitch(D);
  float* pw = a.part + (group * gridDim.x + blockIdx.x) * 2 * pitch;
  auto out = [&](int p, float vw, float vb) {
    if (alone) {
      store_param<T>(a.dw, a.w32, group * D + p, vw);
      store_param<T>(a.db, a.w32, group * D + p, vb);
    } else {
      pw[p] = vw;
      pw[pitch + p] = vb;
    }
  };
  if constexpr (WARP) {
    copies_wait<0>();  // every copy into the ring has landed before it is used for the sums
    float* sm = reinterpret_cast<float*>(ring);
    for (int t = 0; t < kWarps; ++t) {  // the warps' sums in order
      __syncthreads();
      if (warp != t) continue;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        float vw[8], vb[8];
        to_scalars(dw[c], vw);
        to_scalars(db[c], vb);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int p = Chunk<L>::at(first + c * 256, lane, j);
          if (p < D) {
            sm[p] = (t ? sm[p] : 0.f) + vw[j];
            sm[D + p] = (t ? sm[D + p] : 0.f) + vb[j];
          }
        }
      }
    }
    __syncthreads();
    for (int p = threadIdx.x; p < D; p += blockDim.x) out(p, sm[p], sm[D + p]);
  } else {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float vw[8], vb[8];
      to_scalars(dw[c], vw);
      to_scalars(db[c], vb);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int p = Chunk<L>::at(first + c * 256, lane, j);
        if (p < D) out(p, vw[j], vb[j]);
      }
    }
  }
}

// dw and db from the blocks' sums: 16 columns a block, four a thread, so that a warp reads eight workspace rows
// at a time and every load of a thread can be under way at once. Ordinary loads: the kernel may start beside the one that
// writes the workspace, and the read-only path is for what does not change while a kernel runs.
template <typename T>
__global__ void __launch_bounds__(1024) ln_sum_kernel(const float* part, void* dw, void* db, bool w32,
                                                      int blocks, int D) {
  __shared__ float s[256][17];
  wait_predecessor();
  const int tx = threadIdx.x & 3, ty = threadIdx.x >> 2;
  const int col = blockIdx.x * 16 + tx * 4, which = blockIdx.z, pitch = part_pitch(D);
  const int64_t group = blockIdx.y;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (col < D) {
    const float* p = part + (group * blocks * 2 + which) * pitch + col;
#pragma unroll 8
    for (int i = ty; i < blocks; i += 256) {
      const float4 t = *reinterpret_cast<const float4*>(p + (int64_t)i * 2 * pitch);
      v.x += t.x, v.y += t.y, v.z += t.z, v.w += t.w;
    }
  }
  s[ty][tx * 4] = v.x, s[ty][tx * 4 + 1] = v.y, s[ty][tx * 4 + 2] = v.z, s[ty][tx * 4 + 3] = v.w;
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (warp < 16) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += s[i * 32 + lane][warp];
    sum = warp_sum(sum);
    const int out = blockIdx.x * 16 + warp;
    if (lane == 0 && out < D) store_param<T>(which ? db : dw, w32, group * D + out, sum);
  }
}

// Threads a row, and blocks a group: enough to fill the SMs (512 threads on each), but at least two rows a warp or block, and one block where that leaves it
// four rows a warp at most.
struct BwdShape {
  int mode, threads;
  int64_t blocks;
};
BwdShape bwd_shape(int64_t G, int64_t R, int64_t D) {
  BwdShape p;
  p.mode = D <= 512 ? 0 : D <= 8192 ? 1 : 2;
  p.threads = p.mode == 0 ? 32 * kWarps : 32 * (int)((D + 511) / 512);
  const int64_t at_once = p.mode == 0 ? kWarps : 1;
  const int per_sm = p.mode == 0 ? kBlocksPerSm : std::max(1, 512 / p.threads);
  const int64_t room = std::max<int64_t>(1, (int64_t)num_sms() * per_sm / G);
  p.blocks = R <= 4 * at_once ? 1 : std::min<int64_t>(room, (R + 2 * at_once - 1) / (2 * at_once));
  return p;
}

template <typename T, bool VEC, int MODE, int CH, bool KEPT>
int launch_mode(const BwdArgs& a, const BwdShape& p, int64_t G, cudaStream_t s) {
  auto k = ln_bwd_kernel<T, VEC, MODE, CH, KEPT>;
  const size_t ring = (size_t)kStages<T, MODE == 2> * CH * chunk_bytes<T, kLayout<T, VEC>, KEPT>(p.threads);
  const size_t smem = std::max(ring, MODE == 0 ? (size_t)2 * a.D * sizeof(float) : (size_t)0);
  const int st = ensure_dyn_smem(reinterpret_cast<const void*>(k), (int)smem, "layer_norm_bwd shared memory");
  if (st != FLB_OK) return st;
  k<<<dim3((unsigned)p.blocks, (unsigned)G), p.threads, smem, s>>>(a);
  return FLB_OK;
}

template <typename T, bool VEC, bool KEPT>
int launch_bwd(const BwdArgs& a, int64_t G, cudaStream_t s) {
  const int D = a.D;
  const BwdShape p = bwd_shape(G, a.R, D);
  int st;
  if (p.mode == 0) {
    st = D <= 256 ? launch_mode<T, VEC, 0, 1, KEPT>(a, p, G, s) : launch_mode<T, VEC, 0, 2, KEPT>(a, p, G, s);
  } else if (p.mode == 1) {
    st = launch_mode<T, VEC, 1, 2, KEPT>(a, p, G, s);
  } else {
    st = launch_mode<T, VEC, 2, 2, KEPT>(a, p, G, s);
  }
  if (st != FLB_OK) return st;
  count_launches(1);
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess && p.blocks > 1 && (a.dw || a.db)) {
    e = launch_dependent(ln_sum_kernel<T>, dim3((unsigned)((D + 15) / 16), (unsigned)G, 2), dim3(1024), 0, s,
                         (const float*)a.part, a.dw, a.db, a.w32, (int)p.blocks, D);
    count_launches(1);
  }
  return check_cuda(e, "layer_norm_bwd launch");
}

bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <typename T> int dispatch_bwd(const BwdArgs& a, int64_t G, cudaStream_t s) {
  const bool vec = a.D % 8 == 0 && on16(a.x) && a.ldx * sizeof(T) % 16 == 0 && on16(a.codes) && on16(a.w) && on16(a.dy) && on16(a.dx);
  if (a.codes) return vec ? launch_bwd<T, true, true>(a, G, s) : launch_bwd<T, false, true>(a, G, s);
  return vec ? launch_bwd<T, true, false>(a, G, s) : launch_bwd<T, false, false>(a, G, s);
}

}  // namespace

size_t layer_norm_bwd_workspace_bytes(int64_t G, int64_t R, int64_t D) {
  const BwdShape p = bwd_shape(G, R, D);
  return p.blocks > 1 ? (size_t)G * p.blocks * 2 * part_pitch((int)D) * sizeof(float) : 0;
}

int layer_norm_bwd(const void* x, int64_t ldx, const int8_t* codes, const uint8_t* exps, const float* mean,
                   const float* rstd, const void* w, int wdtype, const void* dy, void* dx, void* dw, void* db, int64_t G,
                   int64_t R, int64_t D, int dtype, void* ws, cudaStream_t s) {
  const BwdArgs a{x, ldx, codes, exps, mean, rstd, w, wdtype == FLB_F32, dy, dx, dw, db, reinterpret_cast<float*>(ws), R, (int)D};
  switch (dtype) {
    case FLB_F32: return dispatch_bwd<float>(a, G, s);
    case FLB_F16: return dispatch_bwd<__half>(a, G, s);
    default: return dispatch_bwd<__nv_bfloat16>(a, G, s);
  }
}

}  // namespace flb
