// A token for each row of logits from one uniform number a row.
//
// With temperature T the weights of a row are w_i = exp((l_i - max l) / T). Kept are the top k tokens (those of larger logits,
// of equal ones those of lower index), of these the shortest run from the top on whose weights sum to p of theirs, and of
// these the ones with w_i >= min_p. The token is the first, in the vocabulary's order, at which the sum of kept weights
// passes u of the whole.
//
// Which token comes depends on sums next to a border: a weight is computed in float64 and held as a 64-bit integer in units of
// 2^-F, F as large as the sum over the vocabulary allows (47 for 32000 tokens, 44 for 262144). Integer sums do not depend on their order.
// A weight w is off by at most 4e-14 w and half a unit, so a few draws fall between a border and the real one: with this arithmetic
// against 113 bits, normal logits of deviation 0.5 to 6 at temperatures from 0.5 to 2, at most 7e-9 of them at 32000 tokens, 1e-6 at
// 131071 and 7e-6 at 262144 (most where one token has nearly all of the weight and the others next to none). (In float32 it
// would be one in 200.)
//
// A row is worked on by a block, or by a cluster of up to eight, which holds its logits in shared memory where they fit. What is kept is
// all up to one token in the order from the largest logit down, equal ones by index: the limit. It is found without sorting:
// a histogram over 2048 equal steps of the logit, 32 or 64 of them a halving of the weight, says in which step the k-th
// token lies, or the one at which the sum passes p; the few logits of that step (or, with a small top_k, all from the top to
// there, and then nothing else is looked at again) go into a list, where each counts those before it. Steps too full for the
// list, or the last one, which is open, go through digits of the logits, as integers of the same order, and of the indices instead.
// Bound by instructions where all logits are weighed (an SM issues in 63% of the cycles of 256 rows with top_p, of which the float64 pipe, with 15
// operations a logit, has 17%; 46% and 27% with min_p over 131071) and by what hides their latency, 1.7 blocks an SM; with few rows by
// barriers, 0.6 us for each of a cluster's: 1 x 32000 bf16 with top_k 50 and top_p 0.95 10.3 us, 256 rows with
// top_p 0.9 56 us, 64 x 131071 float32 with min_p 29 us, which is 1.1 TB/s.
#include <cooperative_groups.h>
#include <cfloat>
#include "rows.cuh"

namespace flb {

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kList = 512;
constexpr int kMostBlocks = 8;
constexpr uint32_t kAll = 0xffffffffu;

struct Args {
  const void* logits;
  int64_t ld;
  const void* u;  // float32, or float64
  bool u64;
  int64_t* token;
  int64_t rows;
  int V, slice;   // slice: of a block, in elements
  int frac;       // F
  // a number a row, or one for all
  const float *temperature, *top_p, *min_p;
  const int64_t* top_k;
  double temperature1, top_p1, min_p1;
  int64_t top_k1;
};

// Float32 as integers of the same order, -0 as +0
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

// Eight 16-bit logits, or four of 32 bits, of 16 bytes as they lie in memory
template <typename T> __device__ __forceinline__ void unpack(float (&v)[16 / sizeof(T)], const uint4& x) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      v[i] = __uint_as_float(w[i]);
    } else {
      const float2 f = rows::unpack2<T>(w[i]);
      v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
  }
}

__device__ __forceinline__ uint64_t shfl_up(uint64_t v, int by) { return __shfl_up_sync(kAll, (unsigned long long)v, by); }
__device__ __forceinline__ uint64_t inclusive(uint64_t v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t w = shfl_up(v, o);
    if (lane >= o) v += w;
  }
  return v;
}
__device__ __forceinline__ uint64_t sum_all(uint64_t v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kAll, (unsigned long long)v, o);
  return v;
}

struct Shared {
  uint32_t lo[kBins], hi[kBins];  // this block's histogram: sums of 64 bits in halves, or counts in lo
  uint64_t scan[32];
  uint64_t warp[32];              // each warp's kept weight
  uint32_t top[kMostBlocks];      // each block's largest key, or the NaN mark
  uint32_t index[kMostBlocks];    // its first index of the row's largest key
  uint64_t before, inside;        // what crossing() found: the sum ahead of a bin, and its own
  uint32_t bin;
  uint32_t listed;                // logits that wanted a place in the list
  uint64_t list[kList];           // distance from the top, and index in the lower half
  uint64_t list_weight[kList];
  float limit_value;
  uint32_t limit_index;
  uint32_t win_block, win_warp;
  uint64_t win_target;
  uint64_t merged[];              // with several blocks a row: the cluster's histogram, [kBins]
};

// What is kept by top_k and top_p: all up to this token, from the largest logit down, equal ones by index
struct Limit {
  float value;  // -inf: all
  uint32_t index;
  __device__ __forceinline__ bool keeps(float v, uint32_t i) const { return v > value || (v == value && i <= index); }
};

template <typename T, bool HELD> struct Row {
  static constexpr int VEC = 16 / (int)sizeof(T);

  Shared& sh;
  uint4* held;             // HELD: the slice's logits, at the places that they have from a 16-byte boundary on
  const T* src;            // the same in memory
  int first, n, shift;     // the slice's first index, and number; how far from 16 bytes the first lies, in elements
  int vectors;
  int rank, blocks;
  int frac;                // F
  float top, none;         // the row's largest logit; up to this one none may be chosen
  float lowest;            // logits below count as this one, whose weight is nothing
  double max_value, per_unit;  // the largest logit; log2(e) / temperature

  __device__ __forceinline__ void meet() {
    if (blocks > 1) cg::this_cluster().sync();
    else __syncthreads();
  }
  template <typename U> __device__ __forceinline__ U* in_block(U* p, int block) { return blocks > 1 ? cg::this_cluster().map_shared_rank(p, block) : p; }

  // exp((l - max) / T) in units of 2^-F. 2^y = 2^n 2^f with n = round(y), and 2^f = 1 + f p(f), p of degree 8 through (2^f - 1) / f at
  // Chebyshev's points of [-1/2, 1/2]: within 4e-14 of the value. 15 float64 operations, of several logits a step of
  // each after the other, since each waits for the one before it.
  template <int N> __device__ __forceinline__ void weigh(const float (&v)[N], uint64_t (&w)[N]) const {
    constexpr double kCoefficients[10] = {1.0,
                                          0x1.62e42fefa39efp-1,
                                          0x1.ebfbdff823cedp-3,
                                          0x1.c6b08d7047e52p-5,
                                          0x1.3b2ab7181b755p-7,
                                          0x1.5d87fe86fe88ep-10,
                                          0x1.4308ac85aa947p-13,
                                          0x1.ffcb9515a8016p-17,
                                          0x1.63d136366db24p-20,
                                          0x1.b63880a30e9ffp-24};
    double f[N], p[N];
    int n[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      // (operations that a compiler does not contract: a logit's weight has to be the same integer wherever it is computed)
      const double y = __dmul_rn(__dadd_rn((double)fminf(fmaxf(v[j], lowest), FLT_MAX), -max_value), per_unit);
      const double t = __dadd_rn(y, 0x1.8p52);
      n[j] = __double2loint(t) + frac;
      f[j] = __dadd_rn(y, -__dadd_rn(t, -0x1.8p52));
      p[j] = kCoefficients[9];
    }
#pragma unroll
    for (int i = 8; i >= 0; --i)
#pragma unroll
      for (int j = 0; j < N; ++j) p[j] = fma(p[j], f[j], kCoefficients[i]);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const double x = __hiloint2double(__double2hiint(p[j]) + (n[j] << 20), __double2loint(p[j]));
      // rounded to an integer by the addition, below 2^52
      w[j] = (uint64_t)__double_as_longlong(__dadd_rn(x, 0x1p52)) & 0xfffffffffffffull;
    }
  }
  __device__ __forceinline__ uint64_t weight(float value) const {
    const float v[1] = {value};
    uint64_t w[1];
    weigh(v, w);
    return w[0];
  }

  // A vector of logits from memory, -inf for places outside the slice.
  __device__ __forceinline__ void fetch(float (&v)[VEC], int at) const {
    const int e = at * VEC - shift;  // its first element
    if (e >= 0 && e + VEC <= n) {
      unpack<T>(v, *reinterpret_cast<const uint4*>(src + e));
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[j] = e + j >= 0 && e + j < n ? ld(src + e + j) : -INFINITY;
    }
  }
  __device__ __forceinline__ void load(float (&v)[VEC], int at) const {
    if constexpr (HELD) unpack<T>(v, held[at]);
    else fetch(v, at);
  }
  __device__ __forceinline__ uint32_t index_of(int at, int j) const { return (uint32_t)(first + at * VEC - shift + j); }
  // f(logit, index) of every logit that may be chosen and for which wanted(logit)
  template <typename W, typename F> __device__ __forceinline__ void each(W&& wanted, F&& f) const {
#pragma unroll 1
    for (int at = threadIdx.x; at < vectors; at += kThreads) {
      float v[VEC];
      load(v, at);
      uint32_t which = 0;
#pragma unroll
      for (int j = 0; j < VEC; ++j) which |= v[j] > none && wanted(v[j]) ? 1u << j : 0u;
      if (which) {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (which >> j & 1) f(v[j], index_of(at, j));
      }
    }
  }
  // The step of a logit below the top: steps of 1 / scale, the last one open. Monotone. (To an integer by an addition: conversions run at an
  // eighth of its rate. The top itself apart, for a scale of infinity.)
  __device__ __forceinline__ uint32_t step_of(float v, float scale) const {
    const float steps = fminf((top - v) * scale, (float)(kBins - 1));
    return v == top ? 0u : __float_as_uint(steps + 0x1p23f) & (kBins - 1);
  }
  // No logit of step `bin` lies below reach(bin + 0.75), nor above reach(bin - 0.75): steps are rounded to the nearest, and the quarter is far above
  // their error. Two comparisons where step_of takes six operations.
  __device__ __forceinline__ float reach(float steps, float scale) const { return top - steps / scale; }

  // ---- histograms ----
  __device__ __forceinline__ void clear() {
    for (int i = threadIdx.x; i < kBins; i += kThreads) sh.lo[i] = 0, sh.hi[i] = 0;
    __syncthreads();
  }
  __device__ __forceinline__ void add(uint32_t bin) { atomicAdd(&sh.lo[bin], 1u); }
  __device__ __forceinline__ void add(uint32_t bin, uint64_t w) {
    const uint32_t lo = (uint32_t)w, old = atomicAdd(&sh.lo[bin], lo), hi = (uint32_t)(w >> 32) + (old + lo < old ? 1u : 0u);
    if (hi) atomicAdd(&sh.hi[bin], hi);
  }
  // The weights of logits for which kept(logit, index), to the bins of bin(logit, index)
  template <typename Kept, typename Bin> __device__ __forceinline__ void add_weights(Kept&& kept, Bin&& bin) {
#pragma unroll 1
    for (int at = threadIdx.x; at < vectors; at += kThreads) {
      float v[VEC];
      load(v, at);
#pragma unroll
      for (int h = 0; h < VEC; h += 4) {
        float part[4];
        uint64_t w[4];
        bool keep[4], any = false;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          part[j] = v[h + j];
          keep[j] = part[j] > none && kept(part[j], index_of(at, h + j));
          any |= keep[j];
        }
        if (!any) continue;
        weigh(part, w);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (keep[j]) add(bin(part[j], index_of(at, h + j)), w[j]);
      }
    }
  }
  // After every thread's additions: the cluster's sums in all its blocks.
  template <bool WEIGHTS> __device__ void merge() {
    meet();
    if (blocks == 1) return;
    // each block adds up a part of the bins and leaves it with all (all reads of one bin under way together)
    const int per = kBins / blocks, from = rank * per;
    for (int i = from + threadIdx.x; i < from + per; i += kThreads) {
      uint64_t v[kMostBlocks], s = 0;
#pragma unroll
      for (int b = 0; b < kMostBlocks; ++b)
        if (b < blocks) v[b] = ((uint64_t)(WEIGHTS ? in_block(sh.hi, b)[i] : 0u) << 32) + in_block(sh.lo, b)[i];
#pragma unroll
      for (int b = 0; b < kMostBlocks; ++b)
        if (b < blocks) s += v[b];
#pragma unroll
      for (int b = 0; b < kMostBlocks; ++b)
        if (b < blocks) in_block(sh.merged, b)[i] = s;
    }
    meet();
  }
  // The first bin at which the sum of bins from the first one on reaches target_of(their total): into sh.bin, before and inside, and true;
  // false if the total does not. U: 32 bits hold the sums of counts.
  template <typename U, typename Target> __device__ bool crossing(Target&& target_of) {
    constexpr int kRun = kBins / kThreads;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, from = threadIdx.x * kRun;
    U own[kRun], mine = 0;
#pragma unroll
    for (int j = 0; j < kRun; ++j) {
      own[j] = blocks > 1 ? (U)sh.merged[from + j] : sizeof(U) == 4 ? (U)sh.lo[from + j] : (U)(((uint64_t)sh.hi[from + j] << 32) + sh.lo[from + j]);
      mine += own[j];
    }
    U incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const U w = __shfl_up_sync(kAll, incl, o);
      if (lane >= o) incl += w;
    }
    if (lane == 31) sh.scan[warp] = incl;
    __syncthreads();
    // each warp adds up the warps' sums: those ahead, and all
    U of_warp = lane < kWarps ? (U)sh.scan[lane] : 0, ahead = lane < warp ? of_warp : 0;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      of_warp += __shfl_xor_sync(kAll, of_warp, o);
      ahead += __shfl_xor_sync(kAll, ahead, o);
    }
    const uint64_t target = target_of((uint64_t)of_warp);
    uint64_t at = (uint64_t)ahead + (uint64_t)(incl - mine);
#pragma unroll
    for (int j = 0; j < kRun; ++j) {
      if (at < target && target <= at + own[j]) sh.bin = from + j, sh.before = at, sh.inside = own[j];
      at += own[j];
    }
    __syncthreads();
    return target <= (uint64_t)of_warp;
  }

  // ---- the list, in the first block ----
  __device__ __forceinline__ void put(float v, uint32_t index) {
    const uint32_t at = atomicAdd(in_block(&sh.listed, 0), 1u);
    if (at < (uint32_t)kList) in_block(sh.list, 0)[at] = (uint64_t)(key_of(top) - key_of(v)) << 32 | index;
  }
  __device__ __forceinline__ float listed_value(int i) const { return value_of(key_of(top) - (uint32_t)(sh.list[i] >> 32)); }
  // For each of n listed tokens, by the threads of the first block: use(is it there, which, how many come before it, their weights). Before: in
  // the order by distance and index, or by index alone.
  template <bool BY_INDEX, typename Use> __device__ __forceinline__ void rank_all(int n, Use&& use) {
    int width = 1;  // places, a power of two; the threads of a place are neighbours and share the others between them
    while (width < n) width *= 2;
    const int share = min(32, kThreads / width), place = threadIdx.x / share, part = threadIdx.x % share;
    uint32_t count = 0;
    uint64_t sum = 0;
    if (place < n) {
      const uint64_t own = sh.list[place];
#pragma unroll 4
      for (int j = part; j < n; j += share) {
        const uint64_t other = sh.list[j], w = sh.list_weight[j];
        if (BY_INDEX ? (uint32_t)other < (uint32_t)own : other < own) ++count, sum += w;
      }
    }
    for (int o = share / 2; o; o >>= 1) {
      count += __shfl_xor_sync(kAll, count, o);
      sum += __shfl_xor_sync(kAll, (unsigned long long)sum, o);
    }
    use(place < n && part == 0, place, count, sum);
  }
  __device__ __forceinline__ void weigh_list(int n) {
    for (int i = threadIdx.x; i < n; i += kThreads) sh.list_weight[i] = weight(listed_value(i));
    __syncthreads();
  }
  __device__ __forceinline__ void set_limit(int i) { sh.limit_value = listed_value(i), sh.limit_index = (uint32_t)sh.list[i]; }
  // The limit that the first block found, to all.
  __device__ __forceinline__ Limit publish() {
    if (blocks > 1) {
      if (rank == 0 && threadIdx.x < blocks && threadIdx.x > 0) {
        *in_block(&sh.limit_value, threadIdx.x) = sh.limit_value;
        *in_block(&sh.limit_index, threadIdx.x) = sh.limit_index;
      }
      meet();
    }
    return {sh.limit_value, sh.limit_index};
  }

  struct Found {
    uint32_t value;
    uint64_t ahead;
  };
  // ---- digits, where the list does not do ----
  // Over the values of those logits that `has` takes, 32 bits by 11, 11 and 10: the least at which their number, or the sum of their
  // weights, reaches target, and what is ahead of it.
  template <bool WEIGHTS, typename Has> static __device__ __noinline__ Found digits(Row r, uint64_t target, Has has) {
    uint32_t prefix = 0;
    uint64_t base = 0;
#pragma unroll 1
    for (int shift = 21, above = 32;;) {
      r.clear();
      auto within = [&](float v, uint32_t i) {
        uint32_t value;
        return has(v, i, value) && (above == 32 || value >> above == prefix);
      };
      auto bin = [&](float v, uint32_t i) {
        uint32_t value;
        has(v, i, value);
        return (value >> shift) & (kBins - 1);
      };
      if constexpr (WEIGHTS) {
        r.add_weights(within, bin);
      } else {
        r.each([](float) { return true; }, [&](float v, uint32_t i) {
          if (within(v, i)) r.add(bin(v, i));
        });
      }
      r.template merge<WEIGHTS>();
      r.template crossing<uint64_t>([&](uint64_t) { return target - base; });
      prefix = above == 32 ? r.sh.bin : (prefix << (above - shift)) | r.sh.bin;
      base += r.sh.before;
      r.meet();  // all have read what they need of this level
      if (shift == 0) break;
      above = shift;
      shift = shift == 21 ? 10 : 0;
    }
    return {prefix, base};
  }
};

__host__ __device__ constexpr int shared_bytes(int blocks) { return (int)(sizeof(Shared) + (blocks > 1 ? kBins * 8 : 0) + 15) / 16 * 16; }

template <typename T, bool HELD> __global__ void __launch_bounds__(kThreads, 2) sample_kernel(const Args a) {
  using R = Row<T, HELD>;
  constexpr int VEC = R::VEC;
  extern __shared__ __align__(16) uint8_t dyn[];
  Shared& sh = *reinterpret_cast<Shared*>(dyn);
  auto cluster = cg::this_cluster();
  const int blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int64_t row = blockIdx.x / blocks;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int first = rank * a.slice, n = max(0, min(a.V - first, a.slice));
  const T* src = reinterpret_cast<const T*>(a.logits) + row * a.ld + first;
  const int shift = (int)(reinterpret_cast<uintptr_t>(src) % 16 / sizeof(T));
  R r{sh, reinterpret_cast<uint4*>(dyn + shared_bytes(blocks)), src, first, n, shift, (n + shift + VEC - 1) / VEC, rank, blocks, a.frac};
  // (the other blocks' shared memory is there once all have come this far)
  if (blocks > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");

  float largest = -INFINITY;
  bool nan = false;
  auto look = [&](const float (&v)[VEC]) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      largest = fmaxf(largest, v[j]);
      nan |= !(v[j] <= INFINITY);
    }
  };
  {
    // whole vectors, four loads under way a thread; the slice's ends apart
    const int from = shift ? 1 : 0, to = (n + shift) / VEC;
    const uint4* const whole = reinterpret_cast<const uint4*>(src - shift);
#pragma unroll 1
    for (int at = from + threadIdx.x; at < to; at += 4 * kThreads) {
      uint4 x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (at + i * kThreads < to) x[i] = whole[at + i * kThreads];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (at + i * kThreads >= to) continue;
        float v[VEC];
        unpack<T>(v, x[i]);
        look(v);
        if (HELD) r.held[at + i * kThreads] = x[i];
      }
    }
    if (threadIdx.x < 2) {
      const int at = threadIdx.x ? r.vectors - 1 : 0;
      if (at >= 0 && at < r.vectors && (at < from || at >= to)) {
        float v[VEC];
        r.fetch(v, at);
        look(v);
        if (HELD) {
          T* const to = reinterpret_cast<T*>(r.held + at);
#pragma unroll
          for (int j = 0; j < VEC; ++j) st(to + j, v[j]);
        }
      }
    }
  }
  for (int i = threadIdx.x; i < kBins; i += kThreads) sh.lo[i] = 0, sh.hi[i] = 0;
  constexpr uint32_t kNan = 0xffffffffu;  // no logit's key
  const uint32_t key = __reduce_max_sync(kAll, nan ? kNan : key_of(largest));
  if (lane == 0) sh.scan[warp] = key;
  if (threadIdx.x == 32) sh.index[rank] = ~0u, sh.listed = 0;
  __syncthreads();
  if (blocks > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  if (warp == 0) {
    const uint32_t k = __reduce_max_sync(kAll, lane < kWarps ? (uint32_t)sh.scan[lane] : 0u);
    if (lane < blocks) *r.in_block(&sh.top[rank], lane) = k;
  }
  r.meet();
  uint32_t top = 0;
#pragma unroll
  for (int b = 0; b < kMostBlocks; ++b)
    if (b < blocks) top = max(top, sh.top[b]);
  // (every block of the cluster takes the same way from here on, and none returns while another may reach into it)
  if (top == kNan || top == key_of(-INFINITY)) {
    if (rank == 0 && threadIdx.x == 0) a.token[row] = -1;
    return;
  }
  r.top = value_of(top);
  // (beside +inf nothing else counts)
  r.none = r.top == INFINITY ? FLT_MAX : -INFINITY;
  const double temperature = a.temperature ? (double)a.temperature[row] : a.temperature1;

  if (!(temperature > 0)) {
    uint32_t at = ~0u;
    r.each([&](float v) { return v == r.top; }, [&](float, uint32_t i) { at = min(at, i); });
    at = __reduce_min_sync(kAll, at);
    if (lane == 0 && at != ~0u) atomicMin(&sh.index[rank], at);
    __syncthreads();
    if (threadIdx.x == 0 && rank) *r.in_block(&sh.index[rank], 0) = sh.index[rank];
    r.meet();
    if (rank == 0 && threadIdx.x == 0) {
      for (int b = 0; b < blocks; ++b) at = min(at, sh.index[b]);
      a.token[row] = at;
    }
    return;
  }

  r.max_value = (double)fminf(r.top, FLT_MAX);
  // (not so steep that y of the logit next to the top's would be below -900: its weight is nothing either way)
  const double apart = exp2((double)max((int)(__float_as_uint(r.top) >> 23 & 255), 1) - 150);
  r.per_unit = fmin(0x1.71547652b82fep+0 / fmax(temperature, 1e-290), 900 / apart);
  r.lowest = fmaxf((float)(r.max_value - 900 / r.per_unit), -FLT_MAX);
  const int64_t top_k = a.top_k ? a.top_k[row] : a.top_k1;
  const double top_p = a.top_p ? (double)a.top_p[row] : a.top_p1, min_p_given = a.min_p ? (double)a.min_p[row] : a.min_p1, min_p = min_p_given >= 1 ? 1.0 : min_p_given;
  const double u = a.u64 ? reinterpret_cast<const double*>(a.u)[row] : (double)reinterpret_cast<const float*>(a.u)[row];
  const uint64_t w_least = min_p > 0 ? (uint64_t)ceil(min_p * (double)(1ull << a.frac)) : 0;
  // top_p: a token is kept while the sum before it is below p of the whole; the first one always
  auto share_of = [&](uint64_t total) {
    const double t = ceil(top_p * (double)total);
    return t >= 1 ? min((uint64_t)t, total) : (uint64_t)1;
  };
  // the sum at which the token comes: it passes u of the whole, so it is at least this
  auto draw_at = [&](uint64_t total) { return min(u > 0 ? (uint64_t)(fmin(u, 1.0) * (double)total) + 1 : (uint64_t)1, total); };

  Limit limit{-INFINITY, ~0u};
  bool cleared = true;  // the histogram
  if (top_k > 0 && top_k < a.V) {
    const float scale = (float)(32 * r.per_unit);
#pragma unroll 1
    for (int at = threadIdx.x; at < r.vectors; at += kThreads) {
      float v[VEC];
      r.load(v, at);
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (v[j] > r.none) r.add(r.step_of(v[j], scale));
    }
    r.template merge<false>();
    cleared = false;
    if (r.template crossing<uint32_t>([&](uint64_t) { return (uint64_t)top_k; })) {
      const uint32_t bin = sh.bin;
      const uint64_t before = sh.before, inside = sh.inside;
      const float least = r.reach(bin + 0.75f, scale), most = bin ? r.reach(bin - 0.75f, scale) : INFINITY;
      if (bin < kBins - 1 && before + inside <= kList) {
        // Few are left: the first block lists and weighs them all.
        r.each([&](float v) { return v >= least; }, [&](float v, uint32_t i) {
          if (r.step_of(v, scale) <= bin) r.put(v, i);
        });
        r.meet();
        if (rank) return;
        const int m = (int)(before + inside);
        r.weigh_list(m);
        uint32_t place = 0, ahead = 0;
        uint64_t sum = 0;
        bool mine = false;
        r.template rank_all<false>(m, [&](bool is, int at, uint32_t count, uint64_t s) { mine = is, place = at, ahead = count, sum = s; });
        // the whole of the top_k: what is ahead of its last, and that one
        if (mine && ahead == (uint32_t)top_k - 1) sh.before = sum + sh.list_weight[place];
        __syncthreads();
        const uint64_t share = top_p < 1 ? share_of(sh.before) : ~0ull, w = mine ? sh.list_weight[place] : 0;
        const bool kept = mine && ahead < (uint32_t)top_k && sum < share && w >= w_least;
        __syncthreads();
        if (mine && !kept) sh.list_weight[place] = 0;
        __syncthreads();
        // in the vocabulary's order
        r.template rank_all<true>(m, [&](bool, int, uint32_t, uint64_t s) { sum = s; });
        uint64_t total = kept ? w : 0;
        total = sum_all(total);
        if (lane == 0) sh.scan[warp] = total;
        __syncthreads();
        total = sum_all(lane < kWarps ? sh.scan[lane] : 0);
        const uint64_t target = draw_at(total);
        if (kept && sum < target && target <= sum + w) a.token[row] = (uint32_t)sh.list[place];
        return;
      }
      if (bin < kBins - 1 && inside <= kList) {
        r.each([&](float v) { return v >= least && v <= most; }, [&](float v, uint32_t i) {
          if (r.step_of(v, scale) == bin) r.put(v, i);
        });
        r.meet();
        if (rank == 0) {
          r.template rank_all<false>((int)inside, [&](bool is, int at, uint32_t count, uint64_t) {
            if (is && before + count == (uint64_t)top_k - 1) r.set_limit(at);
          });
          __syncthreads();
          if (threadIdx.x == 0) sh.listed = 0;
        }
        limit = r.publish();
      } else {
        const auto at = R::template digits<false>(r, top_k, [top](float v, uint32_t, uint32_t& value) {
          value = top - key_of(v);
          return true;
        });
        limit.value = value_of(top - at.value);
        limit.index = R::template digits<false>(r, top_k - at.ahead, [limit](float v, uint32_t i, uint32_t& value) {
          value = i;
          return v == limit.value;
        }).value;
      }
    }
  }
  if (top_p < 1) {
    const float scale = (float)(64 * r.per_unit);
    if (!cleared) {
      __syncthreads();
      r.clear();
    }
    r.add_weights([&](float v, uint32_t i) { return limit.keeps(v, i); }, [&](float v, uint32_t) { return r.step_of(v, scale); });
    r.template merge<true>();
    uint64_t target;
    r.template crossing<uint64_t>([&](uint64_t total) { return target = share_of(total); });
    const uint32_t bin = sh.bin;
    const uint64_t before = sh.before;
    const float least = r.reach(bin + 0.75f, scale), most = bin ? r.reach(bin - 0.75f, scale) : INFINITY;
    if (bin < kBins - 1)
      r.each([&](float v) { return v >= least && v <= most; }, [&](float v, uint32_t i) {
        if (r.step_of(v, scale) == bin && limit.keeps(v, i)) r.put(v, i);
      });
    r.meet();
    const uint32_t listed = *r.in_block(&sh.listed, 0);
    if (bin < kBins - 1 && listed <= (uint32_t)kList) {
      if (rank == 0) {
        r.weigh_list((int)listed);
        r.template rank_all<false>((int)listed, [&](bool is, int at, uint32_t, uint64_t s) {
          // the one that reaches it is the last that is kept
          if (is && before + s < target && target <= before + s + sh.list_weight[at]) r.set_limit(at);
        });
        __syncthreads();
      }
      limit = r.publish();
    } else {
      const Limit all = limit;
      const auto at = R::template digits<true>(r, target, [all, top](float v, uint32_t i, uint32_t& value) {
        value = top - key_of(v);
        return all.keeps(v, i);
      });
      limit.value = value_of(top - at.value);
      const uint64_t w = r.weight(limit.value);
      limit.index = R::template digits<false>(r, (target - at.ahead + w - 1) / w, [limit](float v, uint32_t i, uint32_t& value) {
        value = i;
        return v == limit.value;
      }).value;
    }
  }

  // Sums of each warp's run of the slice. With a limit most logits are not kept: those that are go into a queue of the
  // warp's, in the histogram's place, and are weighed 32 at a time.
  constexpr int kQueue = (int)(sizeof(sh.lo) + sizeof(sh.hi)) / kWarps / 4;
  static_assert(kQueue >= 32 * VEC, "a step's logits");
  float* const queue = reinterpret_cast<float*>(sh.lo) + warp * kQueue;
  auto run_sum = [&](int v0, int v1) {
    uint64_t sum = 0;
    if (limit.value == -INFINITY) {
#pragma unroll 1
      for (int at = v0 + lane; at < v1; at += 32) {
        float v[VEC];
        r.load(v, at);
#pragma unroll
        for (int h = 0; h < VEC; h += 4) {
          const float part[4] = {v[h], v[h + 1], v[h + 2], v[h + 3]};
          uint64_t w[4];
          r.weigh(part, w);
#pragma unroll
          for (int j = 0; j < 4; ++j) sum += part[j] > r.none && w[j] >= w_least ? w[j] : 0;
        }
      }
    } else {
      int queued = 0;
      auto empty = [&]() {
        __syncwarp();
        for (int i = lane; i < queued; i += 32) {
          const uint64_t w = r.weight(queue[i]);
          if (w >= w_least) sum += w;
        }
        __syncwarp();
        queued = 0;
      };
#pragma unroll 1
      for (int at = v0; at < v1; at += 32) {
        float v[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = -INFINITY;
        if (at + lane < v1) r.load(v, at + lane);
        uint32_t which = 0;
#pragma unroll
        for (int j = 0; j < VEC; ++j) which |= v[j] >= limit.value ? 1u << j : 0u;
        if (!__any_sync(kAll, which)) continue;
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (v[j] == limit.value && r.index_of(at + lane, j) > limit.index) which &= ~(1u << j);
        const int own = __popc(which);
        int incl = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int x = __shfl_up_sync(kAll, incl, o);
          if (lane >= o) incl += x;
        }
        const int all = __shfl_sync(kAll, incl, 31);
        if (queued + all > kQueue) empty();
        float* to = queue + queued + incl - own;
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (which >> j & 1) *to++ = v[j];
        queued += all;
      }
      empty();
    }
    return sum_all(sum);
  };
  const int per_warp = (r.vectors + kWarps - 1) / kWarps;
  __syncthreads();  // the histogram has been read
  {
    const int v0 = min(r.vectors, warp * per_warp);
    const uint64_t sum = run_sum(v0, min(r.vectors, v0 + per_warp));
    if (lane == 0) sh.warp[warp] = sum;
  }
  r.meet();
  if (warp == 0) {
    // every block finds the warp at which the sum passes u of the whole: a few warps a lane
    constexpr int kMost = kMostBlocks * kWarps / 32;
    const int all = blocks * kWarps, each = (all + 31) / 32;
    uint64_t part[kMost], mine = 0;
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
      const int w = lane * each + i;
      part[i] = i < each && w < all ? r.in_block(sh.warp, w / kWarps)[w % kWarps] : 0;
      mine += part[i];
    }
    const uint64_t incl = inclusive(mine, lane), target = draw_at(__shfl_sync(kAll, (unsigned long long)incl, 31));
    uint64_t at = incl - mine;
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
      if (at < target && target <= at + part[i]) {
        const int w = lane * each + i;
        sh.win_block = w / kWarps, sh.win_warp = w % kWarps, sh.win_target = target - at;
      }
      at += part[i];
    }
  }
  r.meet();
  if (rank != (int)sh.win_block) return;
  // that warp's run once more: where it is long, first in parts by all warps of its block
  uint64_t target = sh.win_target;
  int v0 = min(r.vectors, (int)sh.win_warp * per_warp), v1 = min(r.vectors, v0 + per_warp);
  if (per_warp > 32) {
    const int part = (per_warp + kWarps - 1) / kWarps, w0 = min(v1, v0 + warp * part), w1 = min(v1, w0 + part);
    const uint64_t sum = run_sum(w0, w1);
    if (lane == 0) sh.scan[warp] = sum;
    __syncthreads();
    const uint64_t its = lane < kWarps ? sh.scan[lane] : 0, at = inclusive(its, lane) - its;
    const uint64_t before = __shfl_sync(kAll, (unsigned long long)at, warp), own = __shfl_sync(kAll, (unsigned long long)its, warp);
    if (!(before < target && target <= before + own)) return;
    target -= before, v0 = w0, v1 = w1;
  } else if (warp != (int)sh.win_warp) {
    return;
  }
#pragma unroll 1
  for (int at = v0; at < v1; at += 32) {
    float v[VEC];
    uint64_t w[VEC], here = 0;
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = -INFINITY;
    if (at + lane < v1) r.load(v, at + lane);
    r.weigh(v, w);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      if (!(v[j] > r.none && limit.keeps(v[j], r.index_of(at + lane, j)) && w[j] >= w_least)) w[j] = 0;
      here += w[j];
    }
    const uint64_t incl = inclusive(here, lane), all = __shfl_sync(kAll, (unsigned long long)incl, 31);
    if (target <= all) {
      uint64_t sum = incl - here;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        if (sum < target && target <= sum + w[j]) a.token[row] = r.index_of(at + lane, j);
        sum += w[j];
      }
      return;
    }
    target -= all;
  }
}

template <typename T, bool HELD> int launch_t(const Args& a, int blocks, cudaStream_t s) {
  const int keys = HELD ? (int)(((size_t)a.slice + 16 / sizeof(T)) * sizeof(T) + 15) / 16 * 16 : 0;
  const int st = ensure_dyn_smem(reinterpret_cast<const void*>(sample_kernel<T, HELD>), 200 * 1024, "sample shared memory");
  if (st != FLB_OK) return st;
  cudaLaunchAttribute attr[1];
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.rows * blocks));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = shared_bytes(blocks) + keys;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, sample_kernel<T, HELD>, a);
  count_launches(1);
  return check_cuda(e, "sample launch");
}

// Blocks a row (us, kernel alone, top_k 50 with top_p 0.95 / top_p 0.9): 1 x 32000 bf16 13.0 / 33 with one, 10.3 / 15.4 with eight; 16 rows of them
// 11.5 / 20.4 with four, 13.7 / 20.0 with eight; 64 rows 13.0 / 27.4 with two, 15.1 / 28.2 with four; 1 x 4096 7.9 / 10.9 with
// one, 10.2 / 14.6 with two; 32 x 131071 float32 23 / 53 with four, 20 / 46 with eight. So: a cluster's barriers want 3600 logits a block
// to pay, blocks want an SM each, clusters of eight half of the SMs left free, but long slices rather two blocks on an SM.
int blocks_for(int64_t rows, int V) {
  const int64_t sms = num_sms();
  int blocks = 1;
  for (int b = 2; b <= kMostBlocks; b *= 2) {
    const int64_t slice = (V + b - 1) / b, most = slice >= 16384 ? 2 * sms : b == 8 ? sms * 7 / 16 : sms;
    if (slice < 3600 || rows * b > most) break;
    blocks = b;
  }
  return blocks;
}

template <typename T> int launch(Args a, cudaStream_t s) {
  const int blocks = blocks_for(a.rows, a.V);
  a.slice = (a.V + blocks - 1) / blocks;
  // held where two blocks fit an SM; else each pass reads the logits from L2
  if ((size_t)a.slice * sizeof(T) <= 64 * 1024) return launch_t<T, true>(a, blocks, s);
  return launch_t<T, false>(a, blocks, s);
}

}  // namespace

int sample(const void* logits, int64_t ld, const void* u, bool u64, int64_t* token, int64_t rows, int64_t V, int dtype, const float* temperature,
           const int64_t* top_k, const float* top_p, const float* min_p, double temperature1, int64_t top_k1, double top_p1, double min_p1,
           cudaStream_t s) {
  int bits = 1;
  while (((int64_t)1 << bits) < V) ++bits;
  Args a = {logits, ld, u, u64, token, rows, (int)V, 0, std::min(50, 62 - bits), temperature, top_p, min_p, top_k, temperature1, top_p1, min_p1, top_k1};
  switch (dtype) {
    case FLB_F32: return launch<float>(a, s);
    case FLB_F16: return launch<__half>(a, s);
    default: return launch<__nv_bfloat16>(a, s);
  }
}

}  // namespace flb
