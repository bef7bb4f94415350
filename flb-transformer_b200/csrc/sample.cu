// A token for each row of logits from one uniform number a row.
//
// With temperature T the weights of a row are w_i = exp((l_i - max l) / T). Kept are the top k tokens (those of larger logits,
// of equal ones those of lower index), of these the shortest run from the top on whose weights sum to p of theirs, and of
// these the ones with w_i >= min_p. The token is the first, in the vocabulary's order, at which the sum of kept weights
// passes u of the whole.
//
// Which token comes depends on sums next to a border, so they are exact: a weight is computed in float64 and held
// as a 64-bit integer in units of 2^-F, F as large as the sum over the vocabulary allows (47 for 32000 tokens). Integer
// sums do not depend on their order, and differ from the real ones by 2^-48 a token: one draw in 10^7 falls in between.
// (In float32 it would be one in 200.)
//
// A row is held as ordered keys (integers that compare as the logits do) in the shared memory of a block, or of a cluster's up to
// eight, so that logits are read once. The k-th largest key and the one at which the sum passes p are found by
// histograms over the distance from the largest key: 2048 bins, then 2048 or 32 within the bin where it lies. No sort.
// Bound by the arithmetic of the weights, a float64 exponential a token, and by barriers where rows are few.
#include <cooperative_groups.h>
#include "rows.cuh"

namespace flb {

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2048;
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

// Logits as integers of the same order, -0 as +0. Nothing below or at kNone can be chosen: -inf, and 0 for places without a logit.
template <typename T> struct Key;
template <> struct Key<float> {
  using type = uint32_t;
  static constexpr uint32_t kNone = 0x007fffffu, kInf = 0xff800000u;
  static constexpr int kLevels = 3;
  static __device__ __forceinline__ uint32_t of(uint32_t b, bool& nan) {
    nan |= (b & 0x7fffffffu) > 0x7f800000u;
    if (b == 0x80000000u) b = 0;
    return b & 0x80000000u ? ~b : b | 0x80000000u;
  }
  static __device__ __forceinline__ float value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
};
template <uint32_t INF> struct Key16 {
  using type = uint16_t;
  static constexpr uint32_t kNone = 0x7fffu - INF, kInf = 0x8000u | INF;
  static constexpr int kLevels = 2;
  static __device__ __forceinline__ uint32_t of(uint32_t b, bool& nan) {
    nan |= (b & 0x7fffu) > INF;
    if (b == 0x8000u) b = 0;
    return b & 0x8000u ? ~b & 0xffffu : b | 0x8000u;
  }
  static __device__ __forceinline__ uint32_t bits(uint32_t k) { return k & 0x8000u ? k ^ 0x8000u : ~k & 0xffffu; }
};
template <> struct Key<__nv_bfloat16> : Key16<0x7f80u> {
  static __device__ __forceinline__ float value(uint32_t k) { return __uint_as_float(bits(k) << 16); }
};
template <> struct Key<__half> : Key16<0x7c00u> {
  static __device__ __forceinline__ float value(uint32_t k) { return __half2float(__ushort_as_half((unsigned short)bits(k))); }
};
// The digit of a distance at a level, and the number of bins there
template <int LEVELS> __device__ __forceinline__ int shift_of(int level) { return LEVELS == 2 ? (level ? 0 : 5) : level == 0 ? 21 : level == 1 ? 10 : 0; }
template <int LEVELS> __device__ __forceinline__ int bins_of(int level) { return LEVELS == 2 ? (level ? 32 : kBins) : level == 2 ? 1024 : kBins; }

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

struct WarpSum {
  uint64_t above;  // weights over the threshold
  uint64_t equal;  // logits at it
};

struct Shared {
  uint32_t lo[kBins], hi[kBins];        // this block's histogram: sums of 64 bits in halves, or counts in lo
  uint64_t merged[kBins];               // the cluster's
  uint64_t scan[kWarps];
  WarpSum warp[kWarps];
  uint32_t top[kMostBlocks];            // each block's largest key, or the NaN mark
  uint32_t index[kMostBlocks];          // its first index of the row's largest key
  uint64_t found_before, found_total;
  uint32_t found_bin;
  uint32_t win_block, win_warp;
  uint64_t win_target, win_equal;
};

template <typename T> struct Row {
  using K = Key<T>;
  using KeyT = typename K::type;
  static constexpr int VEC = 16 / (int)sizeof(T);

  const Args& a;
  Shared& sh;
  KeyT* keys;
  int vectors;             // of this block's slice
  int rank, blocks;
  uint32_t top;            // the row's largest key
  double max_value, inverse, unit;
  bool infinite;

  __device__ __forceinline__ void meet() {
    if (blocks > 1) cg::this_cluster().sync();
    else __syncthreads();
  }
  template <typename U> __device__ __forceinline__ U* in_block(U* p, int block) { return blocks > 1 ? cg::this_cluster().map_shared_rank(p, block) : p; }

  __device__ __forceinline__ double real_weight(uint32_t key) const {
    if (infinite) return key == top ? 1.0 : 0.0;
    return exp(((double)K::value(key) - max_value) * inverse);
  }
  __device__ __forceinline__ uint64_t fixed(double w) const {
    // rounded to an integer by the addition, below 2^52
    return (uint64_t)__double_as_longlong(fma(w, unit, 0x1p52)) & 0xfffffffffffffull;
  }
  __device__ __forceinline__ void load(uint32_t (&k)[VEC], int vector) const {
    const uint4 v = reinterpret_cast<const uint4*>(keys)[vector];
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < VEC; ++j) k[j] = sizeof(T) == 4 ? w[j & 3] : (w[j / 2] >> (16 * (j & 1))) & 0xffffu;
  }

  // Among keys above kNone at distance d from the top, with d < limit, and `extra` more of distance limit: the least distance at
  // which the number of them (or the sum of their weights) reaches `target`, of which target(total) is a function. Returns
  // false if the total does not. before: the sum over smaller distances.
  template <bool WEIGHTS, typename Target>
  __device__ bool select(uint32_t limit, uint64_t extra, Target&& target_of, uint32_t& distance, uint64_t& before) {
    uint32_t prefix = 0;
    uint64_t base = 0, target = 0;
#pragma unroll 1
    for (int level = 0; level < K::kLevels; ++level) {
      const int shift = shift_of<K::kLevels>(level), bins = bins_of<K::kLevels>(level);
      const int above = level == 0 ? 32 : shift_of<K::kLevels>(level - 1);
      for (int i = threadIdx.x; i < bins; i += kThreads) sh.lo[i] = 0, sh.hi[i] = 0;
      __syncthreads();
      auto add = [&](uint32_t d, uint64_t w) {
        const uint32_t b = (d >> shift) & (bins - 1);
        if constexpr (WEIGHTS) {
          const uint32_t lo = (uint32_t)w, old = atomicAdd(&sh.lo[b], lo), carry = old + lo < old ? 1u : 0u;
          const uint32_t hi = (uint32_t)(w >> 32) + carry;
          if (hi) atomicAdd(&sh.hi[b], hi);
        } else {
          atomicAdd(&sh.lo[b], (uint32_t)w);
        }
      };
      auto in_prefix = [&](uint32_t d) { return above == 32 || d >> above == prefix; };
      for (int v = threadIdx.x; v < vectors; v += kThreads) {
        uint32_t k[VEC];
        load(k, v);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const uint32_t d = top - k[j];
          if (k[j] > K::kNone && d < limit && in_prefix(d)) add(d, WEIGHTS ? fixed(real_weight(k[j])) : 1);
        }
      }
      if (extra && rank == 0 && threadIdx.x == 0 && in_prefix(limit)) add(limit, WEIGHTS ? extra * fixed(real_weight(top - limit)) : extra);
      meet();
      // the cluster's sums: each block adds up a part of the bins and leaves it with all
      const int per = bins / blocks, first = rank * per;
      for (int i = first + threadIdx.x; i < first + per; i += kThreads) {
        uint64_t s = 0;
        for (int b = 0; b < blocks; ++b) s += ((uint64_t)in_block(sh.hi, b)[i] << 32) + in_block(sh.lo, b)[i];
        for (int b = 0; b < blocks; ++b) in_block(sh.merged, b)[i] = s;
      }
      meet();
      // where it is reached: a run of bins a thread
      constexpr int kRun = kBins / kThreads;
      const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, from = threadIdx.x * kRun;
      uint64_t mine = 0;
#pragma unroll
      for (int j = 0; j < kRun; ++j)
        if (from + j < bins) mine += sh.merged[from + j];
      const uint64_t incl = inclusive(mine, lane);
      if (lane == 31) sh.scan[warp] = incl;
      __syncthreads();
      uint64_t ahead = base, total = base;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) {
        if (i < warp) ahead += sh.scan[i];
        total += sh.scan[i];
      }
      if (level == 0) {
        target = target_of(total);
        if (total < target) {
          __syncthreads();
          return false;
        }
      }
      uint64_t at = ahead + incl - mine;
#pragma unroll
      for (int j = 0; j < kRun; ++j) {
        if (from + j < bins) {
          const uint64_t next = at + sh.merged[from + j];
          if (at < target && target <= next) sh.found_bin = from + j, sh.found_before = at;
          at = next;
        }
      }
      __syncthreads();
      prefix = level == 0 ? sh.found_bin : (prefix << (above - shift)) | sh.found_bin;
      base = sh.found_before;
      __syncthreads();
    }
    distance = prefix, before = base;
    return true;
  }
};

template <typename T> __global__ void __launch_bounds__(kThreads, 2) sample_kernel(const Args a) {
  using R = Row<T>;
  using K = Key<T>;
  extern __shared__ __align__(16) uint8_t dyn[];
  Shared& sh = *reinterpret_cast<Shared*>(dyn);
  auto cluster = cg::this_cluster();
  const int blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int64_t row = blockIdx.x / blocks;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int first = rank * a.slice, n = max(0, min(a.V - first, a.slice));
  R r{a, sh, reinterpret_cast<typename K::type*>(dyn + (sizeof(Shared) + 15) / 16 * 16), 0, rank, blocks};

  // (the other blocks' shared memory is there once all have come this far)
  if (blocks > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");

  // The slice's keys, at the places that its logits have from a 16-byte boundary on
  const T* src = reinterpret_cast<const T*>(a.logits) + row * a.ld + first;
  const int shift = (int)(reinterpret_cast<uintptr_t>(src) % 16 / sizeof(T));
  r.vectors = (n + shift + R::VEC - 1) / R::VEC;
  uint32_t largest = 0;
  bool nan = false;
  for (int v = threadIdx.x; v < r.vectors; v += kThreads) {
    const int e = v * R::VEC - shift;  // the vector's first element
    uint32_t k[R::VEC];
    if (e >= 0 && e + R::VEC <= n) {
      const uint4 w4 = *reinterpret_cast<const uint4*>(src + e);
      const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
      for (int j = 0; j < R::VEC; ++j) k[j] = K::of(sizeof(T) == 4 ? w[j & 3] : (w[j / 2] >> (16 * (j & 1))) & 0xffffu, nan);
    } else {
#pragma unroll
      for (int j = 0; j < R::VEC; ++j)
        k[j] = e + j >= 0 && e + j < n ? K::of(reinterpret_cast<const typename K::type*>(src)[e + j], nan) : 0u;
    }
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < R::VEC; ++j) {
      largest = max(largest, k[j]);
      if (sizeof(T) == 4) w[j & 3] = k[j];
      else w[j / 2] = j & 1 ? w[j / 2] | k[j] << 16 : k[j];
    }
    reinterpret_cast<uint4*>(r.keys)[v] = make_uint4(w[0], w[1], w[2], w[3]);
  }
  constexpr uint32_t kNan = 0xffffffffu;  // no key: a float32 key of this value is a NaN's
  if (nan) largest = kNan;
  largest = __reduce_max_sync(kAll, largest);
  if (lane == 0) sh.scan[warp] = largest;
  __syncthreads();
  if (blocks > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  if (threadIdx.x < 32) {
    uint32_t v = lane < kWarps ? (uint32_t)sh.scan[lane] : 0u;
    v = __reduce_max_sync(kAll, v);
    if (lane < blocks) *r.in_block(&sh.top[rank], lane) = v;
  }
  if (threadIdx.x == 32) sh.index[rank] = ~0u;
  r.meet();
  uint32_t top = 0;
  for (int b = 0; b < blocks; ++b) top = max(top, sh.top[b]);
  // (every block of the cluster takes the same way from here on, and none returns while another may reach into it)
  if (top == kNan || top <= K::kNone) {
    if (rank == 0 && threadIdx.x == 0) a.token[row] = -1;
    r.meet();
    return;
  }
  r.top = top;
  const double temperature = a.temperature ? (double)a.temperature[row] : a.temperature1;

  if (!(temperature > 0)) {
    uint32_t at = ~0u;
    for (int v = threadIdx.x; v < r.vectors; v += kThreads) {
      uint32_t k[R::VEC];
      r.load(k, v);
#pragma unroll
      for (int j = R::VEC - 1; j >= 0; --j)
        if (k[j] == top) at = min(at, (uint32_t)(first + v * R::VEC - shift + j));
    }
    at = __reduce_min_sync(kAll, at);
    if (lane == 0 && at != ~0u) atomicMin(&sh.index[rank], at);
    __syncthreads();
    if (threadIdx.x == 0 && rank) *r.in_block(&sh.index[rank], 0) = sh.index[rank];
    r.meet();
    if (rank == 0 && threadIdx.x == 0) {
      for (int b = 1; b < blocks; ++b) at = min(at, sh.index[b]);
      a.token[row] = min(at, sh.index[0]);
    }
    return;
  }

  r.max_value = (double)K::value(top);
  r.infinite = top == K::kInf;
  r.inverse = 1.0 / fmax(temperature, 1e-300);
  r.unit = (double)(1ull << a.frac);

  // The threshold: distances below it are kept, and the first `at_most` of those at it
  uint32_t limit = ~0u;
  uint64_t at_most = 0;
  const int64_t top_k = a.top_k ? a.top_k[row] : a.top_k1;
  const double top_p = a.top_p ? (double)a.top_p[row] : a.top_p1, min_p = fmin(a.min_p ? (double)a.min_p[row] : a.min_p1, 1.0);
  if (top_k > 0 && top_k < a.V) {
    uint32_t d;
    uint64_t before;
    if (r.template select<false>(limit, 0, [&](uint64_t) { return (uint64_t)top_k; }, d, before)) limit = d, at_most = top_k - before;
  }
  if (top_p < 1) {
    uint32_t d;
    uint64_t before, target = 0;
    auto target_of = [&](uint64_t total) {
      // a token is kept while the sum before it is below p of the whole; the first one always
      const double t = ceil(top_p * (double)total);
      return target = t >= 1 ? min((uint64_t)t, total) : 1;
    };
    if (r.template select<true>(limit, at_most, target_of, d, before)) {
      const uint64_t w = r.fixed(r.real_weight(top - d)), some = (target - before + w - 1) / max(w, (uint64_t)1);
      at_most = d == limit ? min(at_most, some) : some;
      limit = d;
    }
  }
  const double w_limit = limit == ~0u ? 0 : r.real_weight(top - limit);
  if (w_limit < min_p) at_most = 0;
  const uint64_t fixed_limit = r.fixed(w_limit);

  // Sums of each warp's run of the slice
  const int per_warp = (r.vectors + kWarps - 1) / kWarps, v0 = min(r.vectors, warp * per_warp), v1 = min(r.vectors, v0 + per_warp);
  uint64_t above = 0;
  uint32_t equal = 0;
  auto weight = [&](uint32_t k) -> uint64_t {
    if (k <= K::kNone || top - k >= limit) return 0;
    const double w = r.real_weight(k);
    return w >= min_p ? r.fixed(w) : 0;
  };
  for (int v = v0 + lane; v < v1; v += 32) {
    uint32_t k[R::VEC];
    r.load(k, v);
#pragma unroll
    for (int j = 0; j < R::VEC; ++j) {
      above += weight(k[j]);
      equal += k[j] > K::kNone && top - k[j] == limit;
    }
  }
  above = sum_all(above);
  equal = __reduce_add_sync(kAll, equal);
  if (lane == 0) sh.warp[warp] = WarpSum{above, equal};
  r.meet();
  if (warp == 0) {
    // every block finds the warp at which the sum passes u of the whole: a few warps a lane
    const int all = blocks * kWarps, each = all / 32 > 0 ? all / 32 : 1;
    WarpSum part[kMostBlocks * kWarps / 32];
    uint64_t equals = 0;
#pragma unroll
    for (int i = 0; i < kMostBlocks * kWarps / 32; ++i) {
      const int w = lane * each + i;
      part[i] = i < each && w < all ? r.in_block(sh.warp, w / kWarps)[w % kWarps] : WarpSum{0, 0};
      equals += part[i].equal;
    }
    uint64_t left = inclusive(equals, lane) - equals;  // at the threshold before this lane's
    uint64_t sum = 0;
#pragma unroll
    for (int i = 0; i < kMostBlocks * kWarps / 32; ++i) {
      const uint64_t room = at_most > left ? at_most - left : 0;
      left += part[i].equal;
      sum += part[i].above + min(room, part[i].equal) * fixed_limit;
    }
    const uint64_t incl = inclusive(sum, lane), total = __shfl_sync(kAll, (unsigned long long)incl, 31);
    const double u = a.u64 ? reinterpret_cast<const double*>(a.u)[row] : (double)reinterpret_cast<const float*>(a.u)[row];
    // the sum passes u of the whole: is at least this
    uint64_t target = u > 0 ? (uint64_t)(fmin(u, 1.0) * (double)total) + 1 : 1;
    target = min(target, total);
    uint64_t at = incl - sum;
    left = inclusive(equals, lane) - equals;
    if (at < target && target <= incl) {
      bool open = true;
#pragma unroll
      for (int i = 0; i < kMostBlocks * kWarps / 32; ++i) {
        const uint64_t room = at_most > left ? at_most - left : 0, here = part[i].above + min(room, part[i].equal) * fixed_limit;
        if (open && target <= at + here) {
          open = false;
          const int w = lane * each + i;
          sh.win_block = w / kWarps, sh.win_warp = w % kWarps;
          sh.win_target = target - at;
          sh.win_equal = room;
        }
        at += here, left += part[i].equal;
      }
    }
  }
  r.meet();
  if (rank != (int)sh.win_block || warp != (int)sh.win_warp) return;
  // that warp goes through its run once more
  uint64_t target = sh.win_target, room = sh.win_equal;
  for (int v = v0; v < v1; v += 32) {
    uint32_t k[R::VEC];
    uint64_t sum = 0;
    uint32_t mine = 0;
    const bool there = v + lane < v1;
    if (there) r.load(k, v + lane);
#pragma unroll
    for (int j = 0; j < R::VEC; ++j) {
      if (!there) k[j] = 0;
      mine += k[j] > K::kNone && top - k[j] == limit;
    }
    const uint64_t equal_incl = inclusive(mine, lane);
    uint64_t left = room > equal_incl - mine ? room - (equal_incl - mine) : 0;  // for this lane's
    uint64_t w[R::VEC];
#pragma unroll
    for (int j = 0; j < R::VEC; ++j) {
      w[j] = weight(k[j]);
      if (k[j] > K::kNone && top - k[j] == limit && left) w[j] = fixed_limit, --left;
      sum += w[j];
    }
    const uint64_t incl = inclusive(sum, lane), all = __shfl_sync(kAll, (unsigned long long)incl, 31);
    if (target <= all) {
      uint64_t at = incl - sum;
      if (at < target && target <= incl) {
#pragma unroll
        for (int j = 0; j < R::VEC; ++j) {
          if (at < target && target <= at + w[j]) a.token[row] = first + (v + lane) * R::VEC - shift + j;
          at += w[j];
        }
      }
      return;
    }
    target -= all;
    const uint64_t seen = __shfl_sync(kAll, (unsigned long long)equal_incl, 31);
    room = room > seen ? room - seen : 0;
  }
}

template <typename T> int launch(Args a, cudaStream_t s) {
  // Blocks a row: as many as there is room for while a block has 2048 logits or more, and enough to hold the row
  auto smem = [&](int slice) { return (int)((sizeof(Shared) + 15) / 16 * 16 + ((size_t)slice + 16 / sizeof(T)) * sizeof(T) + 15) / 16 * 16; };
  int blocks = 1;
  const int64_t room = 2 * (int64_t)num_sms();
  auto slice_of = [&](int b) { return (a.V + b - 1) / b; };
  while (blocks < kMostBlocks && ((a.rows * blocks * 2 <= room && slice_of(blocks * 2) >= 2048) || smem(slice_of(blocks)) > 200 * 1024)) blocks *= 2;
  a.slice = slice_of(blocks);
  const int bytes = smem(a.slice);
  const int st = ensure_dyn_smem(reinterpret_cast<const void*>(sample_kernel<T>), 220 * 1024, "sample shared memory");
  if (st != FLB_OK) return st;
  cudaLaunchAttribute attr[1];
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.rows * blocks));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, sample_kernel<T>, a);
  count_launches(1);
  return check_cuda(e, "sample launch");
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
