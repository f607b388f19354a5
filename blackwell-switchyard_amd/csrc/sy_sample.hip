// Sampling: one token per row of logits by temperature, top-k, top-p and min-p from a
// given uniform number.
//
// With w_i = rint(2^44 exp((x_i - max) / T)) the candidates, in the order (x falling, i
// rising), are cut behind the k-th (top-k), then behind the one that reaches top_p of
// their weight; both cuts are a last kept candidate (x, i), and a token is kept iff it
// does not come after it. Whole numbers make every sum exact and independent of order:
// counts, weights per bin and the running sums of the draw need no fixed order, and the
// token is the same on every run.
//
// A workgroup of 16 waves per row, which is read from memory once into LDS (rows that do
// not fit are read again, from L2); a wave owns a contiguous run of it. The passes over the
// row are short loops: unrolled over registers they were bound by fetching their own code,
// which each workgroup runs once (8 rows of 32000 bf16 72 us, 256 of 50257 fp32 230). A cut is found without
// sorting: a histogram over 2048 equal steps of the logits' range (counts or weights, LDS
// atomics) gives the step in which it falls, and the few candidates of that step are
// ranked against one another in LDS. Steps with more candidates than fit (rows of equal
// logits) are bisected instead. What is kept is gathered, weighed once more and summed by
// 256 runs of indices; the one that holds the random number's place is ranked by index.
#include <algorithm>

#include "sy_launch.hpp"

namespace sy {

namespace {

constexpr int kBlock = 1024;
constexpr int kWaves = kBlock / 64;
constexpr int kBins = 2048;
constexpr int kRanked = kBlock;  // candidates that are ranked against one another
constexpr int kList = 4096;      // candidates that are gathered
constexpr int kRuns = 256;       // of a row's indices
constexpr double kOne = 17592186044416.0;  // 2^44

typedef unsigned long long u64;

__device__ __forceinline__ u64 shfl_up64(u64 x, int k) {
  const uint32_t lo = __shfl_up((uint32_t)x, k), hi = __shfl_up((uint32_t)(x >> 32), k);
  return ((u64)hi << 32) | lo;
}
__device__ __forceinline__ u64 shfl64(u64 x, int l) {
  const uint32_t lo = __shfl((uint32_t)x, l), hi = __shfl((uint32_t)(x >> 32), l);
  return ((u64)hi << 32) | lo;
}
__device__ __forceinline__ u64 scan64(u64 x) {  // inclusive over the lanes
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int k = 1; k < 64; k *= 2) {
    const u64 y = shfl_up64(x, k);
    if (lane >= k) x += y;
  }
  return x;
}

// exp2(z) for -46 < z <= 0 in double: 2^n times the series of exp over |y| <= ln(2)/2,
// whose first term left out is y^13/13! < 2e-16.
__device__ __forceinline__ double exp2_of(double z) {
  const double n = rint(z);
  const double y = (z - n) * 0.693147180559945309417;
  double p = 1.0 / 479001600.0;
  p = fma(p, y, 1.0 / 39916800.0);
  p = fma(p, y, 1.0 / 3628800.0);
  p = fma(p, y, 1.0 / 362880.0);
  p = fma(p, y, 1.0 / 40320.0);
  p = fma(p, y, 1.0 / 5040.0);
  p = fma(p, y, 1.0 / 720.0);
  p = fma(p, y, 1.0 / 120.0);
  p = fma(p, y, 1.0 / 24.0);
  p = fma(p, y, 1.0 / 6.0);
  p = fma(p, y, 0.5);
  p = fma(p, y, 1.0);
  p = fma(p, y, 1.0);
  return __longlong_as_double(__double_as_longlong(p) + ((long long)(int)n << 52));
}

// A token's weight as a fraction of the largest (e) and in units of 2^-44.
struct Weigher {
  float top;
  double c;  // log2(e) / T
  __device__ __forceinline__ double e(float x) const {
    if (x == top) return 1.0;
    const double z = ((double)x - (double)top) * c;
    return x > -INFINITY && z > -46.0 ? exp2_of(z) : 0.0;
  }
  // rint(e 2^44): 2^52 + w has the whole number in its mantissa
  static __device__ __forceinline__ u64 units(double e) {
    return (u64)__double_as_longlong(fma(e, kOne, 4503599627370496.0)) & 0xfffffffffffffull;
  }
  __device__ __forceinline__ u64 w(float x) const { return units(e(x)); }
};

// The candidates up to (x, i) in their order.
struct Last {
  float x;
  int i;
  __device__ __forceinline__ bool keeps(float y, int j) const { return y > x || (y == x && j <= i); }
};

__device__ __forceinline__ uint32_t key_of(float x) {  // rises with x
  const uint32_t u = __float_as_uint(x);
  return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float float_of(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}

struct Shared {
  u64 mass[kBins];  // weights (or counts) of the steps, then of the ranked
  float lx[kList];
  int li[kList];
  u64 run[kRuns];
  u64 sums[kWaves];
  float tops[kWaves], lows[kWaves];
  int n, bin, rank, tok;
  u64 before, total;
  Last last;
};

// A row, in LDS (`held`) or read from memory each time. A wave has nch chunks a lane of it.
template <class T>
struct Row {
  using S = typename T::storage;
  static constexpr int CE = T::ce;
  const S* p;
  const char* held;
  int vocab, nch, start;

  __device__ __forceinline__ int index(int j) const { return start + (j * 64 + (int)(threadIdx.x & 63)) * CE; }
  __device__ __forceinline__ i32x4_t load(int j) const {
    const int at = index(j);
    if (held != nullptr) return *reinterpret_cast<const i32x4_t*>(held + (int64_t)at * (int)sizeof(S));
    return fetch(at);
  }
  __device__ __forceinline__ i32x4_t fetch(int at) const {
    i32x4_t v;
    if (at + CE <= vocab) {
      __builtin_memcpy(&v, p + at, 16);  // rows start anywhere
    } else {
      S s[CE];
#pragma unroll
      for (int e = 0; e < CE; ++e) s[e] = at + e < vocab ? p[at + e] : S(0);
      __builtin_memcpy(&v, s, 16);
    }
    return v;
  }
  // f(logit, index) over the chunk's elements; NaN as -inf, -0 as 0, past the row -inf.
  template <class F> __device__ __forceinline__ void chunk(const i32x4_t& v, int at, F f) const {
#pragma unroll
    for (int e = 0; e < CE; ++e) {
      float y = elem<T>(v, e);
      y = at + e < vocab && y == y ? y + 0.0f : -INFINITY;
      f(y, at + e);
    }
  }
  template <class F> __device__ __forceinline__ void each(F f) const {
#pragma unroll 1
    for (int j = 0; j < nch; ++j) chunk(load(j), index(j), f);
  }
};

// Sum over the workgroup, known to every thread.
__device__ __forceinline__ u64 block_sum(Shared& sh, u64 x) {
  const u64 t = scan64(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) sh.sums[wave_id()] = t;
  __syncthreads();
  u64 s = 0;
#pragma unroll
  for (int k = 0; k < kWaves; ++k) s += sh.sums[k];
  return s;
}

// The last of the candidates up to `from` that a cut keeps. COUNT: the first `k` of them;
// else those before whose own place less than p of the total weight lies, at least one.
template <bool COUNT, class R>
__device__ __forceinline__ Last find_cut(Shared& sh, const R& row, const Weigher& wt, const Last& from, float low, u64 k, double p) {
  const int tid = threadIdx.x;
  const float span = wt.top - low;
  const float step = wt.top == INFINITY ? 1.0f : span > 0.0f ? (float)kBins / span : 0.0f;
  const auto bin_of = [&](float x) {  // falls with x; anything past the range in the last
    return x == wt.top ? 0 : (int)fminf((wt.top - x) * step, (float)(kBins - 1));
  };
  __syncthreads();
  for (int b = tid; b < kBins; b += kBlock) sh.mass[b] = 0;
  if (tid == 0) {
    sh.n = 0;
    sh.bin = -1;
    sh.rank = -1;
  }
  __syncthreads();
  uint32_t* const count = reinterpret_cast<uint32_t*>(sh.mass);
  row.each([&](float x, int i) {
    if (x == -INFINITY || !from.keeps(x, i)) return;
    const int b = bin_of(x);
    if constexpr (COUNT) {
      atomicAdd(&count[b], 1u);
    } else {
      const u64 w = wt.w(x);
      if (w != 0) atomicAdd(&sh.mass[b], w);
    }
  });
  __syncthreads();
  // Sums before each bin; a thread has two.
  const u64 a0 = COUNT ? count[2 * tid] : sh.mass[2 * tid];
  const u64 a1 = COUNT ? count[2 * tid + 1] : sh.mass[2 * tid + 1];
  const u64 incl = scan64(a0 + a1);
  if ((tid & 63) == 63) sh.sums[wave_id()] = incl;
  __syncthreads();
  u64 before = incl - (a0 + a1), total = 0;
#pragma unroll
  for (int q = 0; q < kWaves; ++q) {
    const u64 s = sh.sums[q];
    before += q < wave_id() ? s : 0;
    total += s;
  }
  // A place is kept where less than the goal lies before it.
  const double goal = COUNT ? (double)k : fmax(p * (double)total, 0.5);
  const auto kept = [&](u64 b) { return (double)b < goal; };
  if (a0 != 0 && kept(before) && !kept(before + a0)) {
    sh.bin = 2 * tid;
    sh.before = before;
  }
  if (a1 != 0 && kept(before + a0) && !kept(before + a0 + a1)) {
    sh.bin = 2 * tid + 1;
    sh.before = before + a0;
  }
  __syncthreads();
  const int bin = sh.bin;
  if (bin < 0) return from;  // the goal is never reached: nothing is cut
  const u64 base = sh.before;
  const auto in = [&](float x, int i) { return x != -INFINITY && bin_of(x) == bin && from.keeps(x, i); };
  row.each([&](float x, int i) {
    if (!in(x, i)) return;
    const int at = atomicAdd(&sh.n, 1);
    if (at < kRanked) {
      sh.lx[at] = x;
      sh.li[at] = i;
      sh.mass[at] = COUNT ? 1 : wt.w(x);
    }
  });
  __syncthreads();
  const int n = sh.n;
  if (n <= kRanked) {
    int rank = 0;
    u64 b = base;
    const bool mine = tid < n;
    const float x = mine ? sh.lx[tid] : 0.0f;
    const int i = mine ? sh.li[tid] : 0;
#pragma unroll 4
    for (int q = 0; q < n; ++q) {
      const bool ahead = sh.lx[q] > x || (sh.lx[q] == x && sh.li[q] < i);
      rank += ahead ? 1 : 0;
      b += ahead ? sh.mass[q] : 0;
    }
    const bool keep = mine && kept(b);
    if (keep) atomicMax(&sh.rank, rank);
    __syncthreads();
    if (keep && rank == sh.rank) sh.last = Last{x, i};
    __syncthreads();
    return sh.last;
  }
  // The highest logit that is reached with everything from it up, by halving the keys;
  // then how many of its equals are kept, and the last one's index, by halving indices.
  const auto measure = [&](auto pick) {
    u64 s = 0;
    row.each([&](float x, int i) {
      if (in(x, i) && pick(x, i)) s += COUNT ? 1 : wt.w(x);
    });
    return block_sum(sh, s);
  };
  uint32_t lo = key_of(-INFINITY), hi = key_of(wt.top);
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo + 1) / 2;
    const u64 s = base + measure([&](float x, int) { return key_of(x) >= mid; });
    if (!kept(s)) lo = mid;
    else hi = mid - 1;
  }
  const float xt = float_of(lo);
  const u64 ahead = base + measure([&](float x, int) { return x > xt; });
  int first = 0, last = row.vocab - 1;  // the last index that is kept among the equals
  while (first < last) {
    const int mid = first + (last - first) / 2;
    const u64 upto = measure([&](float x, int i) { return x == xt && i <= mid; });
    if (kept(ahead + upto)) first = mid + 1;  // the next equal one is kept too
    else last = mid;
  }
  return Last{xt, first};
}

template <class T, int HELD>  // bytes of LDS for the row
__global__ void __launch_bounds__(kBlock) k_sample(const SampleArgs a) {
  __shared__ Shared sh;
  __shared__ __align__(16) char held[HELD ? HELD : 16];
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
  const int64_t r = blockIdx.x;
  constexpr int CE = T::ce;
  Row<T> row;
  row.p = static_cast<const typename T::storage*>(a.logits) + r * a.row_stride;
  row.held = HELD ? held : nullptr;
  row.vocab = a.vocab;
  row.nch = (a.vocab + kBlock * CE - 1) / (kBlock * CE);
  row.start = wave * row.nch * 64 * CE;
  float top = -INFINITY, low = INFINITY;
#pragma unroll 4
  for (int j = 0; j < row.nch; ++j) {
    const int at = row.index(j);
    const i32x4_t v = row.fetch(at);
    if constexpr (HELD != 0) *reinterpret_cast<i32x4_t*>(held + at * (int)sizeof(typename T::storage)) = v;
    row.chunk(v, at, [&](float x, int) {
      top = fmaxf(top, x);
      low = x == -INFINITY ? low : fminf(low, x);
    });
  }
#pragma unroll
  for (int k = 32; k >= 1; k /= 2) {
    top = fmaxf(top, __shfl_xor(top, k));
    low = fminf(low, __shfl_xor(low, k));
  }
  if (lane == 0) {
    sh.tops[wave] = top;
    sh.lows[wave] = low;
  }
  if (tid == 0) sh.tok = 0x7fffffff;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kWaves; ++k) {
    top = fmaxf(top, sh.tops[k]);
    low = fminf(low, sh.lows[k]);
  }
  if (top == -INFINITY) {
    if (tid == 0) a.tokens[r] = -1;
    return;
  }
  const double t = a.how.temperatures != nullptr ? (double)a.how.temperatures[r] : a.how.temperature;
  if (!(t > 0.0)) {
    int at = 0x7fffffff;
    row.each([&](float x, int i) { at = x == top ? min(at, i) : at; });
    if (at != 0x7fffffff) atomicMin(&sh.tok, at);
    __syncthreads();
    if (tid == 0) a.tokens[r] = sh.tok;
    return;
  }
  const double top_p = a.how.top_ps != nullptr ? (double)a.how.top_ps[r] : a.how.top_p;
  const double min_p = fmin(a.how.min_ps != nullptr ? (double)a.how.min_ps[r] : a.how.min_p, 1.0);
  const int64_t top_k = a.how.top_ks != nullptr ? a.how.top_ks[r] : a.how.top_k;
  const Weigher wt{top, 1.44269504088896340736 / t};
  Last last{-INFINITY, 0x7fffffff};
  if (top_k >= 1 && top_k < a.vocab) last = find_cut<true>(sh, row, wt, last, low, (u64)top_k, 0.0);
  if (top_p < 1.0) {
    // Weights are zero from 45 ln 2 = 31.2 temperatures below the largest on.
    const float zero = top - (float)fmin(31.3 * t, 3.0e38);
    last = find_cut<false>(sh, row, wt, last, fmaxf(low, zero), 0, top_p);
  }
  // The draw. What is kept, weighed and summed by runs of indices.
  __syncthreads();
  if (tid == 0) sh.n = 0;
  if (tid < kRuns) sh.run[tid] = 0;
  __syncthreads();
  row.each([&](float x, int i) {
    if (x == -INFINITY || !last.keeps(x, i)) return;
    const int at = atomicAdd(&sh.n, 1);
    if (at < kList) {
      sh.lx[at] = x;
      sh.li[at] = i;
    }
  });
  __syncthreads();
  const int n = sh.n;
  const int len = (a.vocab + kRuns - 1) / kRuns;
  const auto weight = [&](float x) -> u64 {
    const double e = wt.e(x);
    return e >= min_p ? Weigher::units(e) : 0;
  };
  if (n <= kList) {
    for (int q = tid; q < n; q += kBlock) atomicAdd(&sh.run[sh.li[q] / len], weight(sh.lx[q]));
  } else {
    row.each([&](float x, int i) {
      if (x != -INFINITY && last.keeps(x, i)) atomicAdd(&sh.run[i / len], weight(x));
    });
  }
  __syncthreads();
  const u64 mine = tid < kRuns ? sh.run[tid] : 0;
  const u64 incl = scan64(mine);
  if (lane == 63) sh.sums[wave] = incl;
  if (tid == 0) sh.n = 0;
  __syncthreads();
  u64 before = incl - mine, total = 0;
#pragma unroll
  for (int k = 0; k < kRuns / 64; ++k) {
    const u64 s = sh.sums[k];
    before += k < wave ? s : 0;
    total += s;
  }
  const double u = (double)a.u[r];
  u64 goal = u > 0.0 ? (u64)fmin(u * (double)total, 9.0e18) : 0;
  goal = min(goal, total - 1);
  if (tid < kRuns && goal >= before && goal < before + mine) {
    sh.bin = tid;
    sh.before = before;
  }
  __syncthreads();
  // The run that holds the goal: at most 1024 tokens, a thread each, in the order of indices.
  const int i = sh.bin * len + tid;
  u64 w = 0;
  if (tid < len && i < a.vocab) {
    i32x4_t v = {0, 0, 0, 0};
    __builtin_memcpy(&v, row.p + i, sizeof(typename T::storage));
    float x = elem<T>(v, 0);
    x = x == x ? x + 0.0f : -INFINITY;
    if (x != -INFINITY && last.keeps(x, i)) w = weight(x);
  }
  u64 in = scan64(w);
  if (lane == 63) sh.sums[wave] = in;
  __syncthreads();
  in += sh.before;
#pragma unroll
  for (int k = 0; k < kWaves; ++k) in += k < wave ? sh.sums[k] : 0;
  if (goal >= in - w && goal < in) a.tokens[r] = i;
}

template <class T, int HELD>
hipError_t sample_n(const SampleArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((k_sample<T, HELD>), dim3((unsigned)a.n_rows), dim3(kBlock), 0, s, a);
  return hipGetLastError();
}

template <class T>
hipError_t sample_t(const SampleArgs& a, hipStream_t s) {
  // Whole chunks of every lane, which is what the kernel stores. Short rows leave room for
  // a second workgroup on a CU.
  const int64_t chunks = (a.vocab + kBlock * T::ce - 1) / (kBlock * T::ce);
  const int64_t bytes = chunks * kBlock * 16;
  if (bytes <= 16384) return sample_n<T, 16384>(a, s);
  if (bytes <= 98304) return sample_n<T, 98304>(a, s);
  return sample_n<T, 0>(a, s);
}

}  // namespace

hipError_t launch_sample(const SampleArgs& a, int dtype, hipStream_t s) {
  if (dtype == SY_BF16) return sample_t<BF16>(a, s);
  if (dtype == SY_F16) return sample_t<F16>(a, s);
  return sample_t<F32>(a, s);
}

}  // namespace sy
