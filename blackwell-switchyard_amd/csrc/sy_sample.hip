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
// which each workgroup runs once. A cut is found without sorting: a histogram over 2048
// equal steps of the logits' range (counts or weights, LDS atomics) gives the step in which
// it falls, and the few candidates of that step are ranked against one another in LDS.
// Steps with more candidates than fit (rows of equal logits) are bisected instead. What is
// kept is gathered, weighed once more and summed by runs of 64 chunks of the row; the run
// that holds the random number's place is scanned.
//
// 8 rows of 32000 bf16 with top-k and top-p take 17.7 us (72 with the rows in registers):
// one workgroup a CU, bound by the latency of its passes one after another. 256 rows of
// 50257 fp32 with top-p take 82 us (230): the row's 201 KB are read four times from the
// last cache, and of a workgroup's time 42 % go into the histogram with its double exp, 18 %
// into gathering, 14 % into the maximum, 7 % into the ranking and 19 % into the draw.
#include <algorithm>

#include "sy_launch.hpp"

namespace sy {

namespace {

constexpr int kBlock = 1024;
constexpr int kWaves = kBlock / 64;
constexpr int kBins = 2048;
constexpr int kRanked = kBlock;  // candidates that are ranked against one another
constexpr int kRuns = kBlock;    // of a row's indices, a wave's chunk each
constexpr int kGroup = 4;        // chunks that are read from memory together
constexpr double kOne = 17592186044416.0;  // 2^44

typedef unsigned long long u64;

__device__ __forceinline__ u64 scan64(u64 x) { return wave_scan<u64>(x); }  // inclusive over the lanes

// Sums over the 16 lanes of a row, in its last lane.
template <class U> __device__ __forceinline__ U row16_sum(U x) {
  x += dpp_whole<U, 0x111>(x);
  x += dpp_whole<U, 0x112>(x);
  x += dpp_whole<U, 0x114>(x);
  x += dpp_whole<U, 0x118>(x);
  return x;
}

// 2^y for |y| <= 1/2: the series of exp(y ln 2), whose first term left out is below 2e-16.
// (The coefficients are ln(2)^k / k!.)
__device__ __forceinline__ double exp2_near(double y) {
  constexpr double l = 0.693147180559945309417;
  constexpr double c2 = l * l / 2, c3 = c2 * l / 3, c4 = c3 * l / 4, c5 = c4 * l / 5, c6 = c5 * l / 6, c7 = c6 * l / 7,
                   c8 = c7 * l / 8, c9 = c8 * l / 9, c10 = c9 * l / 10, c11 = c10 * l / 11, c12 = c11 * l / 12;
  double p = fma(c12, y, c11);
  p = fma(p, y, c10);
  p = fma(p, y, c9);
  p = fma(p, y, c8);
  p = fma(p, y, c7);
  p = fma(p, y, c6);
  p = fma(p, y, c5);
  p = fma(p, y, c4);
  p = fma(p, y, c3);
  p = fma(p, y, c2);
  p = fma(p, y, l);
  return fma(p, y, 1.0);
}

// A token's weight as a fraction of the largest (e) and in units of 2^-44. Far below the
// largest, and for -inf, e is 2^-60, whose weight is zero.
struct Weigher {
  float top;
  double c;  // log2(e) / T, finite
  __device__ __forceinline__ double e(float x) const {
    if (top == INFINITY) return x == top ? 1.0 : 0.0;
    const double z = fmax(((double)x - (double)top) * c, -60.0);  // (0 times -inf: -60 too)
    const double n = rint(z);
    return ldexp(exp2_near(z - n), (int)n);
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

template <int LIST>  // candidates that are gathered
struct Shared {
  static constexpr int kList = LIST;
  u64 mass[kBins];  // weights (or counts) of the steps, then of the ranked
  float lx[LIST];  // gathered candidates
  int li[LIST];
  float rx[kRanked];  // ranked ones
  int ri[kRanked];
  u64 run[kRuns];
  u64 sums[kWaves];
  float tops[kWaves], lows[kWaves];
  int n, bin, rank, tok, listed;
  u64 before;
  Last last;
};

// The candidates: a row, in LDS (HELD: NaN there as -inf, and past the row) or read from
// memory each time; or what was gathered of it. A wave has nch chunks a lane of a row.
template <class T, bool HELD, class Shared>
struct Row {
  using S = typename T::storage;
  static constexpr int CE = T::ce;
  const S* p;
  char* held;
  Shared* sh;
  int vocab, nch, start;
  int listed;  // gathered candidates, or -1

  __device__ __forceinline__ int index(int j) const { return start + (j * 64 + (int)(threadIdx.x & 63)) * CE; }
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
  // A chunk's logits: NaN as -inf, -0 as 0, past the row -inf.
  __device__ __forceinline__ void clean(const i32x4_t& v, int at, float (&y)[CE]) const {
#pragma unroll
    for (int e = 0; e < CE; ++e) {
      const float x = elem<T>(v, e);
      y[e] = at + e < vocab && x == x ? x + 0.0f : -INFINITY;
    }
  }
  // f(logits, index of the first) of every chunk of the row.
  template <class F> __device__ __forceinline__ void chunks(F f) const {
    float y[CE];
    if constexpr (HELD) {
#pragma unroll 1
      for (int j = 0; j < nch; ++j) {
        const int at = index(j);
        const i32x4_t v = *reinterpret_cast<const i32x4_t*>(held + at * (int)sizeof(S));
#pragma unroll
        for (int e = 0; e < CE; ++e) y[e] = elem<T>(v, e);
        f(y, at);
      }
    } else {
      // Four chunks are on their way while the four before them are worked on.
      i32x4_t next[kGroup];
#pragma unroll
      for (int q = 0; q < kGroup; ++q) next[q] = fetch(index(q));
#pragma unroll 1
      for (int j = 0; j < nch; j += kGroup) {
        i32x4_t v[kGroup];
#pragma unroll
        for (int q = 0; q < kGroup; ++q) v[q] = next[q];
        if (j + kGroup < nch) {
#pragma unroll
          for (int q = 0; q < kGroup; ++q) next[q] = fetch(index(j + kGroup + q));
        }
#pragma unroll
        for (int q = 0; q < kGroup; ++q) {
          const int at = index(j + q);
          clean(v[q], at, y);
          f(y, at);
        }
      }
    }
  }
  // f(logit, index) of every candidate.
  template <class F> __device__ __forceinline__ void each(F f) const {
    if (listed >= 0) {
      for (int q = threadIdx.x; q < listed; q += kBlock) f(sh->lx[q], sh->li[q]);
    } else {
      chunks([&](const float (&y)[CE], int at) {
#pragma unroll
        for (int e = 0; e < CE; ++e) f(y[e], at + e);
      });
    }
  }
  // Gathers the row's logits above `over`, if there is room: a place for a wave's at a time.
  __device__ __forceinline__ void gather(float over) {
    chunks([&](const float (&y)[CE], int at) {
      uint32_t mask = 0;
#pragma unroll
      for (int e = 0; e < CE; ++e) mask |= y[e] > over ? 1u << e : 0u;
      if (!__any(mask)) return;
      const uint32_t n = __popc(mask), incl = wave_scan<uint32_t>(n);
      int base = 0;
      if ((threadIdx.x & 63) == 63) base = atomicAdd(&sh->listed, (int)incl);
      int to = __builtin_amdgcn_readlane(base, 63) + (int)(incl - n);
#pragma unroll
      for (int e = 0; e < CE; ++e) {
        if ((mask >> e & 1) == 0) continue;
        if (to < Shared::kList) {
          sh->lx[to] = y[e];
          sh->li[to] = at + e;
        }
        ++to;
      }
    });
    __syncthreads();
    if (sh->listed <= Shared::kList) listed = sh->listed;
  }
};

// Sum over the workgroup, known to every thread.
template <class Shared> __device__ __forceinline__ u64 block_sum(Shared& sh, u64 x) {
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
// Leaves the candidates that can still be kept gathered, if there is room for them.
// OPEN: nothing is cut yet (`from` keeps all). `clipped`: there are candidates below `low`,
// and all in the last step have no weight, so that it does not matter which of them are kept.
template <bool COUNT, bool OPEN, class Shared, class R>
__device__ __forceinline__ Last find_cut(Shared& sh, R& row, const Weigher& wt, const Last& from, float low, u64 k,
                                         double p, bool clipped) {
  const int tid = threadIdx.x;
  const bool few = !OPEN && row.listed >= 0 && row.listed <= kRanked / 2;  // all of them are ranked
  const float span = wt.top - low;
  const float step = span > 0.0f ? (float)kBins / span : 0.0f;
  const auto bin_of = [&](float x) {  // falls with x; anything past the range in the last
    if (few) return 0;
    if (wt.top == INFINITY) return x == wt.top ? 0 : kBins - 1;
    return (int)fminf((wt.top - x) * step, (float)(kBins - 1));
  };
  const auto left = [&](float x, int i) { return x != -INFINITY && (OPEN || from.keeps(x, i)); };
  __syncthreads();
  if (tid == 0) {
    sh.n = 0;
    sh.bin = -1;
    sh.rank = -1;
    sh.listed = 0;
  }
  int bin = 0;
  u64 base = 0;
  double goal;  // a place is kept where less than the goal lies before it
  const auto kept = [&](u64 b) { return (double)b < goal; };
  if (few) {
    u64 mine = 0;
    row.each([&](float x, int i) {
      if (left(x, i)) mine += COUNT ? 1 : wt.w(x);
    });
    const u64 total = block_sum(sh, mine);
    goal = COUNT ? (double)k : fmax(p * (double)total, 0.5);
    if (kept(total)) return from;
  } else {
    for (int b = tid; b < kBins; b += kBlock) sh.mass[b] = 0;
    __syncthreads();
    uint32_t* const count = reinterpret_cast<uint32_t*>(sh.mass);
    row.each([&](float x, int i) {
      if (!left(x, i)) return;
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
    goal = COUNT ? (double)k : fmax(p * (double)total, 0.5);
    if (a0 != 0 && kept(before) && !kept(before + a0)) {
      sh.bin = 2 * tid;
      sh.before = before;
    }
    if (a1 != 0 && kept(before + a0) && !kept(before + a0 + a1)) {
      sh.bin = 2 * tid + 1;
      sh.before = before + a0;
    }
    __syncthreads();
    bin = sh.bin;
    if (bin < 0) return from;  // the goal is never reached: nothing is cut
    if (clipped && bin == kBins - 1) return from;
    base = sh.before;
  }
  // The goal's bin and those before it are gathered, the ones in it ranked.
  if (row.listed < 0) {
    // A little below the bin's lower edge, whatever the roundings of bin_of.
    const float down = (float)(bin + 1) / step * 1.00001f;
    const bool edge = bin < kBins - 1 && step > 0.0f && wt.top != INFINITY;
    row.gather(edge ? wt.top - down - (fabsf(wt.top) + down) * 1e-6f : -INFINITY);
  }
  row.each([&](float x, int i) {
    if (!left(x, i) || bin_of(x) != bin) return;
    const int at = atomicAdd(&sh.n, 1);
    if (at < kRanked) {
      sh.rx[at] = x;
      sh.ri[at] = i;
      sh.mass[at] = COUNT ? 1 : wt.w(x);
    }
  });
  __syncthreads();
  const auto in = [&](float x, int i) { return left(x, i) && bin_of(x) == bin; };
  const int n = sh.n;
  if (n <= kRanked) {
    // Sixteen lanes count what is ahead of one candidate; the last of them has the sums.
    int best = -1;
    Last mine{};
    for (int at = tid / 16; at < n; at += kBlock / 16) {
      const float x = sh.rx[at];
      const int i = sh.ri[at];
      uint32_t rank = 0;
      u64 b = 0;
      for (int q = tid % 16; q < n; q += 16) {
        const float y = sh.rx[q];
        const u64 m = sh.mass[q];
        const bool ahead = y > x || (y == x && sh.ri[q] < i);
        rank += ahead ? 1 : 0;
        b += ahead ? m : 0;
      }
      rank = row16_sum(rank);
      b = row16_sum(b);
      if (tid % 16 == 15 && kept(base + b) && (int)rank > best) {
        best = (int)rank;
        mine = Last{x, i};
      }
    }
    if (best >= 0) atomicMax(&sh.rank, best);
    __syncthreads();
    if (best >= 0 && best == sh.rank) sh.last = mine;
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
  using Sh = Shared<HELD == 0 ? 14336 : 4096>;
  __shared__ Sh sh;
  __shared__ __align__(16) char held[HELD ? HELD : 16];
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
  const int64_t r = blockIdx.x;
  constexpr int CE = T::ce;
  Row<T, HELD != 0, Sh> row;
  row.p = static_cast<const typename T::storage*>(a.logits) + r * a.row_stride;
  row.held = held;
  row.sh = &sh;
  row.vocab = a.vocab;
  row.nch = (a.vocab + kBlock * CE - 1) / (kBlock * CE);
  if (HELD == 0) row.nch = (row.nch + kGroup - 1) / kGroup * kGroup;
  row.start = wave * row.nch * 64 * CE;
  row.listed = -1;
  // (Asked for before the row, not when they are needed.)
  const double t = a.how.temperatures != nullptr ? (double)a.how.temperatures[r] : a.how.temperature;
  const double top_p = a.how.top_ps != nullptr ? (double)a.how.top_ps[r] : a.how.top_p;
  const double min_p = fmin(a.how.min_ps != nullptr ? (double)a.how.min_ps[r] : a.how.min_p, 1.0);
  const int64_t top_k = a.how.top_ks != nullptr ? a.how.top_ks[r] : a.how.top_k;
  const double u = (double)a.u[r];
  float top = -INFINITY, low = INFINITY;
#pragma unroll 4
  for (int j = 0; j < row.nch; ++j) {
    const int at = row.index(j);
    float y[CE];
    row.clean(row.fetch(at), at, y);
#pragma unroll
    for (int e = 0; e < CE; ++e) {
      top = fmaxf(top, y[e]);
      low = y[e] == -INFINITY ? low : fminf(low, y[e]);
    }
    if constexpr (HELD != 0) *reinterpret_cast<i32x4_t*>(held + at * (int)sizeof(typename T::storage)) = pack<T>(y);
  }
  top = wave_max(top);
  low = -wave_max(-low);
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
  if (!(t > 0.0)) {
    int at = 0x7fffffff;
    row.each([&](float x, int i) { at = x == top ? min(at, i) : at; });
    if (at != 0x7fffffff) atomicMin(&sh.tok, at);
    __syncthreads();
    if (tid == 0) a.tokens[r] = sh.tok;
    return;
  }
  const Weigher wt{top, fmin(1.44269504088896340736 / t, 1e200)};
  Last last{-INFINITY, 0x7fffffff};
  if (top_k >= 1 && top_k < a.vocab) {
    // The steps end at 32 temperatures below the largest, past the last weight that is not
    // zero (and past that sum's rounding): tokens ruled out by the type's lowest number would
    // leave all others in the first step, to be bisected. 64 rows of 32000 bf16 with one such
    // token 18 us, 234 with the steps down to it.
    const float floor = top - (float)fmin(32.0 * t, 3.0e38) - (fabsf(top) + 1e-20f) * 2.4e-7f;
    last = find_cut<true, true>(sh, row, wt, last, fmaxf(low, floor), (u64)top_k, 0.0, low < floor);
  }
  if (top_p < 1.0) {
    // Weights are zero from 45 ln 2 = 31.2 temperatures below the largest on.
    const float zero = top - (float)fmin(31.3 * t, 3.0e38);
    if (last.x == -INFINITY)
      last = find_cut<false, true>(sh, row, wt, last, fmaxf(low, zero), 0, top_p, false);
    else
      last = find_cut<false, false>(sh, row, wt, last, fmaxf(low, zero), 0, top_p, false);
  }
  // The draw: what is kept, summed by runs of indices, which are a wave's chunk each.
  constexpr int kLen = 64 * CE;
  __syncthreads();
  sh.run[tid] = 0;
  __syncthreads();
  const auto weight = [&](float x, int i) -> u64 {
    if (x == -INFINITY || !last.keeps(x, i)) return 0;
    const double e = wt.e(x);
    return e >= min_p ? Weigher::units(e) : 0;
  };
  if (row.listed >= 0) {
    for (int q = tid; q < row.listed; q += kBlock) {
      const int i = sh.li[q];
      atomicAdd(&sh.run[i / kLen], weight(sh.lx[q], i));
    }
  } else {
    row.chunks([&](const float (&y)[CE], int at) {
      u64 w = 0;
#pragma unroll
      for (int e = 0; e < CE; ++e) w += weight(y[e], at + e);
      w = scan64(w);
      if (lane == 63 && at < kRuns * kLen) sh.run[at / kLen] = w;
    });
  }
  __syncthreads();
  const u64 mine = sh.run[tid];
  const u64 incl = scan64(mine);
  if (lane == 63) sh.sums[wave] = incl;
  __syncthreads();
  u64 before = incl - mine, total = 0;
#pragma unroll
  for (int k = 0; k < kWaves; ++k) {
    const u64 s = sh.sums[k];
    before += k < wave ? s : 0;
    total += s;
  }
  u64 goal = u > 0.0 ? (u64)fmin(u * (double)total, 9.0e18) : 0;
  goal = min(goal, total - 1);
  if (goal >= before && goal < before + mine) {
    sh.bin = tid;
    sh.before = before;
  }
  __syncthreads();
  // The run that holds the goal, a thread a token, in the order of indices.
  const int i = sh.bin * kLen + tid;
  u64 w = 0;
  if (tid < kLen && i < a.vocab) {
    i32x4_t v = {0, 0, 0, 0};
    __builtin_memcpy(&v, row.p + i, sizeof(typename T::storage));
    const float x = elem<T>(v, 0);
    w = weight(x == x ? x + 0.0f : -INFINITY, i);
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
hipError_t sample_rows(const SampleArgs& a, hipStream_t s) {
  // Whole chunks of every lane, which is what the kernel stores. (Less LDS for short rows
  // would put no second workgroup on a CU: sixteen waves of 90 registers fill it.)
  const int64_t chunks = (a.vocab + kBlock * T::ce - 1) / (kBlock * T::ce);
  const int64_t bytes = chunks * kBlock * 16;
  if (bytes <= 81920) return sample_n<T, 81920>(a, s);
  return sample_n<T, 0>(a, s);
}

// A launch has less than 2^32 threads: 2^21 rows at a time.
template <class T>
hipError_t sample_t(const SampleArgs& a, hipStream_t s) {
  constexpr int64_t kMost = 1 << 21;
  hipError_t e = hipSuccess;
  for (int64_t r = 0; r < a.n_rows && e == hipSuccess; r += kMost) {
    SampleArgs b = a;
    const auto from = [&](auto& p) {
      if (p != nullptr) p += r;
    };
    b.logits = static_cast<const typename T::storage*>(a.logits) + r * a.row_stride;
    from(b.u);
    from(b.tokens);
    from(b.how.temperatures);
    from(b.how.top_ps);
    from(b.how.min_ps);
    from(b.how.top_ks);
    b.n_rows = std::min(a.n_rows - r, kMost);
    e = sample_rows<T>(b, s);
  }
  return e;
}

}  // namespace

hipError_t launch_sample(const SampleArgs& a, int dtype, hipStream_t s) {
  if (dtype == SY_BF16) return sample_t<BF16>(a, s);
  if (dtype == SY_F16) return sample_t<F16>(a, s);
  return sample_t<F32>(a, s);
}

}  // namespace sy
