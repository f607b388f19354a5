// What is done to logits before a token is drawn from them: penalties for tokens that were
// there before, biases, and a mask of the tokens that are allowed.
//
//   y = x                                   token not among the row's `length` first ones
//   y = (x > 0 ? x / r : x r) - f n - p [n > 0]  else; n counts it behind the prompt
//   out = y + bias, or -inf where the token is not allowed
#include <algorithm>

#include "sy_launch.hpp"

namespace sy {

namespace {

typedef uint32_t u32x2_any_t __attribute__((ext_vector_type(2), aligned(1)));

constexpr int kBlock = 256;
constexpr uint32_t kPrompt = 0x80000000u;  // of a token's count: it was in the prompt

// Which of CE tokens from v on are allowed, a bit each.
template <int CE>
__device__ __forceinline__ uint32_t allowed(const AdjustArgs& a, int64_t row, int v, bool full) {
  constexpr uint32_t all = (1u << CE) - 1u;
  if (a.mask == nullptr) return all;
  if (a.mask_bytes) {
    const uint8_t* const m = static_cast<const uint8_t*>(a.mask) + row * a.mask_stride + v;
    uint32_t r = 0;
    if (full) {
      uint32_t w[2] = {0, 0};
      if constexpr (CE == 8) {
        const u32x2_any_t x = *reinterpret_cast<const u32x2_any_t*>(m);
        w[0] = x[0], w[1] = x[1];
      } else {
        __builtin_memcpy(w, m, 4);
      }
#pragma unroll
      for (int e = 0; e < CE; ++e) r |= (w[e / 4] >> (8 * (e % 4)) & 0xffu ? 1u : 0u) << e;
    } else {
#pragma unroll
      for (int e = 0; e < CE; ++e)
        if (v + e < a.vocab && m[e] != 0) r |= 1u << e;
    }
    return r;
  }
  return static_cast<const uint32_t*>(a.mask)[row * a.mask_stride + (v >> 5)] >> (v & 31) & all;
}

__device__ __forceinline__ void count(uint32_t* seen, int64_t token, int lo, int n, bool said) {
  const int64_t at = token - lo;
  if ((uint64_t)at >= (uint64_t)n) return;
  if (said) atomicAdd(&seen[at], 1u);
  else atomicOr(&seen[at], kPrompt);
}

// The row's first `len` tokens, eight a thread on their way at a time.
template <class I>
__device__ __forceinline__ void count_all(uint32_t* seen, const I* t, int64_t len, int64_t prompt, int lo, int n) {
  constexpr int kAhead = 8;
  for (int64_t i0 = threadIdx.x; i0 < len; i0 += kBlock * kAhead) {
    I x[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int64_t i = i0 + j * kBlock;
      x[j] = i < len ? t[i] : (I)-1;
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) count(seen, x[j], lo, n, i0 + j * kBlock >= prompt);
  }
}

// CE neighbouring numbers at p as fp32; those from `n` on are zero.
template <class T, int CE> __device__ __forceinline__ void ld_row_part(const void* p, int n, float (&f)[CE]) {
  using S = typename T::storage;
  const S* const s = static_cast<const S*>(p);
  if (n >= CE) {
#pragma unroll
    for (int q = 0; q < CE / T::ce; ++q) {
      const i32x4_t w = *reinterpret_cast<const i32x4_any_t*>(s + q * T::ce);
#pragma unroll
      for (int e = 0; e < T::ce; ++e) f[q * T::ce + e] = elem<T>(w, e);
    }
  } else {
#pragma unroll
    for (int e = 0; e < CE; ++e) f[e] = e < n ? load_elem(s, e, T::code) : 0.0f;
  }
}

// A workgroup takes a slice of one row, IT chunks a thread, all of them on their way while it
// reads the row's history and counts in LDS what falls into its slice: in whole numbers, so in
// any order. Chunks with nothing allowed are not read; in place and without a bias only those
// are that something was counted in, and all that stay as they are are not written.
template <class T, int IT>
__global__ void __launch_bounds__(kBlock) k_adjust(const AdjustArgs a, int slices) {
  using S = typename T::storage;
  constexpr int CE = T::ce, kSlice = kBlock * CE * IT;
  constexpr uint32_t all = (1u << CE) - 1u;
  extern __shared__ uint32_t seen[];
  const int64_t row = blockIdx.x / slices;
  const int lo = (int)(blockIdx.x % slices) * kSlice, n = min(kSlice, a.vocab - lo);
  const S* const x = static_cast<const S*>(a.logits) + row * a.row_stride + lo;
  S* const y = static_cast<S*>(a.out) + row * a.out_stride + lo;
  const bool in_place = static_cast<const void*>(x) == static_cast<const void*>(y);
  const bool lazy = in_place && a.bias == nullptr;
  uint32_t keep[IT];
#pragma unroll
  for (int k = 0; k < IT; ++k) {
    const int c = (k * kBlock + threadIdx.x) * CE;
    keep[k] = c < n ? allowed<CE>(a, row, lo + c, c + CE <= n) : 0u;
  }
  float v[IT][CE];
  if (!lazy) {
#pragma unroll
    for (int k = 0; k < IT; ++k) {
      const int c = (k * kBlock + threadIdx.x) * CE;
#pragma unroll
      for (int e = 0; e < CE; ++e) v[k][e] = 0.0f;
      if (keep[k] != 0) ld_row_part<T, CE>(x + c, n - c, v[k]);
    }
  }
  const double r = a.repetitions != nullptr ? a.repetitions[row] : a.repetition;
  const double p = a.presences != nullptr ? a.presences[row] : a.presence;
  const double f = a.frequencies != nullptr ? a.frequencies[row] : a.frequency;
  const double inv_r = 1.0 / r;  // (its rounding is 2^-53, and a division a token was 1 us)
  const bool counted = a.tokens != nullptr && (r != 1.0 || p != 0.0 || f != 0.0);
  if (counted) {
#pragma unroll
    for (int k = 0; k < IT; ++k)
#pragma unroll
      for (int q = 0; q < CE / 4; ++q)
        *reinterpret_cast<i32x4_t*>(seen + (k * kBlock + threadIdx.x) * CE + 4 * q) = i32x4_t{0, 0, 0, 0};
    __syncthreads();
    const int64_t len = a.lengths != nullptr ? min(max((int64_t)a.lengths[row], (int64_t)0), a.n_tokens) : a.n_tokens;
    const int64_t prompt = a.prompts != nullptr ? a.prompts[row] : 0;
    if (a.tokens64) count_all(seen, static_cast<const int64_t*>(a.tokens) + row * a.tokens_stride, len, prompt, lo, n);
    else count_all(seen, static_cast<const int32_t*>(a.tokens) + row * a.tokens_stride, len, prompt, lo, n);
    __syncthreads();
  }
#pragma unroll
  for (int k = 0; k < IT; ++k) {
    const int c = (k * kBlock + threadIdx.x) * CE;
    if (c >= n) break;
    uint32_t cnt[CE], any = 0;
#pragma unroll
    for (int e = 0; e < CE; ++e) cnt[e] = 0;
    if (counted) {
#pragma unroll
      for (int q = 0; q < CE / 4; ++q) {
        const i32x4_t w = *reinterpret_cast<const i32x4_t*>(seen + c + 4 * q);
#pragma unroll
        for (int e = 0; e < 4; ++e) cnt[4 * q + e] = (uint32_t)w[e], any |= (uint32_t)w[e];
      }
    }
    if (lazy) {
      const uint32_t there = n - c >= CE ? all : (1u << (n - c)) - 1u;
      if (any == 0 && (keep[k] & there) == there) continue;
#pragma unroll
      for (int e = 0; e < CE; ++e) v[k][e] = 0.0f;
      if (keep[k] != 0) ld_row_part<T, CE>(x + c, n - c, v[k]);
    }
    if (any != 0) {
#pragma unroll
      for (int e = 0; e < CE; ++e) {
        const uint32_t said = cnt[e] & ~kPrompt;
        const double z = v[k][e];
        const double y = fma(z, z > 0.0 ? inv_r : r, said != 0 ? -fma(f, (double)said, p) : 0.0);
        v[k][e] = cnt[e] != 0 ? (float)y : v[k][e];
      }
    }
    if (a.bias != nullptr && keep[k] != 0) {
      const int64_t at = row * a.bias_stride + lo + c;
      float b[CE];
      if (a.bias_f32) ld_row_part<F32, CE>(static_cast<const float*>(a.bias) + at, n - c, b);
      else ld_row_part<T, CE>(static_cast<const S*>(a.bias) + at, n - c, b);
#pragma unroll
      for (int e = 0; e < CE; ++e) v[k][e] += b[e];
    }
#pragma unroll
    for (int e = 0; e < CE; ++e)
      if ((keep[k] >> e & 1u) == 0) v[k][e] = -__builtin_inff();
    if (c + CE <= n) {
      // (Where there is much to write it goes past the caches: 256 rows of 50257 in fp32 25.8 ->
      // 23.9 us; 8 of 32000 in bf16 8.1 -> 8.6.)
      i32x4_any_t* const to = reinterpret_cast<i32x4_any_t*>(y + c);
      if constexpr (IT == 4) __builtin_nontemporal_store((i32x4_any_t)pack<T>(v[k]), to);
      else *to = pack<T>(v[k]);
    } else {
#pragma unroll
      for (int e = 0; e < CE; ++e)
        if (c + e < n) store_elem(y, c + e, v[k][e], T::code);
    }
  }
}

template <class T, int IT>
hipError_t adjust_it(const AdjustArgs& a, hipStream_t s) {
  constexpr int kSlice = kBlock * T::ce * IT;
  const int slices = (a.vocab + kSlice - 1) / kSlice;
  const int64_t rows = std::max<int64_t>(1, (1 << 22) / slices);  // of a launch: 2^30 threads
  for (int64_t r0 = 0; r0 < a.n_rows; r0 += rows) {
    AdjustArgs part = a;
    part.n_rows = std::min(rows, a.n_rows - r0);
    const int64_t es = sizeof(typename T::storage);
    part.logits = static_cast<const char*>(a.logits) + r0 * a.row_stride * es;
    part.out = static_cast<char*>(a.out) + r0 * a.out_stride * es;
    if (a.tokens) part.tokens = static_cast<const char*>(a.tokens) + r0 * a.tokens_stride * (a.tokens64 ? 8 : 4);
    if (a.lengths) part.lengths += r0;
    if (a.prompts) part.prompts += r0;
    if (a.repetitions) part.repetitions += r0;
    if (a.presences) part.presences += r0;
    if (a.frequencies) part.frequencies += r0;
    if (a.bias) part.bias = static_cast<const char*>(a.bias) + r0 * a.bias_stride * (a.bias_f32 ? 4 : es);
    if (a.mask) part.mask = static_cast<const char*>(a.mask) + r0 * a.mask_stride * (a.mask_bytes ? 1 : 4);
    hipLaunchKernelGGL((k_adjust<T, IT>), dim3((unsigned)(part.n_rows * slices)), dim3(kBlock),
                       a.tokens ? kSlice * sizeof(uint32_t) : 0, s, part, slices);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <class T>
hipError_t adjust_t(const AdjustArgs& a, hipStream_t s) {
  const int64_t chunks = a.n_rows * ((a.vocab + kBlock * T::ce - 1) / (kBlock * T::ce));  // workgroups of one each
  if (chunks >= 4096) return adjust_it<T, 4>(a, s);
  if (chunks >= 2048) return adjust_it<T, 2>(a, s);
  return adjust_it<T, 1>(a, s);
}

}  // namespace

hipError_t launch_adjust(const AdjustArgs& a, int dtype, hipStream_t s) {
  if (dtype == SY_BF16) return adjust_t<BF16>(a, s);
  if (dtype == SY_F16) return adjust_t<F16>(a, s);
  return adjust_t<F32>(a, s);
}

}  // namespace sy
