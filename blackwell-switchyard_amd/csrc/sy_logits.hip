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

// A barrier for what is in LDS alone: loads from memory stay on their way across it.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Eight tokens a thread of a row of `n_tokens`, from i0 on; what is no token of 31 bits is -1.
constexpr int kAhead = 8;
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
template <int kBlock>
__device__ __forceinline__ void ld_tokens(const AdjustArgs& a, int64_t row, int i0, int (&x)[kAhead]) {
  const int first = i0 + (int)threadIdx.x;
  if (a.tokens64) {
    const u32x2_t* const t = static_cast<const u32x2_t*>(a.tokens) + row * a.tokens_stride + first;
    u32x2_t w[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) w[j] = first + j * kBlock < (int)a.n_tokens ? t[j * kBlock] : u32x2_t{0, 1};
#pragma unroll
    for (int j = 0; j < kAhead; ++j) x[j] = w[j][1] == 0 ? (int)w[j][0] : -1;
  } else {
    const int* const t = static_cast<const int*>(a.tokens) + row * a.tokens_stride + first;
#pragma unroll
    for (int j = 0; j < kAhead; ++j) x[j] = first + j * kBlock < (int)a.n_tokens ? t[j * kBlock] : -1;
  }
}

// A chunk as it lies in memory; elements from `n` on are zero.
template <class T> __device__ __forceinline__ i32x4_t ld_chunk(const typename T::storage* p, int n) {
  if (n >= T::ce) return *reinterpret_cast<const i32x4_any_t*>(p);
  i32x4_t r = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < T::ce; ++e) {
    if (e >= n) continue;
    if constexpr (T::ce == 4) r[e] = __float_as_int(p[e]);
    else r[e / 2] |= (int)((uint32_t)p[e] << (16 * (e % 2)));
  }
  return r;
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

// The elements of a chunk that `keep` has a bit for; -inf for the others.
template <class T> __device__ __forceinline__ i32x4_t masked(const i32x4_t& x, uint32_t keep) {
  constexpr int kInf = T::code == F32::code ? (int)0xff800000 : T::code == BF16::code ? (int)0xff80ff80 : (int)0xfc00fc00;
  const auto all = [&](int e) { return (int)(keep << (31 - e)) >> 31; };
  i32x4_t r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int m = T::ce == 4 ? all(i) : (all(2 * i) & 0xffff) | (all(2 * i + 1) & (int)0xffff0000);
    r[i] = (x[i] & m) | (kInf & ~m);
  }
  return r;
}

// A workgroup takes a slice of one row, IT chunks a thread, all of them on their way (and left
// as they come) while it deals with the row's history. It counts in LDS what falls into its
// slice, in whole numbers, so in any order, and lists the tokens that are there; then penalises
// those, a thread each, puts the results in the counts' places and sets a bit for each (worked
// out in the chunks that hold them, 82 rows of 92375 in fp16 with 1290 tokens 13.9 us, so 9.7;
// 8 rows with 3808 tokens 5.5, so 7.3). Then one pass over the chunks. Those with
// nothing allowed are not read; in place and without a bias only those are that something was
// counted in, and all that stay as they are are not written. Memory bounds many rows: 256 of
// 50257 in fp32 with 1500 tokens, biases and a mask 106 MB in 24.5 us, 4.3 TB/s; latency, of
// the history above all, few: 8 of 32000 in bf16 with 4000 tokens 6.0.
template <class T, int IT, int kBlock>
__global__ void __launch_bounds__(kBlock) k_adjust(const AdjustArgs a, int slices) {
  using S = typename T::storage;
  constexpr int CE = T::ce, kSlice = kBlock * CE * IT;
  constexpr uint32_t all = (1u << CE) - 1u;
  extern __shared__ uint32_t seen[];
  uint32_t* const there = seen + kSlice;  // a bit a token
  uint32_t* const listed = there + kSlice / 32;
  uint16_t* const list = reinterpret_cast<uint16_t*>(listed + 1);
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
  int ahead[kAhead];
  if (a.tokens != nullptr) ld_tokens<kBlock>(a, row, 0, ahead);
  i32x4_t raw[IT];
#pragma unroll
  for (int k = 0; k < IT; ++k) {
    const int c = (k * kBlock + threadIdx.x) * CE;
    raw[k] = i32x4_t{0, 0, 0, 0};
    if (!lazy && keep[k] != 0) raw[k] = ld_chunk<T>(x + c, n - c);
  }
  const double r = a.repetitions != nullptr ? a.repetitions[row] : a.repetition;
  const double p = a.presences != nullptr ? a.presences[row] : a.presence;
  const double f = a.frequencies != nullptr ? a.frequencies[row] : a.frequency;
  const bool counted = a.tokens != nullptr && (r != 1.0 || p != 0.0 || f != 0.0);
  if (counted) {
    const int len = a.lengths != nullptr ? min(a.lengths[row], (int)a.n_tokens) : (int)a.n_tokens;
    const int prompt = a.prompts != nullptr ? a.prompts[row] : 0;
#pragma unroll
    for (int k = 0; k < IT * CE / 4; ++k)
      *reinterpret_cast<i32x4_t*>(seen + (k * kBlock + threadIdx.x) * 4) = i32x4_t{0, 0, 0, 0};
    if (threadIdx.x < kSlice / 128) *reinterpret_cast<i32x4_t*>(there + threadIdx.x * 4) = i32x4_t{0, 0, 0, 0};
    if (threadIdx.x == 0) *listed = 0;
    lds_barrier();
    for (int i0 = 0; i0 < len; i0 += kBlock * kAhead) {
      int next[kAhead];
      if (i0 + kBlock * kAhead < len) ld_tokens<kBlock>(a, row, i0 + kBlock * kAhead, next);
      uint32_t before[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int i = i0 + j * kBlock + (int)threadIdx.x;
        ahead[j] -= lo;
        before[j] = 1;
        if (i >= len || (uint32_t)ahead[j] >= (uint32_t)n) continue;
        before[j] = i >= prompt ? atomicAdd(&seen[ahead[j]], 1u) : atomicOr(&seen[ahead[j]], kPrompt);
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
        if (before[j] == 0) list[atomicAdd(listed, 1u)] = (uint16_t)ahead[j];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) ahead[j] = next[j];
    }
    lds_barrier();
    const int count = (int)*listed;
    for (int i = threadIdx.x; i < count; i += kBlock) {
      const int at = list[i];
      const uint32_t said = seen[at] & ~kPrompt;
      const double z = load_elem(x, at, T::code);
      seen[at] = __float_as_uint((float)((z > 0.0 ? z / r : z * r) - (said != 0 ? fma(f, (double)said, p) : 0.0)));
      atomicOr(&there[at >> 5], 1u << (at & 31));
    }
    lds_barrier();
  }
#pragma unroll
  for (int k = 0; k < IT; ++k) {
    const int c = (k * kBlock + threadIdx.x) * CE;
    if (c >= n) break;
    const uint32_t set = counted ? there[c >> 5] >> (c & 31) & all : 0u;
    if (lazy) {
      const uint32_t inside = n - c >= CE ? all : (1u << (n - c)) - 1u;
      if (set == 0 && (keep[k] & inside) == inside) continue;
      if (keep[k] != 0) raw[k] = ld_chunk<T>(x + c, n - c);
    }
    if ((set != 0 || a.bias != nullptr) && keep[k] != 0) {
      float v[CE];
#pragma unroll
      for (int e = 0; e < CE; ++e) v[e] = elem<T>(raw[k], e);
      if (set != 0) {
#pragma unroll
        for (int q = 0; q < CE / 4; ++q) {
          const i32x4_t w = *reinterpret_cast<const i32x4_t*>(seen + c + 4 * q);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[4 * q + e] = set >> (4 * q + e) & 1u ? __int_as_float(w[e]) : v[4 * q + e];
        }
      }
      if (a.bias != nullptr) {
        const int64_t at = row * a.bias_stride + lo + c;
        float b[CE];
        if (a.bias_f32) ld_row_part<F32, CE>(static_cast<const float*>(a.bias) + at, n - c, b);
        else ld_row_part<T, CE>(static_cast<const S*>(a.bias) + at, n - c, b);
#pragma unroll
        for (int e = 0; e < CE; ++e) v[e] += b[e];
      }
      raw[k] = pack<T>(v);
    }
    if (a.mask != nullptr) raw[k] = masked<T>(raw[k], keep[k]);
    if (c + CE <= n) {
      // (Where there is much to write it goes past the caches: 256 rows of 50257 in fp32 25.8 ->
      // 23.9 us, 82 of 92375 in fp16 10.9 -> 9.7; 8 of 32000 in bf16 8.1 -> 8.6.)
      i32x4_any_t* const to = reinterpret_cast<i32x4_any_t*>(y + c);
      if constexpr (CE * IT == 16) __builtin_nontemporal_store((i32x4_any_t)raw[k], to);
      else *to = raw[k];
    } else {
#pragma unroll
      for (int e = 0; e < CE; ++e)
        if (c + e < n) store_elem(y, c + e, elem<T>(raw[k], e), T::code);
    }
  }
}

template <class T, int IT, int kBlock>
hipError_t adjust_it(const AdjustArgs& a, hipStream_t s) {
  constexpr int kSlice = kBlock * T::ce * IT;
  const int slices = (a.vocab + kSlice - 1) / kSlice;
  const int64_t rows = std::max<int64_t>(1, (1 << 22) / slices);  // of a launch: 2^30 threads
  // A count and a bit a token, and the tokens that are there.
  const int lds = a.tokens ? kSlice * 4 + kSlice / 8 + 4 + 2 * (int)std::min<int64_t>(kSlice, a.n_tokens) : 0;
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
    hipLaunchKernelGGL((k_adjust<T, IT, kBlock>), dim3((unsigned)(part.n_rows * slices)), dim3(kBlock),
                       lds, s, part, slices);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

// Slices as long as leave every CU workgroups: each reads the row's whole history. Past 4096
// tokens of a 16-bit row the counts would leave too few workgroups to a CU: 98 rows of 116414 in
// bf16 with 1290 tokens 15.9 us with slices of 8192, 13.8 with 4096. Where rows are few and
// histories long, 1024 threads read them faster: 8 rows of 32000 in bf16 with 2000 tokens 5.0
// us, 4000 5.6, 14000 9.2, with 256 threads 5.0, 6.9 and 16.0; but 98 rows of 116414 with 4000
// 27.4 and 20.5.
template <class T>
hipError_t adjust_t(const AdjustArgs& a, hipStream_t s) {
  if (a.tokens != nullptr && a.n_tokens > 2048 && a.n_rows * ((a.vocab + 1024 * T::ce - 1) / (1024 * T::ce)) <= 512)
    return adjust_it<T, 1, 1024>(a, s);
  const int64_t chunks = a.n_rows * ((a.vocab + 256 * T::ce - 1) / (256 * T::ce));  // workgroups of one each
  if constexpr (T::ce == 4) {
    if (chunks >= 4096) return adjust_it<T, 4, 256>(a, s);
  }
  return chunks >= 2048 ? adjust_it<T, 2, 256>(a, s) : adjust_it<T, 1, 256>(a, s);
}

}  // namespace

hipError_t launch_adjust(const AdjustArgs& a, int dtype, hipStream_t s) {
  if (dtype == SY_BF16) return adjust_t<BF16>(a, s);
  if (dtype == SY_F16) return adjust_t<F16>(a, s);
  return adjust_t<F32>(a, s);
}

}  // namespace sy
