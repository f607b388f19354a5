// The norm of every query and key head with the rotation to its position, and the split of
// a fused projection into attention's layout, in one pass each way.
//
//   u = x r,  r = 1 / sqrt(mean(x^2) + eps)         over a head's channels
//   y = R_t (g u)    channel i of the first half turns with channel i of the second
//
//   backward, from dy:  e = R_t^T dy,  dg = sum e u,  dx = r (g e - u mean(g e u))
#include <algorithm>
#include <type_traits>

#include "sy_launch.hpp"

namespace sy {

namespace {

constexpr int kBlock = 256;
constexpr int kWaves = kBlock / 64;

typedef int i32x2_t __attribute__((ext_vector_type(2)));

// VE neighbouring channels as fp32. They are read once, and asked for as such: forward and
// backward of 4 x 2048 tokens of 16 heads of 128 in bf16 99 -> 91 us.
template <class T, int VE>
__device__ __forceinline__ void ld_part(const typename T::storage* p, float (&f)[VE]) {
  i32x4_t x;
  if constexpr (VE == T::ce) {
    x = __builtin_nontemporal_load(reinterpret_cast<const i32x4_t*>(p));
  } else {
    const i32x2_t y = __builtin_nontemporal_load(reinterpret_cast<const i32x2_t*>(p));
    x = i32x4_t{y[0], y[1], 0, 0};
  }
#pragma unroll
  for (int e = 0; e < VE; ++e) f[e] = elem<T>(x, e);
}
template <class T, int VE>
__device__ __forceinline__ void st_part(typename T::storage* p, const float (&f)[VE]) {
  float g[T::ce] = {};
#pragma unroll
  for (int e = 0; e < VE; ++e) g[e] = f[e];
  const i32x4_t x = pack<T>(g);
  if constexpr (VE == T::ce) *reinterpret_cast<i32x4_t*>(p) = x;
  else *reinterpret_cast<i32x2_t*>(p) = i32x2_t{x[0], x[1]};
}

// L lanes a head, each with the two parts of VE channels that turn together (lanes past the
// head do nothing); a wave has 64 / L neighbouring tokens of one head, so it writes one run of
// memory. The waves of gridDim.y workgroups share the heads out in runs: a wave goes over its
// queries, then its keys, then its values, and over all its tokens for each; it holds one gain,
// and the sums of one gain's gradient, at a time. Memory bounds it: 4 x 2048 tokens of 16 heads
// of 128 in bf16 move 201 MB forward in 36.7 us, 5.5 TB/s, and 269 MB backward in 50.2, 5.4
// TB/s; with two heads' loads on their way 8 us more.
template <class T, int VE, int L, bool BWD>
__global__ void __launch_bounds__(kBlock) k_head_norm(const HeadNormArgs a) {
  using S = typename T::storage;
  constexpr int kSlots = 64 / L;
  [[maybe_unused]] __shared__ float fold[BWD ? kWaves : 1][2][2][L * VE];
  const int lane = threadIdx.x & 63, part = lane % L, slot = lane / L;
  const int half = a.hd / 2, ch = part * VE;
  const bool in_row = ch < half;
  const int rows = a.heads + 2 * a.kv_heads;
  const int per = (rows + (int)gridDim.y * kWaves - 1) / ((int)gridDim.y * kWaves);
  const int first = ((int)blockIdx.y * kWaves + wave_id()) * per, last = min(rows, first + per);
  const float inv_hd = 1.0f / (float)a.hd;
  // Rows [lo, hi) of which (0 queries, 1 keys, 2 values), the first of which is row `from`.
  const auto run = [&](auto kind, int from, int lo, int hi) {
    constexpr int which = decltype(kind)::value;
    constexpr bool kTurned = which < 2;
    float gain[2][VE] = {};
    [[maybe_unused]] float dg[2][VE] = {};
    if (kTurned && in_row) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        ld_gains<T, VE>(which == 0 ? a.q_gain : a.k_gain, h * half + ch, a.gain_dtype == F32::code, gain[h]);
    }
    S* const base = static_cast<S*>(which == 0 ? a.q : which == 1 ? a.k : a.v);
    const int64_t head_stride = a.strides[which][1];
    for (int64_t t0 = (int64_t)blockIdx.x * kSlots; t0 < a.n_tok && lo < hi; t0 += (int64_t)gridDim.x * kSlots) {
      const int64_t tok = t0 + slot;
      const bool live = in_row && tok < a.n_tok;
      const int64_t b = live ? tok / a.seq : 0;
      const int t = live ? (int)(tok % a.seq) : 0;
      [[maybe_unused]] float co[VE] = {}, si[VE] = {};
      if (kTurned && live) {
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          co[e] = a.cosv[(int64_t)t * half + ch + e];
          si[e] = a.sinv[(int64_t)t * half + ch + e];
        }
      }
      S* const split = base + b * a.strides[which][0] + t * a.strides[which][2] + ch;
      const int64_t packed = tok * rows * a.hd + ch;
      for (int row = lo; row < hi; ++row) {
        const S* const x = static_cast<const S*>(a.qkv) + packed + row * a.hd;
        S* const there = split + (row - from) * head_stride;
        float u[2][VE] = {}, y[2][VE] = {};
        if (live) {
          if (BWD || !kTurned) {
            ld_part<T, VE>(BWD ? there : x, y[0]);
            ld_part<T, VE>((BWD ? there : x) + half, y[1]);
          }
          if (kTurned) {
            ld_part<T, VE>(x, u[0]);
            ld_part<T, VE>(x + half, u[1]);
          }
        }
        if constexpr (kTurned) {
          float r = head_rinv<VE, L>(u[0], u[1], inv_hd, a.eps);
          if constexpr (BWD) {
            if (!live) r = 0.0f;  // (without eps the root of nothing is infinite, and dg takes every slot's)
            float c = 0.0f;
#pragma unroll
            for (int e = 0; e < VE; ++e) turn(y[0][e], y[1][e], co[e], -si[e]);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int e = 0; e < VE; ++e) {
                u[h][e] *= r;
                const float eu = y[h][e] * u[h][e];
                dg[h][e] += eu;
                c = fmaf(gain[h][e], eu, c);
              }
            c = lane_sum<L>(c) * inv_hd;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int e = 0; e < VE; ++e) y[h][e] = r * fmaf(gain[h][e], y[h][e], -u[h][e] * c);
          } else {
#pragma unroll
            for (int e = 0; e < VE; ++e) {
              y[0][e] = u[0][e] * (r * gain[0][e]);
              y[1][e] = u[1][e] * (r * gain[1][e]);
              turn(y[0][e], y[1][e], co[e], si[e]);
            }
          }
        }
        if (!live) continue;
        S* const to = BWD ? static_cast<S*>(a.dqkv) + packed + row * a.hd : there;
        st_part<T, VE>(to, y[0]);
        st_part<T, VE>(to + half, y[1]);
      }
    }
    if constexpr (BWD && kTurned) {  // the wave's tokens, in a fixed order
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          float x = dg[h][e];
#pragma unroll
          for (int d = L; d < 64; d *= 2) x += __shfl_xor(x, d);
          if (slot == 0) fold[wave_id()][which][h][part * VE + e] = x;
        }
    }
  };
  const int keys = a.heads, values = a.heads + a.kv_heads;
  run(std::integral_constant<int, 0>{}, 0, first, min(last, keys));
  run(std::integral_constant<int, 1>{}, keys, max(first, keys), min(last, values));
  run(std::integral_constant<int, 2>{}, values, max(first, values), last);
  if constexpr (BWD) {  // then the workgroup's waves
    __syncthreads();
    const int64_t at = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
    for (int i = threadIdx.x; i < 2 * a.hd; i += kBlock) {
      const int w = i / a.hd, c = i % a.hd, h = c / half;
      float x = 0.0f;
#pragma unroll
      for (int v = 0; v < kWaves; ++v) x += fold[v][w][h][c - h * half];
      a.partial[((int64_t)w * a.rows + at) * a.hd + c] = x;
    }
  }
}

// Eight columns a workgroup, 32 strands of rows folded in order. Latency: 3.8 us for the two
// gains of 128 of those tokens.
__global__ void __launch_bounds__(kBlock)
k_head_norm_gains(const float* partial, int rows, int hd, void* dq_gain, void* dk_gain, int dtype) {
  __shared__ float fold[32][8];
  const int c0 = (int)blockIdx.x * 8, w = c0 / hd, c = c0 % hd + (threadIdx.x & 7), strand = threadIdx.x >> 3;
  const float* const p = partial + (int64_t)w * rows * hd + c;
  float x = 0.0f;
#pragma unroll 8
  for (int r = strand; r < rows; r += 32) x += p[(int64_t)r * hd];
  fold[strand][threadIdx.x & 7] = x;
  __syncthreads();
  if (strand != 0) return;
  x = 0.0f;
#pragma unroll
  for (int s = 0; s < 32; ++s) x += fold[s][threadIdx.x & 7];
  store_elem(w == 0 ? dq_gain : dk_gain, c, x, dtype);
}

// Channels a lane has of each half, and the lanes of a head.
int part_of(int hd, int dtype) { return dtype != SY_F32 && hd % 16 == 0 ? 8 : 4; }
int lanes_of(int hd, int ve) {
  int l = 1;
  while (l * ve < hd / 2) l *= 2;
  return l;
}

// Workgroups over the tokens, and over the heads where tokens alone are too few.
void grid_of(const HeadNormArgs& a, int dtype, unsigned* gx, unsigned* gy) {
  const int slots = 64 / lanes_of(a.hd, part_of(a.hd, dtype));
  const int64_t groups = (a.n_tok + slots - 1) / slots;
  *gx = (unsigned)std::min<int64_t>(groups, 2048);
  const int most = (a.heads + 2 * a.kv_heads + kWaves - 1) / kWaves;
  *gy = (unsigned)std::min<int64_t>(most, std::max<int64_t>(1, 1024 / *gx));
}

template <class T, int VE, int L>
hipError_t run_norm(const HeadNormArgs& a, hipStream_t s) {
  unsigned gx, gy;
  grid_of(a, T::code, &gx, &gy);
  if (a.dqkv != nullptr) hipLaunchKernelGGL((k_head_norm<T, VE, L, true>), dim3(gx, gy), dim3(kBlock), 0, s, a);
  else hipLaunchKernelGGL((k_head_norm<T, VE, L, false>), dim3(gx, gy), dim3(kBlock), 0, s, a);
  return hipGetLastError();
}

template <class T, int VE>
hipError_t norm_lanes(const HeadNormArgs& a, hipStream_t s) {
  switch (lanes_of(a.hd, VE)) {
    case 1: return run_norm<T, VE, 1>(a, s);
    case 2: return run_norm<T, VE, 2>(a, s);
    case 4: return run_norm<T, VE, 4>(a, s);
    case 8: return run_norm<T, VE, 8>(a, s);
    case 16: return run_norm<T, VE, 16>(a, s);
    case 32: return run_norm<T, VE, 32>(a, s);
    default: return hipErrorInvalidConfiguration;
  }
}

template <class T>
hipError_t norm_t(const HeadNormArgs& a, hipStream_t s) {
  if constexpr (T::ce == 8) {
    if (part_of(a.hd, T::code) == 8) return norm_lanes<T, 8>(a, s);
  }
  return norm_lanes<T, 4>(a, s);
}

}  // namespace

int head_norm_rows(const HeadNormArgs& a, int dtype) {
  unsigned gx, gy;
  grid_of(a, dtype, &gx, &gy);
  return (int)(gx * gy);
}

hipError_t launch_head_norm(const HeadNormArgs& a, int dtype, hipStream_t s) {
  if (dtype == SY_BF16) return norm_t<BF16>(a, s);
  if (dtype == SY_F16) return norm_t<F16>(a, s);
  return norm_t<F32>(a, s);
}

hipError_t launch_head_norm_gains(const HeadNormArgs& a, void* dq_gain, void* dk_gain, hipStream_t s) {
  hipLaunchKernelGGL(k_head_norm_gains, dim3((unsigned)(2 * a.hd / 8)), dim3(kBlock), 0, s, a.partial, a.rows, a.hd,
                     dq_gain, dk_gain, a.gain_dtype);
  return hipGetLastError();
}

}  // namespace sy
