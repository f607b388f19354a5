// Projections with 4-bit weights, and what lays such weights out.
//
//   out[m][n] = sum_k x[m][k] w[n][k],   w[n][k] = s[n][g] (c[n][k] - z[n][g]),   g = k / group
//
// with whole codes c in 0..15 and, without zero points, z = 8.
#include <algorithm>
#include <type_traits>

#include "sy_launch.hpp"

namespace sy {

namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------------- layout
//
// Tiles of 16 features by 128 columns, 1 KiB each, a feature tile's tiles one after another
// over the columns. Lane l of a wave reads 16 bytes of a tile: word j holds feature l % 16
// at columns 32 j + 8 (l / 16) + (0..7), which is what the lane brings to the matrix
// instruction over columns 32 j .. 32 j + 31. The nibble of column c of a word lies at bits
// 4 p + 3, p = c / 2 + 4 (c % 2), so one mask leaves a pair of columns in the two halves.
// Scales and zero points are [feature tile][column tile][16][groups of the tile].
constexpr int kTileK = 128;

__host__ __device__ constexpr int64_t tiles_of(int64_t n) { return (n + 15) / 16; }
__host__ __device__ constexpr int64_t steps_of(int64_t k) { return (k + kTileK - 1) / kTileK; }

// Once for a weight: 28672 x 8192 in 206 us.
__global__ void __launch_bounds__(256) k_pack4(const PackArgs a) {
  const int64_t words = tiles_of(a.n) * steps_of(a.k) * 256;
  const int64_t row_bytes = (a.k + 1) / 2;
  const int steps = (int)steps_of(a.k);
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < words; i += (int64_t)gridDim.x * 256) {
    const int j = (int)(i & 3), lane = (int)(i >> 2) & 63;
    const int64_t tile = i >> 8;
    const int64_t n = tile / steps * 16 + (lane & 15);
    const int64_t k = tile % steps * kTileK + 32 * j + 8 * (lane >> 4);
    uint32_t w = 0;
    if (n < a.n) {
      const uint8_t* const row = a.codes + n * row_bytes;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int64_t at = k / 2 + b;
        const uint32_t two = at < row_bytes ? row[at] : 0u;
        w |= (two & 15u) << (4 * b) | (two >> 4) << (4 * b + 16);
      }
    }
    a.tiles[i] = w << 3 | w >> 29;
  }
  // Groups that only pad a tile have scale zero.
  const int64_t groups = (a.k + a.group - 1) / a.group;
  const int ng = kTileK / a.group;
  const int64_t cells = tiles_of(a.n) * steps * 16 * ng;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < cells; i += (int64_t)gridDim.x * 256) {
    const int64_t tile = i / ng >> 4;
    const int64_t n = tile / steps * 16 + (i / ng & 15), g = tile % steps * ng + i % ng;
    const bool in = n < a.n && g < groups;
    if (a.esize == 4)
      static_cast<uint32_t*>(a.scales_out)[i] = in ? static_cast<const uint32_t*>(a.scales)[n * groups + g] : 0u;
    else
      static_cast<uint16_t*>(a.scales_out)[i] = in ? static_cast<const uint16_t*>(a.scales)[n * groups + g] : (uint16_t)0;
    if (a.zeros != nullptr) a.zeros_out[i] = in ? a.zeros[n * groups + g] : (uint8_t)0;
  }
}

// Rounding to codes: sixteen lanes a group, each with group / 16 neighbours. Symmetric: s =
// max |w| / 7, c = round(w / s) + 8 (1 to 15); with zero points s = (max - min) / 15 over a
// range that holds zero, z = round(-min / s), c = round(w / s) + z. s is rounded to the
// weights' type first, so the codes fit the scale that is kept; where that leaves the group's ends
// half a step or more outside the codes (s a few of the type's smallest steps, or 0) s is the next
// number up. A group of zeros has s = 0, one with an infinity or NaN s = NaN, which its products
// show (minima and maxima pass over NaN).
// Once for a weight too: 28672 x 8192 in bf16 in 380 us, 1.5 TB/s.
template <class T, int E>
__global__ void __launch_bounds__(256) k_quantize4(const QuantizeArgs a) {
  using S = typename T::storage;
  const int64_t groups = (a.k + a.group - 1) / a.group, items = a.n * groups;
  const int sub = threadIdx.x & 15;
  for (int64_t i0 = (int64_t)blockIdx.x * 16; i0 < items; i0 += (int64_t)gridDim.x * 16) {
    const int64_t i = i0 + (threadIdx.x >> 4);
    const bool live = i < items;
    const int64_t n = live ? i / groups : 0, g = live ? i % groups : 0;
    const int64_t k0 = g * a.group + sub * E;
    const S* const row = static_cast<const S*>(a.w) + n * a.row_stride;
    float w[E], lo = 0.0f, hi = 0.0f;
    float sum = 0.0f;  // NaN where one of them is
#pragma unroll
    for (int e = 0; e < E; ++e) {
      w[e] = live && k0 + e < a.k ? load_elem(row, k0 + e, T::code) : 0.0f;
      sum += w[e];
      lo = fminf(lo, w[e]);
      hi = fmaxf(hi, w[e]);
    }
#pragma unroll
    for (int d = 1; d < 16; d *= 2) {
      lo = fminf(lo, __shfl_xor(lo, d, 16));
      hi = fmaxf(hi, __shfl_xor(hi, d, 16));
    }
    const float range = a.zeros != nullptr ? hi - lo : fmaxf(hi, -lo), spans = a.zeros != nullptr ? 15.0f : 7.0f;
    float f[T::ce] = {isfinite(range) ? range / spans : hi / spans - lo / spans};  // (hi - lo may be past fp32)
    if ((__ballot(sum != sum) >> (threadIdx.x & 48) & 0xffff) != 0 || isinf(hi) || isinf(lo))
      f[0] = __int_as_float(0x7fc00000);
    i32x4_t kept = pack<T>(f);
    constexpr float kNormal = T::code == F16::code ? 0x1p-14f : 0x1p-126f;  // (above, roundings are too small for it)
    if (range > 0.0f && elem<T>(kept, 0) < kNormal && range / elem<T>(kept, 0) >= spans + 0.5f)
      ++kept[0];  // (the other elements are 0)
    const float s = elem<T>(kept, 0);
    const auto steps_in = [s](float x) { return s > 0.0f ? rintf(x / s) : 0.0f; };
    const float z = a.zeros != nullptr ? fminf(fmaxf(steps_in(-lo), 0.0f), 15.0f) : 8.0f;
    if (!live) continue;
    if (sub == 0) {
      __builtin_memcpy(static_cast<S*>(a.scales) + i, &kept, sizeof(S));
      if (a.zeros != nullptr) a.zeros[i] = (uint8_t)z;
    }
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      if (k0 + e >= a.k) break;
      uint32_t c[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) c[h] = (uint32_t)fminf(fmaxf(steps_in(w[e + h]) + z, 0.0f), 15.0f);
      a.codes[n * ((a.k + 1) / 2) + (k0 + e) / 2] = (uint8_t)(c[0] | c[1] << 4);
    }
  }
}

// ------------------------------------------------------------------ product
//
// Products run on v_mfma_f32_16x16x32 with sixteen rows of x against sixteen features. A code
// becomes 1 + c / 16 in x's type by putting its four bits at the top of the mantissa of 1.0: a
// shift, a mask and an or for two weights, and exact. So is every product with x, and
//
//   sum_k x (c - z) / 16 = sum_k x (1 + c / 16) - (1 + z / 16) sum_k x
//
// over a group; the last sum comes from the same instruction against a constant, and is what
// the accumulator starts from. Group sums are scaled and added in fp32: nothing is rounded to
// fewer bits before the output.
//
// fp32 rows are taken as three bf16 numbers of eight bits each, which hold all 24, and codes as
// the bf16 numbers c - z, in twice the instructions: both sums above are several times the
// result, and their roundings show in 24 bits (5 rows of 1407 x 2001: 5.5e-7 off in the norm, with
// c - z 1.1e-7).
template <class T> struct Mma;
template <> struct Mma<BF16> {
  static constexpr int planes = 1;
  static constexpr uint32_t one = 0x3f803f80u, mask = 0x00780078u;
  static __device__ __forceinline__ f32x4_t run(const i32x4_t& a, const i32x4_t& b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c,
                                                   0, 0, 0);
  }
};
template <> struct Mma<F16> {
  static constexpr int planes = 1;
  static constexpr uint32_t one = 0x3c003c00u, mask = 0x03c003c0u;
  static __device__ __forceinline__ f32x4_t run(const i32x4_t& a, const i32x4_t& b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0,
                                                  0, 0);
  }
};
template <> struct Mma<F32> : Mma<BF16> {
  static constexpr int planes = 3;
};

__device__ __forceinline__ uint32_t ror(uint32_t x, int n) { return __builtin_amdgcn_alignbit(x, x, n); }

// The eight weights of a word as 1 + c / 16. Mask and one are held in registers, opaque to the
// compiler, which else takes them as literals and splits each and-or in two (2048 rows of 2048 x
// 5632 so take 2% less time, 32 of 11264 x 2048 5%).
template <class T> struct Codes {
  static constexpr float unit = 16.0f;  // of the sums
  uint32_t mask = Mma<T>::mask, one = Mma<T>::one;
  __device__ __forceinline__ Codes() { asm("" : "+v"(mask), "+v"(one)); }
  __device__ __forceinline__ i32x4_t operator()(uint32_t w, float) const {
    i32x4_t r;
    if constexpr (T::code == F16::code) {
      r[0] = (int)((w << 3 & mask) | one);
      r[1] = (int)((w >> 1 & mask) | one);
      r[2] = (int)((w >> 5 & mask) | one);
      r[3] = (int)((ror(w, 9) & mask) | one);
    } else {
      r[0] = (int)((w & mask) | one);
      r[1] = (int)((w >> 4 & mask) | one);
      r[2] = (int)((w >> 8 & mask) | one);
      r[3] = (int)((ror(w, 12) & mask) | one);
    }
    return r;
  }
};

// c - z for fp32 rows.
template <> struct Codes<F32> {
  static constexpr float unit = 1.0f;
  __device__ __forceinline__ i32x4_t operator()(uint32_t w, float z) const {
    const uint32_t v = ror(w, 3), half[2] = {v & 0x0f0f0f0fu, v >> 4 & 0x0f0f0f0fu};
    i32x4_t r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t x = half[i & 1] >> (8 * (i >> 1));
      const float lo = (float)(x & 0xffu) - z, hi = (float)(x >> 16 & 0xffu) - z;
      r[i] = (int)__builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
    }
    return r;
  }
};

// -1, or -1.5 = -(1 + 8 / 16), in every element: what the sum over x is taken against.
template <class T, bool ZEROS> __device__ __forceinline__ i32x4_t minus() {
  constexpr uint32_t x = 0x80008000u | Mma<T>::one | (ZEROS ? 0u : T::code == F16::code ? 0x02000200u : 0x00400040u);
  return i32x4_t{(int)x, (int)x, (int)x, (int)x};
}


// 16 bytes of a row from column k on; WHOLE: all are before k_end, else those behind it are
// zero. Rows start anywhere.
template <class T, bool WHOLE>
__device__ __forceinline__ i32x4_t ld_x(const typename T::storage* row, int k, int k_end) {
  if (WHOLE) return *reinterpret_cast<const i32x4_any_t*>(row + k);
  i32x4_t r = {0, 0, 0, 0};
  if constexpr (T::ce == 4) {
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = k + e < k_end ? __float_as_int(row[k + e]) : 0;
  } else {
    // The row's last eight, with those before k shifted out.
    typedef uint64_t u64x2_t __attribute__((ext_vector_type(2)));
    u64x2_t x = {0, 0};
    int past = k - (k_end - 8);
    if (k_end >= 8) {
      const i32x4_t y = *reinterpret_cast<const i32x4_any_t*>(row + min(k, k_end - 8));
      x = __builtin_bit_cast(u64x2_t, y);
    } else {  // a row of fewer
      past = k;
#pragma unroll 1
      for (int e = k_end - 1; e >= 0; --e) {
        x[1] = x[1] << 16 | x[0] >> 48;
        x[0] = x[0] << 16 | row[e];
      }
    }
    if (past > 0) {
      const int bits = 16 * (past & 3);
      if (past & 4) x = u64x2_t{x[1], 0};
      if (bits != 0) x = u64x2_t{x[0] >> bits | x[1] << (64 - bits), x[1] >> bits};
      if (past >= 8) x = u64x2_t{0, 0};
    }
    r = __builtin_bit_cast(i32x4_t, x);
  }
  return r;
}

// Eight elements of a row.
template <class T> struct Raw {
  static constexpr int words = 8 / T::ce;
  i32x4_t x[words];
};

// Its fragments: itself, or the three bf16 parts of each element.
template <class T> __device__ __forceinline__ void parts_of(const Raw<T>& r, i32x4_t (&f)[Mma<T>::planes]) {
  if constexpr (Raw<T>::words == 1) {
    f[0] = r.x[0];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) x[h] = __int_as_float(r.x[(2 * i + h) / 4][(2 * i + h) % 4]);
#pragma unroll
      for (int p = 0; p < 3; ++p) {
        const uint32_t a = __float_as_uint(x[0]), b = __float_as_uint(x[1]);
        f[p][i] = (int)((b & 0xffff0000u) | a >> 16);
        x[0] -= __uint_as_float(a & 0xffff0000u);
        x[1] -= __uint_as_float(b & 0xffff0000u);
      }
    }
  }
}

// The N scales and zero points of a column in a tile, in one load each.
template <class T, int N> __device__ __forceinline__ void ld_scales(const typename T::storage* p, float (&s)[N]) {
  typename T::storage raw[N];
  __builtin_memcpy(raw, __builtin_assume_aligned(p, N * sizeof(raw[0])), sizeof(raw));
#pragma unroll
  for (int g = 0; g < N; ++g) s[g] = load_elem(raw, g, T::code);
}
template <class T, int N> __device__ __forceinline__ void ld_zeros(const uint8_t* p, float (&z)[N]) {
  uint8_t raw[N];
  __builtin_memcpy(raw, __builtin_assume_aligned(p, N), sizeof(raw));
#pragma unroll
  for (int g = 0; g < N; ++g) z[g] = T::code == F32::code ? (float)raw[g] : 1.0f + (float)raw[g] * 0.0625f;
}

// What a wave needs of one column tile.
template <class T, int MT, int NT, int NG, bool ZEROS> struct Step {
  i32x4_t w[NT];
  float s[NT][NG], z[NT][NG];
  Raw<T> x[MT][4];
};

// A workgroup has NT feature tiles and 16 MT rows; its waves share the columns out tile by tile
// and fold their sums in LDS in their order. GS: 32-column pieces of a group. The weights' bytes
// bound it where there are many: 16 rows of 28672 x 8192 29.3 us, 4.2 TB/s (its waves wait half
// their time, the vector units work 43% of it), 8 rows of 32000 x 2048 8.2, 4.2; else latency, 1 row
// of 6144 x 2048 3.7 where launches follow one another. More waves, a wave's next tile asked for
// ahead, loads past the caches and other orders of the columns gained nothing over all shapes. (32
// rows by 64 features are bound to two waves a SIMD: with the registers of three the compiler asks
// for less at a time, and 32 rows of 28672 x 8192 take 1.4 times as long.)
template <class T, int MT, int NT, int WAVES, bool STAGED, int GS, bool ZEROS>
__global__ void __launch_bounds__(64 * WAVES < 512 ? 512 : 64 * WAVES)
__attribute__((amdgpu_waves_per_eu(WAVES < 16 ? 2 : 4, MT * NT == 8 ? 2 : 8))) k_linear4(const Linear4Args a) {
  using S = typename T::storage;
  constexpr int P = Mma<T>::planes, NG = 4 / GS;
  extern __shared__ float fold[];
  const int lane = threadIdx.x & 63, wave = wave_id(), waves = blockDim.x >> 6;
  const int col = lane & 15, quad = lane >> 4;
  const int64_t tile0 = (int64_t)blockIdx.x * NT, n_tiles = tiles_of(a.n);
  const int steps = (int)steps_of(a.k);
  const int64_t m0 = (int64_t)blockIdx.y * (16 * MT);
  // Rows behind the last are the last one's again: their sums are not stored. STAGED: a load is
  // whole rows of a tile, four of 256 bytes or two of 512, which go through LDS to the lanes
  // that need them.
  constexpr int W = Raw<T>::words, kChunks = kTileK / T::ce, kLoads = kChunks / 4;  // of a row, and of 16 rows
  const int r0 = lane / kChunks, c0 = lane % kChunks;
  const S* rows[MT][STAGED ? kLoads : 1];
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int j = 0; j < (STAGED ? kLoads : 1); ++j)
      rows[t][j] = static_cast<const S*>(a.x) +
                   min(m0 + 16 * t + (STAGED ? 16 / kLoads * j + r0 : col), a.m - 1) * a.x_stride;
  i32x4_t* const stage = reinterpret_cast<i32x4_t*>(fold) + wave * (MT * 16 * kChunks);
  const i32x4_t neg = minus<T, ZEROS>();
  const Codes<T> codes;
  f32x4_t tot[MT][NT];
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int u = 0; u < NT; ++u) tot[t][u] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  // Where the feature tiles begin (those behind the last are the last one: not stored either).
  const char *w_at[NT], *s_at[NT], *z_at[NT];
#pragma unroll
  for (int u = 0; u < NT; ++u) {
    const int64_t tile = min(tile0 + u, n_tiles - 1) * steps;
    w_at[u] = reinterpret_cast<const char*>(a.tiles) + tile * 1024;
    s_at[u] = static_cast<const char*>(a.scales) + tile * (16 * NG * (int)sizeof(S));
    if constexpr (ZEROS) z_at[u] = reinterpret_cast<const char*>(a.zeros) + tile * (16 * NG);
  }
  using Tile = Step<T, MT, NT, NG, ZEROS>;
  const auto load = [&](int step, Tile& r, auto whole) {
    const uint32_t cell = (uint32_t)(step * 16 + col) * NG;
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      r.w[u] = *reinterpret_cast<const i32x4_t*>(w_at[u] + (uint32_t)(step * 1024 + lane * 16));
      ld_scales<T, NG>(reinterpret_cast<const S*>(s_at[u] + cell * (uint32_t)sizeof(S)), r.s[u]);
      if constexpr (ZEROS) ld_zeros<T, NG>(reinterpret_cast<const uint8_t*>(z_at[u] + cell), r.z[u]);
    }
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const int k = step * kTileK + (STAGED ? T::ce * c0 : 32 * (j / W) + 8 * quad + T::ce * (j % W));
        r.x[t][j / W].x[j % W] = ld_x<T, decltype(whole)::value>(rows[t][STAGED ? j : 0], k, a.k);
      }
  };
  const auto add = [&](const Tile& r) {
    i32x4_t f[MT][4][P];
    if constexpr (STAGED) {
      // Chunk c of a row lies at c ^ row: neither side has two lanes on a bank. (Only this wave
      // reads what it wrote.)
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
          const int row = 16 / kLoads * j + r0;
          stage[(t * 16 + row) * kChunks + (c0 ^ row)] = r.x[t][j / W].x[j % W];
        }
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          Raw<T> x;
#pragma unroll
          for (int i = 0; i < W; ++i) x.x[i] = stage[(t * 16 + col) * kChunks + (((4 * j + quad) * W + i) ^ col)];
          parts_of<T>(x, f[t][j]);
        }
      __builtin_amdgcn_wave_barrier();
    } else {
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) parts_of<T>(r.x[t][j], f[t][j]);
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      f32x4_t sums[MT];
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        sums[t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        if constexpr (P == 1) {
#pragma unroll
          for (int j = g * GS; j < (g + 1) * GS; ++j) sums[t] = Mma<T>::run(f[t][j][0], neg, sums[t]);
        }
      }
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        f32x4_t acc[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[t] = ZEROS && P == 1 ? sums[t] * r.z[u][g] : sums[t];
#pragma unroll
        for (int j = g * GS; j < (g + 1) * GS; ++j) {
          const i32x4_t c = codes((uint32_t)r.w[u][j], ZEROS ? r.z[u][g] : 8.0f);
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int p = 0; p < P; ++p) acc[t] = Mma<T>::run(f[t][j][p], c, acc[t]);
        }
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) tot[t][u][i] = fmaf(r.s[u][g], acc[t][i], tot[t][u][i]);
      }
    }
  };
  // Whole tiles, then the rest.
  const int full = a.k / kTileK;
  Tile r;
  for (int step = wave; step < full; step += waves) {
    load(step, r, std::true_type{});
    add(r);
  }
  if (full < steps && full % waves == wave) {
    load(full, r, std::false_type{});
    add(r);
  }
  constexpr int kSums = MT * NT * 256;
  if constexpr (STAGED) __syncthreads();  // (the sums go where the waves' rows were)
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) fold[wave * kSums + ((t * NT + u) * 4 + i) * 64 + lane] = tot[t][u][i];
  __syncthreads();
  S* const out = static_cast<S*>(a.out);
  for (int i = threadIdx.x; i < kSums; i += blockDim.x) {
    float y = 0.0f;
    for (int v = 0; v < waves; ++v) y += fold[v * kSums + i];
    const int l = i & 63, r = i >> 6 & 3, u = (i >> 8) % NT, t = (i >> 8) / NT;
    const int64_t m = m0 + 16 * t + 4 * (l >> 4) + r, n = (tile0 + u) * 16 + (l & 15);
    if (m < a.m && n < a.n) store_elem(out, m * a.n + n, Codes<T>::unit * y, T::code);
  }
}

// The sum of a chunk's eight elements, added to acc.
template <class T> __device__ __forceinline__ float sum8(const i32x4_t& x, float acc) {
  constexpr int one = (int)Mma<T>::one;
  return dot<T>(x, i32x4_t{one, one, one, one}, acc);
}

// 16 bytes a lane from memory to LDS, lane i's at byte `at` + 16 i of the workgroup's LDS; done
// when vmcnt says so. The compiler does not count these loads: a wait of its own for an earlier
// one would wait for them too.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_to_lds(const void* from, uint32_t at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(at), "v"(from) : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ __forceinline__ uint32_t lds_byte(void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)p;
}

// N bytes, 1 to 8, as they lie in memory.
template <int N> struct Bytes {
  uint32_t w[(N + 3) / 4];
  __device__ __forceinline__ void load(const char* p) {
    if constexpr (N == 1) w[0] = *reinterpret_cast<const uint8_t*>(p);
    else if constexpr (N == 2) w[0] = *reinterpret_cast<const uint16_t*>(p);
    else __builtin_memcpy(w, __builtin_assume_aligned(p, N), N);
  }
  __device__ __forceinline__ void wait() {
#pragma unroll
    for (uint32_t& x : w) asm volatile("" : "+v"(x));
  }
  __device__ __forceinline__ uint32_t half(int i) const { return w[i / 2] >> (16 * (i % 2)) & 0xffffu; }
  __device__ __forceinline__ uint32_t byte(int i) const { return w[i / 4] >> (8 * (i % 4)) & 0xffu; }
};

// Many rows: a workgroup has 64 rows by 64 NT features. Four waves with NT feature tiles each
// share a column tile of the rows in LDS, double-buffered; with PARTS 2, two such groups of
// waves take every other column tile and add up at the end. A tile's sums over each group's
// columns are formed where it is written to LDS, by the lanes that hold it; DIRECT: the tile goes
// straight to LDS, for which rows start at 16-byte boundaries, and each wave takes the sums off
// the matrix units (512 rows of 2048 x 5632 so take 9% less time, 4096 of 11264 x 2048 4%, 2048 of
// 2048 x 5632 1%: 24.2, 221 and 55.8 us). Vector instructions bound it, next to waits: the last of
// those is 847 TFLOP/s; codes to numbers and scaling are a third of them each. The library's
// product with bf16 weights takes 54.5.
template <class T, int NT, int PARTS, bool DIRECT, int GS, bool ZEROS>
__global__ void __launch_bounds__(256 * PARTS) __attribute__((amdgpu_waves_per_eu(2)))
k_linear4_many(const Linear4Args a, int n_blocks, int blocks) {
  using S = typename T::storage;
  constexpr int NG = 4 / GS, MT = 4, kRows = 16 * MT, kChunks = kRows * 16;
  __shared__ __align__(16) i32x4_t stage[PARTS][2][kChunks];
  __shared__ __align__(16) float sums[PARTS][2][NG][kRows];  // (not DIRECT)
  static_assert(PARTS == 1 || sizeof(stage) >= 4 * MT * NT * 1024, "the second group's sums fit");
  // Neighbouring blocks on one XCD: workgroups go to the eight of them in turn.
  const int per = (blocks + 7) / 8, block = (int)(blockIdx.x % 8) * per + (int)(blockIdx.x / 8);
  if ((int)(blockIdx.x / 8) >= per || block >= blocks) return;
  const int lane = threadIdx.x & 63, wave = wave_id(), part = wave >> 2;
  const int col = lane & 15, quad = lane >> 4;
  const int64_t n_tiles = tiles_of(a.n), m0 = (int64_t)(block / n_blocks) * kRows;
  const int64_t tile0 = ((int64_t)(block % n_blocks) * 4 + (wave & 3)) * NT;
  const int steps = (int)steps_of(a.k);
  const Codes<T> codes;
  // A thread of a group loads four chunks of the tile: rows r0, r0 + 16, r0 + 32, r0 + 48.
  const int r0 = threadIdx.x >> 4 & 15, c0 = threadIdx.x & 15;
  const S* rows[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) rows[i] = static_cast<const S*>(a.x) + min(m0 + r0 + 16 * i, a.m - 1) * a.x_stride;
  const char *w_at[NT], *s_at[NT], *z_at[NT];
#pragma unroll
  for (int u = 0; u < NT; ++u) {
    const int64_t tile = min(tile0 + u, n_tiles - 1) * steps;
    w_at[u] = reinterpret_cast<const char*>(a.tiles) + tile * 1024;
    s_at[u] = static_cast<const char*>(a.scales) + tile * (16 * NG * (int)sizeof(S));
    if constexpr (ZEROS) z_at[u] = reinterpret_cast<const char*>(a.zeros) + tile * (16 * NG);
  }
  struct Weights {
    i32x4_t w[NT];
    Bytes<NG * (int)sizeof(S)> s[NT];
    Bytes<NG> z[NT];
  };
  const auto load_w = [&](int step, Weights& r) {
    const uint32_t cell = (uint32_t)(step * 16 + col) * NG;
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      r.w[u] = *reinterpret_cast<const i32x4_t*>(w_at[u] + (uint32_t)(step * 1024 + lane * 16));
      r.s[u].load(s_at[u] + cell * (uint32_t)sizeof(S));
      if constexpr (ZEROS) r.z[u].load(z_at[u] + cell);
    }
  };
  const auto load_x = [&](int step, i32x4_t (&x)[MT]) {
    const int k = step * kTileK + 8 * c0;
    if ((step + 1) * kTileK <= a.k) {
#pragma unroll
      for (int i = 0; i < MT; ++i) x[i] = ld_x<T, true>(rows[i], k, a.k);
    } else {
#pragma unroll
      for (int i = 0; i < MT; ++i) x[i] = ld_x<T, false>(rows[i], k, a.k);
    }
  };
  const auto put = [&](int buffer, const i32x4_t (&x)[MT]) {
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      stage[part][buffer][(r0 + 16 * i) * 16 + (c0 ^ r0)] = x[i];
      if (DIRECT) continue;
      const float s = lane_sum<4 * GS>(sum8<T>(x[i], 0.0f)) * (ZEROS ? -1.0f : -1.5f);
      if (c0 % (4 * GS) == 0) sums[part][buffer][c0 / (4 * GS)][r0 + 16 * i] = s;
    }
  };
  f32x4_t tot[MT][NT];
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int u = 0; u < NT; ++u) tot[t][u] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  const auto add = [&](int buffer, const Weights& r) {
    const i32x4_t* const at = stage[part][buffer] + col * 16;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      i32x4_t f[GS][MT];
      f32x4_t from[MT];
#pragma unroll
      for (int t = 0; t < MT; ++t)
        from[t] = DIRECT ? f32x4_t{0.0f, 0.0f, 0.0f, 0.0f}
                         : *reinterpret_cast<const f32x4_t*>(&sums[part][buffer][g][16 * t + 4 * quad]);
#pragma unroll
      for (int j = 0; j < GS; ++j)
#pragma unroll
        for (int t = 0; t < MT; ++t) f[j][t] = at[t * 256 + ((4 * (g * GS + j) + quad) ^ col)];
      if constexpr (DIRECT) {
#pragma unroll
        for (int j = 0; j < GS; ++j)
#pragma unroll
          for (int t = 0; t < MT; ++t) from[t] = Mma<T>::run(f[j][t], minus<T, ZEROS>(), from[t]);
      }
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        f32x4_t acc[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[t] = ZEROS ? from[t] * (1.0f + (float)r.z[u].byte(g) * 0.0625f) : from[t];
#pragma unroll
        for (int j = 0; j < GS; ++j) {
          const i32x4_t c = codes((uint32_t)r.w[u][g * GS + j], 0.0f);
#pragma unroll
          for (int t = 0; t < MT; ++t) acc[t] = Mma<T>::run(f[j][t], c, acc[t]);
        }
        const S raw = (S)r.s[u].half(g);
        const float s = load_elem(&raw, 0, T::code);
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) tot[t][u][i] = fmaf(s, acc[t][i], tot[t][u][i]);
      }
    }
  };
  // Both groups go round as often; one may have nothing to add in the last round.
  const int last = steps - 1, rounds = (steps + PARTS - 1) / PARTS;
  i32x4_t x[MT];
  Weights w, next;
  // A column tile to LDS, straight where all of it is there.
  const uint32_t stage_at = lds_byte(&stage[part][0][(wave & 3) * 64]);
  const auto fill = [&](int step, int buffer) {
    if ((step + 1) * kTileK <= a.k) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
        load_to_lds(rows[i] + step * kTileK + 8 * (c0 ^ r0),
                    __builtin_amdgcn_readfirstlane(stage_at + (buffer * kChunks + i * 256) * 16));
    } else {
      load_x(step, x);
      put(buffer, x);
    }
  };
  const auto landed = [&](Weights& r) {
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      asm volatile("" : "+v"(r.w[u]));
      r.s[u].wait();
      if constexpr (ZEROS) r.z[u].wait();
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  };
  load_w(min(part, last), w);
  if constexpr (DIRECT) {
    fill(min(part, last), 0);
    landed(w);
  } else {
    load_x(min(part, last), x);
    put(0, x);
  }
  __syncthreads();
  const auto round = [&](int i, const Weights& now, Weights& then) {
    const int step = PARTS * i + part, at = min(step + PARTS, last);
    load_w(at, then);
    if constexpr (DIRECT) {
      fill(at, (i + 1) & 1);
      if (step <= last) add(i & 1, now);
      landed(then);
    } else {
      load_x(at, x);
      if (step <= last) add(i & 1, now);
      put((i + 1) & 1, x);
    }
    __syncthreads();
  };
  for (int i = 0; i < rounds; i += 2) {
    round(i, w, next);
    if (i + 1 < rounds) round(i + 1, next, w);
  }
  // The second group's sums to the first, a lane's own.
  float* const mine = reinterpret_cast<float*>(stage) + (wave & 3) * (MT * NT * 256) + lane;
  if constexpr (PARTS == 2) {
    if (part == 1) {
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int u = 0; u < NT; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) mine[((t * NT + u) * 4 + i) * 64] = tot[t][u][i];
    }
    __syncthreads();
    if (part == 1) return;
  }
  S* const out = static_cast<S*>(a.out);
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t m = m0 + 16 * t + 4 * quad + i, n = (tile0 + u) * 16 + col;
        if (m < a.m && n < a.n)
          store_elem(out, m * a.n + n, Codes<T>::unit * (PARTS == 2 ? tot[t][u][i] + mine[((t * NT + u) * 4 + i) * 64] : tot[t][u][i]),
                     T::code);
      }
}

template <class T, int NT, int PARTS, bool DIRECT, int GS, bool ZEROS>
hipError_t run4_direct(const Linear4Args& a, hipStream_t s) {
  const int n_blocks = (int)((tiles_of(a.n) + 4 * NT - 1) / (4 * NT));  // (at most 2^18)
  const int64_t rows = 64 * ((1 << 21) / n_blocks);  // of a launch: 2^30 threads
  for (int64_t m0 = 0; m0 < a.m; m0 += rows) {
    Linear4Args part = a;
    part.m = std::min(rows, a.m - m0);
    const int64_t es = sizeof(typename T::storage);
    part.x = static_cast<const char*>(a.x) + m0 * a.x_stride * es;
    part.out = static_cast<char*>(a.out) + m0 * a.n * es;
    const int blocks = (int)((part.m + 63) / 64) * n_blocks;
    hipLaunchKernelGGL((k_linear4_many<T, NT, PARTS, DIRECT, GS, ZEROS>), dim3((unsigned)(blocks + 7) / 8 * 8), dim3(256 * PARTS), 0, s,
                       part, n_blocks, blocks);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <class T, int MT, int NT, int WAVES, bool STAGED, int GS, bool ZEROS>
hipError_t run4(const Linear4Args& a, hipStream_t s) {
  const int steps = (int)steps_of(a.k);
  int waves = WAVES;
  while (waves > 1 && waves > steps) waves /= 2;
  const unsigned gx = (unsigned)((tiles_of(a.n) + NT - 1) / NT);
  constexpr int kRows16 = T::ce == 8 ? 4 : 8;  // KiB of a column tile of 16 rows
  const int lds = waves * MT * (STAGED ? std::max(kRows16, NT) : NT) * 1024;
  static_assert(WAVES * MT * NT <= 64 && (!STAGED || WAVES * MT * kRows16 <= 64), "at most 64 KiB of LDS");
  constexpr int64_t kRows = 16 * MT * 256;  // of a launch: at most 2^28 workgroups
  for (int64_t m0 = 0; m0 < a.m; m0 += kRows) {
    Linear4Args part = a;
    part.m = std::min(kRows, a.m - m0);
    const int64_t es = sizeof(typename T::storage);
    part.x = static_cast<const char*>(a.x) + m0 * a.x_stride * es;
    part.out = static_cast<char*>(a.out) + m0 * a.n * es;
    const unsigned gy = (unsigned)((part.m + 16 * MT - 1) / (16 * MT));
    hipLaunchKernelGGL((k_linear4<T, MT, NT, WAVES, STAGED, GS, ZEROS>), dim3(gx, gy), dim3(64 * waves), lds, s,
                       part);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <class T, int NT, int PARTS, int GS, bool ZEROS>
hipError_t run4_many(const Linear4Args& a, hipStream_t s) {
  const bool direct = reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && a.x_stride % 8 == 0;
  return direct ? run4_direct<T, NT, PARTS, true, GS, ZEROS>(a, s) : run4_direct<T, NT, PARTS, false, GS, ZEROS>(a, s);
}

// The kernel and its tile by rows and feature tiles; us on both sides, bf16 unless stated, of the
// sweep that the costs were fitted to (captured launches on one machine; others are up to 6% off).
//   up to 16         straight from memory with one or two feature tiles, where a load's lanes touch
//                    few lines, or through LDS with one, two or four, by the costs below. In their
//                    order: 1 row of 6144 x 2048 3.5, 3.6, and 4.0 at best through LDS; 8 of 2048 x
//                    5632 5.7, 7.0, 4.6, 5.5, 7.8; of 32000 x 2048 12.4, 8.9, 15.7, 9.4, 10.5; 16 of
//                    28672 x 8192 56, 41, 49, 32.7, 29.5; 9 of 17951 x 1092 6.4, 5.1, 7.5, 7.4, 8.8.
//                    Of 296 shapes the choice takes 3% longer than the best on average, 43% at most.
//                    More than one row at odd places goes through LDS: 8 rows of 9055 x 3715 8.5,
//                    straight 22.
//                    fp32 up to 8 rows straight from memory, two feature tiles from 256 on: 1 row of
//                    6144 x 2048 6.0, one 7.2; 5 of 1408 x 2048 6.1, one 4.9.
//   more             16 or 32 rows a workgroup through LDS, or 64 with one or two groups of waves,
//                    whichever the costs below say is done first. In their order: 32 rows of 2048 x
//                    5632 5.1, 6.2, 7.9, 10.5, of the last four 21 at best; 24 of 28672 x 8192 79,
//                    49, 49, 39, 54 at best; 128 of 6144 x 2048 23, 12.2, 12.4, 13.8, 22.3, 23.4,
//                    15.1, 11.3; 256 of 11264 x 2048 73, 36, 40, 36, 24.2, 24.2, 27.3, 25.0; 2048 of
//                    2048 x 5632 57.5, 62.1, 68.8 and 81.2 with the last four. Of 207 shapes (17 to
//                    1400 rows, 300 to 30000 features, 200 to 9000 columns, groups of 64 and 128)
//                    the choice takes 2% longer than the best on average, 38% at most.
//   fp32 past 8      through LDS, 16 rows a workgroup, and up to four feature tiles: 16 rows of 2048
//                    x 5632 11.2 with one, 14.2 with two, 19.7 with four, 12.6 straight; 64 of 2048
//                    x 2048 8.7, 7.3, 9.3, 10.6; 16 of 11264 x 2048 11.6, 11.1, 10.3, 15.3. 32 rows
//                    and four feature tiles where all CUs have work and every wave a few column
//                    tiles: 2048 rows of 2048 x 5632 200, 16 rows 296; 512 of 2048 x 2048 26, 36;
//                    but 128 of 2048 x 5632 38, 20, and 239 of 22848 x 704 73, 63.

// A launch's time in us, fitted to those shapes on 256 CUs: base + step (column tiles + more) for
// each round of up to 512 workgroups that fill the CUs twice over; the last counts as 1 / full of
// that if there are 256 in it or fewer. Up to 16 rows the smaller workgroups fill in evenly, and
// each row adds its part of a step.
struct Cost {
  int rows, tiles;  // of a workgroup
  double base, step, more, full, row;
  double of(int64_t m, int64_t n_tiles, int steps) const {
    const int64_t blocks = (m + rows - 1) / rows * ((n_tiles + tiles - 1) / tiles), rest = blocks % 512;
    return base + step * (steps + more) * ((double)(blocks / 512) * full + (rest > 256 ? full : rest > 0 ? 1.0 : 0.0));
  }
  double few(int64_t m, int64_t n_tiles, int steps) const {
    const int64_t blocks = (n_tiles + tiles - 1) / tiles;
    return base + step * (steps + more) * (1.0 + row * (double)m) *
                      (blocks <= 256 ? 1.0 : 1.0 + (full - 1.0) * (double)(blocks - 256) / 256.0);
  }
};
constexpr Cost kCosts[] = {{16, 1, 3.0, 0.056, 1.0, 3.2, 0.0}, {16, 2, 2.8, 0.099, 4.0, 1.8, 0.0},
                           {16, 4, 3.4, 0.14, 4.0, 2.3, 0.0},  {32, 4, 3.1, 0.20, 9.0, 2.3, 0.0},
                           {64, 16, 0.5, 1.1, 7.0, 2.1, 0.0},  {64, 16, 4.0, 1.2, 3.0, 1.7, 0.0},
                           {64, 8, 0.5, 0.69, 8.0, 1.9, 0.0},  {64, 4, 2.5, 0.45, 6.0, 1.8, 0.0}};
// Two that take rows straight from memory, three through LDS.
constexpr Cost kFewCosts[] = {{16, 1, 2.6, 0.039, 0.0, 2.3, 0.085}, {16, 2, 2.4, 0.085, 2.0, 2.0, 0.036},
                              {16, 1, 3.1, 0.041, 0.0, 3.2, 0.012}, {16, 2, 2.6, 0.096, 3.0, 2.1, 0.011},
                              {16, 4, 3.4, 0.13, 3.0, 3.3, 0.007}};
template <class F>
int cheapest(const Cost* costs, int from, int to, const F& us) {
  int best = from;
  double least = us(costs[from]);
  for (int i = from + 1; i < to; ++i) {
    const double x = us(costs[i]);
    if (x < least) best = i, least = x;
  }
  return best;
}

template <class T, int GS, bool ZEROS>
hipError_t linear4_m(const Linear4Args& a, hipStream_t s) {
  const int64_t tiles = tiles_of(a.n);
  if constexpr (T::code == F32::code) {
    if (a.m <= 8)
      return tiles >= 256 ? run4<T, 1, 2, 8, false, GS, ZEROS>(a, s) : run4<T, 1, 1, 8, false, GS, ZEROS>(a, s);
    const int64_t blocks = tiles * ((a.m + 15) / 16);
    if (steps_of(a.k) >= 16 && tiles * ((a.m + 31) / 32) >= 4 * 256) return run4<T, 2, 4, 4, true, GS, ZEROS>(a, s);
    if (blocks < 256) return run4<T, 1, 1, 8, true, GS, ZEROS>(a, s);
    return blocks < 704 ? run4<T, 1, 2, 8, true, GS, ZEROS>(a, s) : run4<T, 1, 4, 8, true, GS, ZEROS>(a, s);
  } else {
    const int steps = (int)steps_of(a.k);
    if (a.m <= 16) {
      const bool even = (reinterpret_cast<uintptr_t>(a.x) | (uintptr_t)a.x_stride * 2) % 4 == 0;
      switch (cheapest(kFewCosts, a.m == 1 || even ? 0 : 2, 5, [&](const Cost& c) { return c.few(a.m, tiles, steps); })) {
        case 0: return run4<T, 1, 1, 8, false, GS, ZEROS>(a, s);
        case 1: return run4<T, 1, 2, 8, false, GS, ZEROS>(a, s);
        case 2: return run4<T, 1, 1, 16, true, GS, ZEROS>(a, s);
        case 3: return run4<T, 1, 2, 8, true, GS, ZEROS>(a, s);
        default: return run4<T, 1, 4, 8, true, GS, ZEROS>(a, s);
      }
    }
    switch (cheapest(kCosts, 0, 8, [&](const Cost& c) { return c.of(a.m, tiles, steps); })) {
      case 0: return run4<T, 1, 1, 16, true, GS, ZEROS>(a, s);
      case 1: return run4<T, 1, 2, 8, true, GS, ZEROS>(a, s);
      case 2: return run4<T, 1, 4, 8, true, GS, ZEROS>(a, s);
      case 3: return run4<T, 2, 4, 8, true, GS, ZEROS>(a, s);
      case 4: return run4_many<T, 4, 2, GS, ZEROS>(a, s);
      case 5: return run4_many<T, 4, 1, GS, ZEROS>(a, s);
      case 6: return run4_many<T, 2, 2, GS, ZEROS>(a, s);
      default: return run4_many<T, 1, 2, GS, ZEROS>(a, s);
    }
  }
}

template <class T, bool ZEROS>
hipError_t linear4_g(const Linear4Args& a, hipStream_t s) {
  switch (a.group) {
    case 32: return linear4_m<T, 1, ZEROS>(a, s);
    case 64: return linear4_m<T, 2, ZEROS>(a, s);
    default: return linear4_m<T, 4, ZEROS>(a, s);
  }
}

template <class T>
hipError_t linear4_t(const Linear4Args& a, hipStream_t s) {
  return a.zeros != nullptr ? linear4_g<T, true>(a, s) : linear4_g<T, false>(a, s);
}

template <class T>
hipError_t quantize_t(const QuantizeArgs& a, hipStream_t s) {
  const int64_t items = a.n * ((a.k + a.group - 1) / a.group);
  const unsigned grid = (unsigned)std::min<int64_t>((items + 15) / 16, 1 << 16);
  if (a.group == 32) hipLaunchKernelGGL((k_quantize4<T, 2>), dim3(grid), dim3(256), 0, s, a);
  else if (a.group == 64) hipLaunchKernelGGL((k_quantize4<T, 4>), dim3(grid), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((k_quantize4<T, 8>), dim3(grid), dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_pack4(const PackArgs& a, hipStream_t s) {
  const int64_t words = tiles_of(a.n) * steps_of(a.k) * 256;
  const unsigned grid = (unsigned)std::min<int64_t>((words + 255) / 256, 1 << 16);
  hipLaunchKernelGGL(k_pack4, dim3(grid), dim3(256), 0, s, a);
  return hipGetLastError();
}

hipError_t launch_quantize4(const QuantizeArgs& a, int dtype, hipStream_t s) {
  if (dtype == SY_BF16) return quantize_t<BF16>(a, s);
  if (dtype == SY_F16) return quantize_t<F16>(a, s);
  return quantize_t<F32>(a, s);
}

hipError_t launch_linear4(const Linear4Args& a, int dtype, hipStream_t s) {
  if (dtype == SY_BF16) return linear4_t<BF16>(a, s);
  if (dtype == SY_F16) return linear4_t<F16>(a, s);
  return linear4_t<F32>(a, s);
}

}  // namespace sy
