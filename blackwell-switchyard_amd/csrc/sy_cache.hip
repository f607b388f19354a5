// Serving: the rotation of a fused projection on its way into a paged cache, and
// attention of the new tokens over the cache's pages.
#include <algorithm>

#include "sy_launch.hpp"

namespace sy {

namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef short i16x4_t __attribute__((ext_vector_type(4)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x2_t __attribute__((ext_vector_type(2)));

constexpr int kBlock = 256;
constexpr int kWaves = kBlock / 64;

// ------------------------------------------------------------------ sequences

// One sequence's rows of the packed tensors, its length, and how many of its tokens the
// cache can hold: later ones are not there. The prefix pass takes every row as one sequence
// over the prefix's keys.
struct Seq {
  int row0, n, len, keys;
};

__device__ __forceinline__ int clamp(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }

__device__ __forceinline__ Seq seq_of(const CacheArgs& c, int b) {
  Seq s;
  if (c.starts != nullptr) {
    s.row0 = clamp(c.starts[b], 0, c.n_tok);
    s.n = clamp(c.starts[b + 1], s.row0, c.n_tok) - s.row0;
  } else {
    s.row0 = b * c.each;
    s.n = c.each;
  }
  s.len = clamp(c.lengths[b], 0, 0x7fffff00);  // (with room for a tile's rows)
  s.keys = min(s.len, (int)c.cap);
  return s;
}

// Rows before the first sequence and behind the last.
__device__ __forceinline__ bool outside(const CacheArgs& c, int row) {
  return c.starts != nullptr && (row < c.starts[0] || row >= c.starts[c.n_seq]);
}

// The sequence that holds a packed row, or -1: every lane looks at another sequence, so
// 64 of them cost two loads.
__device__ __forceinline__ int find_seq(const CacheArgs& c, int row) {
  if (c.starts == nullptr) return row / c.each;
  const int lane = threadIdx.x & 63;
  for (int b0 = 0; b0 < c.n_seq; b0 += 64) {
    const int b = b0 + lane;
    const bool in = b < c.n_seq && c.starts[b] <= row && row < c.starts[b + 1];
    const uint64_t hit = __ballot(in);
    if (hit != 0) return b0 + __ffsll((unsigned long long)hit) - 1;
  }
  return -1;
}

// Bytes from a cache's start to the row of token j (head 0) in page `id`.
__device__ __forceinline__ uint64_t row_at(const CacheArgs& c, int id, int j) {
  return (uint64_t)(uint32_t)id * c.page_bytes + (uint32_t)(j & ((1 << c.page_shift) - 1)) * c.row_bytes;
}
template <class S> __device__ __forceinline__ S* bytes_on(S* p, uint64_t n) {
  return reinterpret_cast<S*>(reinterpret_cast<uintptr_t>(p) + n);
}

// --------------------------------------------------------------------- append
//
// A workgroup per token, a thread per two chunks of VE elements that turn together
// (channel i of a head's first half with channel i of its second). Every byte is read once
// and written once. Prompts are bound by memory: 5754 tokens of 16 heads of 128 in bf16, 144
// MB, take 31 us at 4.7 TB/s; a large copy runs at 5.2. One token each of 8 sequences is bound
// by latency: starts or lengths, the table's entry and the row, 4 us of the 6.6 a call takes.
template <class T, int VE>
struct Chunk {
  float f[VE];
};
template <class T, int VE>
__device__ __forceinline__ Chunk<T, VE> ld_chunk(const typename T::storage* p) {
  Chunk<T, VE> r;
  if constexpr (VE * sizeof(typename T::storage) == 16) {
    const i32x4_t x = *reinterpret_cast<const i32x4_t*>(p);
#pragma unroll
    for (int e = 0; e < VE; ++e) r.f[e] = elem<T>(x, e);
  } else if constexpr (VE * sizeof(typename T::storage) == 8) {
    const i32x2_t x = *reinterpret_cast<const i32x2_t*>(p);
    const i32x4_t y = {x[0], x[1], 0, 0};
#pragma unroll
    for (int e = 0; e < VE; ++e) r.f[e] = elem<T>(y, e);
  } else {
    i32x4_t y = {0, 0, 0, 0};
    __builtin_memcpy(&y, p, sizeof(typename T::storage));
    r.f[0] = elem<T>(y, 0);
  }
  return r;
}
template <class T, int VE>
__device__ __forceinline__ void st_chunk(typename T::storage* p, const Chunk<T, VE>& c) {
  float f[T::ce] = {};
#pragma unroll
  for (int e = 0; e < VE; ++e) f[e] = c.f[e];
  const i32x4_t x = pack<T>(f);
  if constexpr (VE * sizeof(typename T::storage) == 16) {
    *reinterpret_cast<i32x4_t*>(p) = x;
  } else if constexpr (VE * sizeof(typename T::storage) == 8) {
    *reinterpret_cast<i32x2_t*>(p) = i32x2_t{x[0], x[1]};
  } else {
    __builtin_memcpy(p, &x, sizeof(typename T::storage));
  }
}

template <class T, int VE>
__global__ void __launch_bounds__(kBlock) k_append(const AppendArgs a) {
  using S = typename T::storage;
  const CacheArgs& c = a.c;
  const int half = c.hd / 2;
  const int per_head = half / VE;
  const int items = (c.heads + 2 * c.kv_heads) * per_head;
  S* const q = static_cast<S*>(a.q);
  for (int tok = blockIdx.x; tok < c.n_tok; tok += gridDim.x) {
    const S* const row = static_cast<const S*>(a.qkv) + tok * a.tok_stride;
    const int b = find_seq(c, tok);
    if (b < 0) {
      if (a.fill && outside(c, tok)) {
        const Chunk<T, VE> zero{};
        for (int i = threadIdx.x; i < c.heads * per_head * 2; i += kBlock)
          st_chunk<T, VE>(q + (int64_t)tok * c.heads * c.hd + i * VE, zero);
      }
      continue;
    }
    const Seq s = seq_of(c, b);
    const int j = s.len - s.n + (tok - s.row0);  // position among the sequence's own tokens
    const int64_t at = j + a.offset;
    uint64_t dst = 0;
    bool placed = j >= 0 && j < c.cap && at < a.n_pos;
    if (placed) {
      const int id = c.table[b * c.table_stride + (j >> c.page_shift)];
      placed = (unsigned)id < (unsigned)c.n_pages;
      if (placed) dst = row_at(c, id, j);
    }
    for (int i = threadIdx.x; i < items; i += kBlock) {
      const int head = i / per_head;
      const int ch = (i - head * per_head) * VE;
      const S* const src = row + head * a.head_stride + ch;
      Chunk<T, VE> lo = ld_chunk<T, VE>(src);
      Chunk<T, VE> hi = ld_chunk<T, VE>(src + half);
      if (head < c.heads + c.kv_heads && placed) {
        const float* const cp = a.cosv + at * half + ch;
        const float* const sp = a.sinv + at * half + ch;
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const float x = lo.f[e], y = hi.f[e], co = cp[e], si = sp[e];
          lo.f[e] = x * co - y * si;
          hi.f[e] = x * si + y * co;
        }
      }
      S* out;
      if (head < c.heads) {
        if (!placed) {
#pragma unroll
          for (int e = 0; e < VE; ++e) lo.f[e] = hi.f[e] = __int_as_float(0x7fc00000);
        }
        out = q + ((int64_t)tok * c.heads + head) * c.hd + ch;
      } else {
        if (!placed) continue;
        const bool key = head < c.heads + c.kv_heads;
        const int h = head - c.heads - (key ? 0 : c.kv_heads);
        out = bytes_on(static_cast<S*>(key ? c.k : c.v) + h * c.head_stride + ch, dst);
      }
      st_chunk<T, VE>(out, lo);
      st_chunk<T, VE>(out + half, hi);
    }
  }
}

// The same behind a norm of every query and key head, u = x r g with r = 1 / sqrt(mean(x^2) +
// eps): L lanes a head, a power of two, of which the ones past it do nothing, each with two
// chunks of VE elements that turn together; the sum of squares stays among them. `split` waves
// share a token's heads, kAhead rounds of them on their way before the first is needed, and
// before the token's place is known. Memory bounds it: 6728 tokens of 40 heads of 64 in fp16 move
// 70 MB in 17.2 us, 4.1 TB/s (loads after the place, 35.6); 8 single tokens of 48 heads of 128
// take 4.1, three dependent loads.
template <class T, int VE, int L>
__global__ void __launch_bounds__(kBlock) k_append_norm(const AppendArgs a, int split, int first) {
  using S = typename T::storage;
  constexpr int kHeads = 64 / L, kAhead = 3;  // heads of a wave's round
  const CacheArgs& c = a.c;
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int half = c.hd / 2, ch = lane % L * VE;
  const int rows = c.heads + 2 * c.kv_heads;
  const float inv_hd = 1.0f / (float)c.hd;
  const bool in_head = ch < half;
  S* const q = static_cast<S*>(a.q);
  const int tok = first + (int)blockIdx.x * (kWaves / split) + wave / split;
  if (tok >= c.n_tok) return;
  const S* const from = static_cast<const S*>(a.qkv) + tok * a.tok_stride + ch;
  int head = wave % split * kHeads + lane / L;
  i32x4_t raw[kAhead][2];  // (as they lie in memory: half the registers)
  const auto load = [&]() {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int h = head + i * split * kHeads;
      raw[i][0] = raw[i][1] = i32x4_t{0, 0, 0, 0};
      if (!in_head || h >= rows) continue;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const S* const p = from + h * a.head_stride + k * half;
        if constexpr (VE == T::ce) raw[i][k] = *reinterpret_cast<const i32x4_t*>(p);
        else __builtin_memcpy(&raw[i][k], __builtin_assume_aligned(p, 8), 8);
      }
    }
  };
  load();
  float gain[2][2][VE] = {};
  if (in_head) {
    const bool wide = a.gain_dtype == F32::code;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      ld_gains<T, VE>(a.q_gain, h * half + ch, wide, gain[0][h]);
      ld_gains<T, VE>(a.k_gain, h * half + ch, wide, gain[1][h]);
    }
  }
  const int b = find_seq(c, tok);
  if (b < 0) {
    if (a.fill && outside(c, tok)) {
      const Chunk<T, VE> zero{};
      for (int i = wave % split * 64 + lane; i < c.heads * c.hd / VE; i += split * 64)
        st_chunk<T, VE>(q + (int64_t)tok * c.heads * c.hd + i * VE, zero);
    }
    return;
  }
  const Seq s = seq_of(c, b);
  const int j = s.len - s.n + (tok - s.row0);  // position among the sequence's own tokens
  const int64_t at = j + a.offset;
  uint64_t dst = 0;
  bool placed = j >= 0 && j < c.cap && at < a.n_pos;
  float co[VE] = {}, si[VE] = {};
  if (placed) {
    const int id = c.table[b * c.table_stride + (j >> c.page_shift)];
    if (in_head) {
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        co[e] = a.cosv[at * half + ch + e];
        si[e] = a.sinv[at * half + ch + e];
      }
    }
    placed = (unsigned)id < (unsigned)c.n_pages;
    if (placed) dst = row_at(c, id, j);
  }
  // (The bounds are the wave's: its lanes add up their squares.)
  for (int round = wave % split * kHeads; round < rows; round += kAhead * split * kHeads) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int h = head + i * split * kHeads;
      Chunk<T, VE> lo, hi;
#pragma unroll
      for (int e = 0; e < VE; ++e) lo.f[e] = elem<T>(raw[i][0], e), hi.f[e] = elem<T>(raw[i][1], e);
      const float r = head_rinv<VE, L>(lo.f, hi.f, inv_hd, a.eps);
      if (!in_head || h >= rows) continue;
      const bool key = h >= c.heads, turned = h < c.heads + c.kv_heads;
      if (turned) {
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          lo.f[e] *= r * (key ? gain[1][0][e] : gain[0][0][e]);
          hi.f[e] *= r * (key ? gain[1][1][e] : gain[0][1][e]);
          turn(lo.f[e], hi.f[e], co[e], si[e]);
        }
      }
      S* out;
      if (!key) {
        if (!placed) {
#pragma unroll
          for (int e = 0; e < VE; ++e) lo.f[e] = hi.f[e] = __int_as_float(0x7fc00000);
        }
        out = q + ((int64_t)tok * c.heads + h) * c.hd + ch;
      } else {
        if (!placed) continue;
        const int kv = h - c.heads - (turned ? 0 : c.kv_heads);
        out = bytes_on(static_cast<S*>(turned ? c.k : c.v) + kv * c.head_stride + ch, dst);
      }
      st_chunk<T, VE>(out, lo);
      st_chunk<T, VE>(out + half, hi);
    }
    head += kAhead * split * kHeads;
    if (round + kAhead * split * kHeads < rows) load();
  }
}

// ------------------------------------------------------------------ attention
//
// One pass over the keys with the running maximum m and sum l of a softmax:
//   s_j = scale <q, k_j>,  o <- o 2^(m - m') + sum_j 2^(s_j - m') v_j   (s in base 2)
//
// A tile is KT tokens of one kv head against RT = 16 NT query rows; the rows of a kv head
// are the (token, head) pairs that read it, token-major, so grouped heads share a tile.
// Both products run transposed, S^T = K Q^T and O^T = V^T P^T: a lane then owns one query
// row (column lane % 16), so the statistics are lane-local up to two exchanges between
// the four groups of 16 lanes, the rescaling of O is a lane-local factor, and the
// products P leave the first multiplication in the places where the second wants them
// (the order of the tokens within a tile is free, as long as V's is the same). K goes
// from memory straight into the first product's registers. V passes through a
// wave-private piece of LDS: 16-bit rows come back transposed by ds_read_b64_tr_b16,
// fp32 ones element by element.
//
// The work is cut into units of one tile, ordered (kv head, sequence, row tile, key
// tile), and every workgroup of a fixed grid takes an equal run of them whatever the
// lengths are: a long sequence is shared by many workgroups, short ones lie many in one.
// The four waves of a workgroup take the tiles of a segment in turn, each with its own
// registers and LDS and no barrier between tiles, and join their results through LDS at
// the segment's end. Bound by memory: 32 sequences of any lengths up to 4096, 16 heads of
// 128 in bf16, read 567 MB in 111 us with the merge (5.1 TB/s; 5.9 where nothing is merged;
// a plain read of as much runs at 6.5), two of 131000 tokens and 4 kv heads 469 MB in 94.
// Single tokens over a few hundred are bound by latency: lengths, page ids, keys and the
// fold through LDS one after another, 10 us. A run begins and ends inside at most one segment each, so two
// partial results (o, m, l) a workgroup are enough; k_merge joins them. Nothing here
// depends on lengths the host knows. Where no sequence can be longer than a few tiles a
// wave, a workgroup takes one whole segment instead, and nothing is left to merge.
template <class T> struct Mma;
template <> struct Mma<BF16> {
  static __device__ __forceinline__ f32x4_t run(const i32x4_t& a, const i32x4_t& b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                   __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  }
};
template <> struct Mma<F16> {
  static __device__ __forceinline__ f32x4_t run(const i32x4_t& a, const i32x4_t& b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a),
                                                  __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  }
};
template <> struct Mma<F32> {
  static __device__ __forceinline__ f32x4_t run(const i32x4_t& a, const i32x4_t& b, f32x4_t c) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(__int_as_float(a[j]), __int_as_float(b[j]), c, 0, 0, 0);
    return c;
  }
};

__device__ __forceinline__ float group_sum(float x) {  // over the four 16-lane groups
  const uint32_t u = __float_as_uint(x);
  const auto p = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t y = __float_as_uint(__uint_as_float(p[0]) + __uint_as_float(p[1]));
  const auto r = __builtin_amdgcn_permlane32_swap(y, y, false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float group_max(float x) {
  const uint32_t u = __float_as_uint(x);
  const auto p = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t y = __float_as_uint(fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1])));
  const auto r = __builtin_amdgcn_permlane32_swap(y, y, false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// x y, rounded (never part of a fused operation).
__device__ __forceinline__ float product(float x, float y) {
#pragma clang fp contract(off)
  return x * y;
}

// What a pass takes the exponentials relative to: the largest score, or a little below it.
// fp16 ends at 2^-14 (2^-24 with fewer bits), and a context of 10^5 faint tokens behind one
// strong one has weights below both that make up a percent of a row together. Their sum is
// what the row is divided by, so the second product must not lose them: weights start at
// 2^LIFT instead of 1. A weight is then off by its own rounding or 2^-(25 + LIFT) of the
// largest, whichever is more. Scores from 2^22 on are whole steps apart in fp32, and with
// them the difference would be: they keep their place. bf16 and fp32 reach down to 2^-126.
constexpr float kWholeScores = 4194304.0f;
template <class T, int LIFT> __device__ __forceinline__ float reference_of(float top) {
  if constexpr (T::code == SY_F16) return fabsf(top) < kWholeScores ? top - (float)LIFT : top;
  else return top;
}

template <class T> constexpr int tokens_of() { return T::code == SY_F32 ? 16 : 32; }

// How a pass over the keys is cut, the same for the kernel, the merge and the host.
struct Cut {
  int pre;      // 1: every row over the prefix's keys
  int few;      // sequences of more rows a kv head are k_flash's (none: INT_MAX)
  int rt;       // rows a tile
  int kt;       // tokens a tile
  int workers;  // workgroups
  int least;    // fewest units a worker takes; 0: every worker takes one whole segment
  int rs;       // rows a partial result holds
  float* o;     // partial results [2 workers][rs][hd], and m, l
  float* ml;
};

__device__ __forceinline__ Seq pass_seq(const CacheArgs& c, int pre, int prefix_len, int b) {
  if (!pre) return seq_of(c, b);
  Seq s;
  s.row0 = c.starts != nullptr ? clamp(c.starts[0], 0, c.n_tok) : 0;
  s.n = (c.starts != nullptr ? clamp(c.starts[c.n_seq], s.row0, c.n_tok) : c.n_tok) - s.row0;
  s.len = s.keys = prefix_len;
  return s;
}

struct Tiles {
  int row_tiles, key_tiles;
};
__device__ __forceinline__ Tiles tiles_of(const Cut& u, int group, const Seq& s) {
  const int rows = s.n * group;
  if (rows == 0 || (!u.pre && rows > u.few)) return {0, 0};
  const int k = (s.keys + u.kt - 1) / u.kt;  // rows that see nothing still have to be written
  return {(rows + u.rt - 1) / u.rt, k < 1 ? 1 : k};
}

// Sums and searches over the sequences, `count(b)` units each: every lane looks at another
// sequence, so 64 of them cost one round of loads.
template <class F> __device__ __forceinline__ int total_of(int upto, F count) {
  int x = 0;
  for (int b = threadIdx.x & 63; b < upto; b += 64) x += count(b);
  return __builtin_amdgcn_readlane((int)wave_scan<uint32_t>(x), 63);
}
// The sequence that holds a unit, and the units before it; false past the last.
template <class F> __device__ __forceinline__ bool locate(int n_seq, int unit, F count, int* seq, int* base) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int b0 = 0; b0 < n_seq; b0 += 64) {
    const int mine = b0 + lane < n_seq ? count(b0 + lane) : 0;
    const int incl = (int)wave_scan<uint32_t>(mine);
    const uint64_t hit = __ballot(before + incl > unit);
    if (hit != 0) {
      const int l = __ffsll((unsigned long long)hit) - 1;
      *seq = b0 + l;
      *base = before + __builtin_amdgcn_readlane(incl - mine, l);
      return true;
    }
    before += __builtin_amdgcn_readlane(incl, 63);
  }
  return false;
}
// Units a worker takes (the host sees to it that all numbers of units fit 31 bits).
__device__ __forceinline__ int share_of(const Cut& u, int units) {
  return max((units + u.workers - 1) / u.workers, u.least);
}
// The unit-th of all units in the order of their distance from their sequence's last one
// (the last units of all sequences, then those before them, ...): that sequence and the
// unit's number in it. With `most` the largest number of units a sequence can have. The
// second `fold` units are taken in reverse: workgroups are handed out to one place of every
// CU, then to the next, so a CU's second one is the shorter the longer its first.
template <class F>
__device__ __forceinline__ bool locate_last(int n_seq, int unit, int most, int fold, F count, int* seq, int* number) {
  const int lane = threadIdx.x & 63;
  const int mine = lane < n_seq ? count(lane) : 0;  // (up to 64 sequences are asked once)
  const auto nearer = [&](int k) {  // units at most k - 1 before their sequence's last
    int x = min(mine, k);
    for (int b = lane + 64; b < n_seq; b += 64) x += min(count(b), k);
    return __builtin_amdgcn_readlane((int)wave_scan<uint32_t>(x), 63);
  };
  const int total = nearer(most);
  if (unit >= total) return false;
  if (unit >= fold && unit < 2 * fold) unit = min(2 * fold, total) - 1 - (unit - fold);
  int lo = 0, hi = most - 1;  // the distance: the largest k with nearer(k) <= unit
  while (lo < hi) {
    const int mid = lo + (hi - lo + 1) / 2;
    if (nearer(mid) <= unit) lo = mid;
    else hi = mid - 1;
  }
  int skip = unit - nearer(lo);  // sequences of more than `lo` units to pass over
  for (int b0 = 0; b0 < n_seq; b0 += 64) {
    const int n = b0 == 0 ? mine : b0 + lane < n_seq ? count(b0 + lane) : 0;
    const int incl = (int)wave_scan<uint32_t>(n > lo ? 1 : 0);
    const uint64_t hit = __ballot(incl > skip);
    if (hit != 0) {
      const int l = __ffsll((unsigned long long)hit) - 1;
      *seq = b0 + l;
      *number = __builtin_amdgcn_readlane(n, l) - 1 - lo;
      return true;
    }
    skip -= __builtin_amdgcn_readlane(incl, 63);
  }
  return false;
}
__device__ __forceinline__ int units_of(const CacheArgs& c, const Cut& u, int prefix_len, int b) {
  const Tiles t = tiles_of(u, c.group, pass_seq(c, u.pre, prefix_len, b));
  return t.row_tiles * t.key_tiles;
}

// Whether any of a chunk's elements is an infinity or NaN.
template <class T> __device__ __forceinline__ bool nonfinite(const i32x4_t& x) {
  bool bad = false;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t w = (uint32_t)x[k];
    if constexpr (T::code == SY_F32) {
      bad |= (w & 0x7f800000u) == 0x7f800000u;
    } else {
      constexpr uint32_t e = T::code == SY_BF16 ? 0x7f80u : 0x7c00u;
      bad |= (w & e) == e || ((w >> 16) & e) == e;
    }
  }
  return bad;
}

// Rows before the first sequence and behind the last become zero.
template <class T> __device__ __forceinline__ void zero_outside(const AttendArgs& a) {
  using S = typename T::storage;
  const CacheArgs& c = a.c;
  const int lo = clamp(c.starts[0], 0, c.n_tok), hi = clamp(c.starts[c.n_seq], lo, c.n_tok);
  const int64_t width = (int64_t)c.heads * c.hd;
  S* const out = static_cast<S*>(a.out);
  const int64_t at = (int64_t)blockIdx.x * kBlock + threadIdx.x, step = (int64_t)gridDim.x * kBlock;
  for (int64_t i = at; i < lo * width; i += step) out[i] = S(0);
  for (int64_t i = hi * width + at; i < c.n_tok * width; i += step) out[i] = S(0);
}

// LDS of a workgroup: a piece a wave, then the statistics of a segment's results.
template <class T, int HD> constexpr int value_stride() {
  // A row's start moves by 32 (fp32: 16) bytes from row to row modulo all banks.
  return HD * (int)sizeof(typename T::storage) + (T::code == SY_F32 ? 16 : 32);
}
template <class T, int HD> constexpr int attend_lds() {
  return kWaves * tokens_of<T>() * value_stride<T, HD>() + kWaves * 16 * 2 * 4;
}

template <class T, int HD, int NT, bool EXACT>
__device__ __forceinline__ void attend(const AttendArgs& a, const Cut& u, const int direct, float* const row_o,
                                       float* const row_ml, const int worker, char* const shared) {
  using S = typename T::storage;
  constexpr int CE = T::ce;
  constexpr int KT = tokens_of<T>();
  constexpr int MT = KT / 16;
  constexpr int KC = HD / (4 * CE);  // chunks a lane holds of a row
  constexpr int MD = HD / 16;        // output tiles
  constexpr bool kF32 = T::code == SY_F32;
  constexpr int LS = value_stride<T, HD>();
  constexpr int OS = HD * 4 + 16;  // stride of a row of results in the same space
  static_assert(16 * OS <= KT * LS, "results fit the values' space");
  const auto stats = reinterpret_cast<float (*)[16][2]>(shared + kWaves * KT * LS);
  const CacheArgs& c = a.c;
  const int lane = threadIdx.x & 63;
  const int col = lane & 15, grp = lane >> 4;
  const int wave = wave_id();
  char* const vt = shared + wave * (KT * LS);
  const int n_seq = u.pre ? 1 : c.n_seq;
  const int plen = (int)a.prefix_len;
  const int hd = EXACT ? HD : c.hd;
  const float sl = a.scale * 1.44269504088896340736f;

  int h, b, rtile, tile;
  Seq s;
  Tiles ti;
  int unit = 0, end = 0;
  bool some;
  if (u.least == 0) {
    // Equal row tiles for every sequence: no search.
    const int per_seq = (c.each * c.group + u.rt - 1) / u.rt;
    h = worker / (per_seq * n_seq);
    b = worker / per_seq - h * n_seq;
    rtile = worker - (h * n_seq + b) * per_seq;
    tile = 0;
    s = pass_seq(c, u.pre, plen, b);
    ti = tiles_of(u, c.group, s);
    end = ti.key_tiles;
    some = true;
  } else {
    const auto count = [&](int x) { return units_of(c, u, plen, x); };
    const int per_head = total_of(n_seq, count);
    const int units = per_head * c.kv_heads;
    const int share = share_of(u, units);
    unit = worker * share;
    end = min(unit + share, units);
    int at = 0, base = 0;
    some = unit < end && per_head > 0;  // (overlapping sequences can have more units than fit)
    if (some) {
      h = unit / per_head;
      at = unit - h * per_head;
      some = locate(n_seq, at, count, &b, &base);
    }
    if (some) {
      s = pass_seq(c, u.pre, plen, b);
      ti = tiles_of(u, c.group, s);
      rtile = (at - base) / ti.key_tiles;
      tile = at - base - rtile * ti.key_tiles;
    }
  }

  if (some) {
    while (true) {
      const int count = min(ti.key_tiles - tile, end - unit);
      const bool begins = tile == 0, whole = begins && count == ti.key_tiles;

      // ---- this segment: kv head h, row tile rtile of sequence b, key tiles [tile, tile + count)
      const int rows = s.n * c.group;
      const int r0 = rtile * 16 * NT;
      const int past = u.pre ? plen : s.len - s.n + 1;  // keys the first token sees
      const int last = min(r0 + 16 * NT, rows) - 1;
      const int least = u.pre ? plen : min(past + r0 / c.group, s.keys);
      const int most = u.pre ? plen : min(past + last / c.group, s.keys);
      int limit[NT];
      i32x4_t q[NT][KC];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int r = min(r0 + 16 * n + col, last);  // rows past the last repeat it and are not stored
        const int t = r / c.group;
        limit[n] = u.pre ? plen : min(past + t, s.keys);
        const S* const qp = static_cast<const S*>(a.q) + (s.row0 + t) * a.q_tok_stride +
                            (h * c.group + (r - t * c.group)) * a.q_head_stride;
#pragma unroll
        for (int k = 0; k < KC; ++k) {
          const int ch = (k * 4 + grp) * CE;
          q[n][k] = i32x4_t{0, 0, 0, 0};
          if (EXACT || ch < hd) q[n][k] = *reinterpret_cast<const i32x4_t*>(qp + ch);
        }
      }
      float m[NT], l[NT];
      f32x4_t o[NT][MD];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        m[n] = -INFINITY;
        l[n] = 0.0f;
#pragma unroll
        for (int d = 0; d < MD; ++d) o[n][d] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
      }

      const int32_t* const pages = u.pre ? a.prefix_pages : c.table + b * c.table_stride;
      const S* const kb = static_cast<const S*>(c.k) + h * c.head_stride;
      const S* const vb = static_cast<const S*>(c.v) + h * c.head_stride;
      const int tiles = min(tile + count, (most + KT - 1) / KT);  // later ones hold nothing visible
      // Page ids run two tiles ahead of the products, keys and values one.
      int id[MT];
      bool ok[MT], okn[MT];
      i32x4_t kx[MT][KC], vx[MT][KC];
      uint64_t off[MT];
      // Ids are read whether or not a token is there (within the row): the first ones do
      // not wait for the sequence's length.
      const int last_page = u.pre ? (plen - 1) >> c.page_shift : (int)(c.cap >> c.page_shift) - 1;
      const auto ask_ids = [&](int t) {
#pragma unroll
        for (int x = 0; x < MT; ++x) id[x] = pages[min((t * KT + x * 16 + col) >> c.page_shift, last_page)];
      };
      const auto place = [&](int t) {  // ids -> offsets; a key with no place reads the cache's first row
#pragma unroll
        for (int x = 0; x < MT; ++x) {
          const int j = t * KT + x * 16 + col;
          okn[x] = (unsigned)id[x] < (unsigned)c.n_pages && j < most;
          off[x] = okn[x] ? row_at(c, id[x], j) : 0;
        }
      };
      const auto ask = [&](const S* base_p, i32x4_t (&dst)[MT][KC]) {
#pragma unroll
        for (int x = 0; x < MT; ++x)
#pragma unroll
          for (int k = 0; k < KC; ++k) {
            const int ch = (k * 4 + grp) * CE;
            dst[x][k] = *reinterpret_cast<const i32x4_t*>(bytes_on(base_p, off[x]) + (EXACT || ch < hd ? ch : 0));
          }
      };
      ask_ids(tile + wave);
      place(tile + wave);
      ask(kb, kx);
      ask(vb, vx);
      ask_ids(tile + wave + kWaves);
      for (int t = tile + wave; t < tiles; t += kWaves) {
#pragma unroll
        for (int x = 0; x < MT; ++x) ok[x] = okn[x];
        bool all_ok = true;
#pragma unroll
        for (int x = 0; x < MT; ++x) all_ok = all_ok && ok[x];
        const bool full = __all(all_ok) && (t + 1) * KT <= least;
        bool odd = false;  // a value that some rows must not see is no number
        if (!full) {
#pragma unroll
          for (int x = 0; x < MT; ++x) {
            const int j = t * KT + x * 16 + col;
#pragma unroll
            for (int k = 0; k < KC; ++k) {
              if (!ok[x]) vx[x][k] = i32x4_t{0, 0, 0, 0};
              if (j >= least) odd = odd || nonfinite<T>(vx[x][k]);
            }
          }
          odd = __any(odd);
        }
        asm volatile("" ::: "memory");
#pragma unroll
        for (int x = 0; x < MT; ++x)
#pragma unroll
          for (int k = 0; k < KC; ++k)
            *reinterpret_cast<i32x4_t*>(vt + (x * 16 + col) * LS + (k * 4 + grp) * 16) = vx[x][k];
        if (!EXACT) {
#pragma unroll
          for (int x = 0; x < MT; ++x)
#pragma unroll
            for (int k = 0; k < KC; ++k)
              if ((k * 4 + grp) * CE >= hd) kx[x][k] = i32x4_t{0, 0, 0, 0};
        }
        place(t + kWaves);
        if (t + kWaves < tiles) ask(vb, vx);
        // S^T
        f32x4_t st[NT][MT];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int x = 0; x < MT; ++x) {
            st[n][x] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < KC; ++k) st[n][x] = Mma<T>::run(kx[x][k], q[n][k], st[n][x]);
          }
        if (t + kWaves < tiles) ask(kb, kx);
        ask_ids(t + 2 * kWaves);
        // softmax of the tile; a lane holds tokens 4 grp .. 4 grp + 3 of each 16
        i32x4_t p16[NT], p16r[NT];
        float pf[NT][MT * 4];
        bool any_new = false;
        float scale_o[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float y[MT * 4];
#pragma unroll
          for (int x = 0; x < MT; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) y[x * 4 + e] = product(st[n][x][e], sl);  // as the maximum is
          if (!full) {
#pragma unroll
            for (int x = 0; x < MT; ++x) {
              const uint32_t bits = (uint32_t)__ballot(ok[x]) & 0xffffu;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int at = 4 * grp + e;
                const bool see = ((bits >> at) & 1u) != 0 && t * KT + x * 16 + at < limit[n];
                y[x * 4 + e] = see ? y[x * 4 + e] : -INFINITY;
              }
            }
          }
          float top = y[0];
#pragma unroll
          for (int e = 1; e < MT * 4; ++e) top = fmaxf(top, y[e]);
          const float mn = fmaxf(m[n], reference_of<T, 15>(group_max(top)));  // weights of at most 2^15.2
          const float mu = mn == -INFINITY ? 0.0f : mn;  // nothing seen yet
          scale_o[n] = __builtin_amdgcn_exp2f(m[n] - mu);
          any_new = any_new || mn != m[n];
          m[n] = mn;
          float sum = 0.0f;
#pragma unroll
          for (int e = 0; e < MT * 4; ++e) {
            pf[n][e] = __builtin_amdgcn_exp2f(y[e] - mu);
            sum += pf[n][e];
          }
          l[n] = fmaf(l[n], scale_o[n], sum);
          // The second product takes a weight as two numbers of the values' dtype, the
          // rounded weight and what it lacks: rounded once the weights alone would put 0.7 of
          // the output's own rounding on top of it (bf16 relative error 1.9e-3, so 1.7e-3),
          // and this kernel waits for memory, not for products. (fp16: a weight is off by
          // 2^-22 of itself or 2^-40 of the largest.)
          if constexpr (!kF32) {
            p16[n] = pack<T>(pf[n]);
            float rest[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) rest[e] = pf[n][e] - elem<T>(p16[n], e);
            p16r[n] = pack<T>(rest);
          }
        }
        if (__any(any_new)) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int d = 0; d < MD; ++d) o[n][d] *= scale_o[n];
        }
        asm volatile("" ::: "memory");
        // O^T
        if (__builtin_expect(!odd, 1)) {
#pragma unroll
          for (int d = 0; d < MD; ++d) {
            if (!EXACT && d * 16 >= hd) continue;
            if constexpr (kF32) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float w = *reinterpret_cast<const float*>(vt + (4 * grp + e) * LS + (d * 16 + col) * 4);
#pragma unroll
                for (int n = 0; n < NT; ++n)
                  o[n][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(w, pf[n][e], o[n][d], 0, 0, 0);
              }
            } else {
              i32x4_t w;
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                char* const from = vt + (x * 16 + 4 * grp + (col >> 2)) * LS + d * 32 + (col & 3) * 8;
                const i16x4_t r = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) i16x4_t*)from);
                const i32x2_t r2 = __builtin_bit_cast(i32x2_t, r);
                w[2 * x] = r2[0];
                w[2 * x + 1] = r2[1];
              }
#pragma unroll
              for (int n = 0; n < NT; ++n) o[n][d] = Mma<T>::run(w, p16r[n], Mma<T>::run(w, p16[n], o[n][d]));
            }
          }
        } else {
          // Rows that do not see a token leave its value out: 0 times an infinity is none.
#pragma unroll 1
          for (int j = 0; j < KT; ++j) {
            const int e = (j >> 4) * 4 + (j & 3), from = ((j >> 2) & 3) * 16 + col;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              float pv = pf[n][0];
#pragma unroll
              for (int x = 1; x < MT * 4; ++x) pv = e == x ? pf[n][x] : pv;
              pv = __shfl(pv, from);
              if (t * KT + j >= limit[n]) continue;
#pragma unroll
              for (int d = 0; d < MD; ++d) {
                const S* const vr = reinterpret_cast<const S*>(vt + j * LS) + d * 16 + 4 * grp;
                i32x4_t x4 = {0, 0, 0, 0};
                __builtin_memcpy(&x4, vr, 4 * sizeof(S));
#pragma unroll
                for (int i = 0; i < 4; ++i) o[n][d][i] = fmaf(pv, elem<T>(x4, i), o[n][d][i]);
              }
            }
          }
        }
        asm volatile("" ::: "memory");
      }

      // ---- results of the segment: the waves' joined, in their order
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float sum = group_sum(l[n]);
        if (grp == 0) {
          stats[wave][col][0] = m[n];
          stats[wave][col][1] = sum;
        }
#pragma unroll
        for (int d = 0; d < MD; ++d)
          *reinterpret_cast<f32x4_t*>(vt + col * OS + (d * 16 + 4 * grp) * 4) = o[n][d];
        __syncthreads();
        const int here = min(16, last + 1 - r0 - 16 * n);
        const int per_row = hd / 4;
        for (int i = threadIdx.x; i < here * per_row; i += kBlock) {
          const int row = i / per_row, ch = (i - row * per_row) * 4;
          float top = -INFINITY;
#pragma unroll
          for (int w = 0; w < kWaves; ++w) top = fmaxf(top, stats[w][row][0]);
          const float mu = top == -INFINITY ? 0.0f : top;
          float all = 0.0f;
          f32x4_t x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int w = 0; w < kWaves; ++w) {
            const float lw = stats[w][row][1];
            const float f = lw != lw ? 1.0f : __builtin_amdgcn_exp2f(stats[w][row][0] - mu);
            all = fmaf(lw, f, all);
            x += f * *reinterpret_cast<const f32x4_t*>(shared + w * (KT * LS) + row * OS + ch * 4);
          }
          const int r = r0 + 16 * n + row;
          const int t = r / c.group;
          const int64_t at = (int64_t)(s.row0 + t) * c.heads + h * c.group + (r - t * c.group);
          if (whole && direct) {
            float f[T::ce] = {};
#pragma unroll
            for (int e = 0; e < 4; ++e) f[e] = all == 0.0f ? 0.0f : x[e] / all;
            const i32x4_t x4 = pack<T>(f);
            __builtin_memcpy(static_cast<S*>(a.out) + at * hd + ch, &x4, 4 * sizeof(S));
          } else {
            const int64_t slot = whole ? at : (2 * (int64_t)worker + (begins ? 1 : 0)) * u.rs + (r - r0);
            *reinterpret_cast<f32x4_t*>((whole ? row_o : u.o) + slot * hd + ch) = x;
            if (ch == 0) {
              float* const pm = (whole ? row_ml : u.ml) + slot * 2;
              pm[0] = top;
              pm[1] = all;
            }
          }
        }
        __syncthreads();
      }

      unit += count;
      if (unit >= end) break;
      tile = 0;
      if (++rtile == ti.row_tiles) {
        rtile = 0;
        do {
          if (++b == n_seq) {
            b = 0;
            ++h;
          }
          s = pass_seq(c, u.pre, plen, b);
          ti = tiles_of(u, c.group, s);
        } while (ti.row_tiles == 0);
      }
    }
  }
}

template <class T, int HD, int NT, bool EXACT>
__global__ void __launch_bounds__(kBlock, NT == 1 && HD <= 128 ? 2 : 1)
k_attend(const AttendArgs a, const Cut u, const int direct, const int zero, float* const row_o, float* const row_ml) {
  __shared__ __align__(16) char shared[attend_lds<T, HD>()];
  attend<T, HD, NT, EXACT>(a, u, direct, row_o, row_ml, blockIdx.x, shared);
  if (zero) zero_outside<T>(a);
}

// ------------------------------------------------- attention of many rows (16-bit)
//
// The same pass where a sequence brings more rows than a tile of 16: a workgroup takes 128
// query rows of a kv head, a wave 32 of them, and all four waves read the same tiles of 64
// keys and values from LDS. Tile t + 1 is on its way from memory to the other half of LDS
// while tile t is multiplied, without passing through registers; one barrier a tile. The
// products run on v_mfma_f32_32x32x16 in the same transposed form. The maximum is only
// followed when a score passes it by more than 2^8 (weights stay below 256, fp16's lifted
// ones below 2^15.4, and the ratio to their sum is what counts), so the results are hardly
// ever rescaled.
//
// Bound by the matrix cores and, next to them, by the exponentials (a quarter of the
// vector rate): a wave's tile of heads of 128 is 1024 cycles of products and about as many of
// softmax, which two waves a SIMD overlap. Long even sequences run at 760 TFLOP/s (heads of
// 128, 16 of each kind), 930 (32 that share 8), 750 (heads of 64) and 465 (256, one workgroup
// a CU); four prompts of up to 2048 tokens at 530, as the causal triangles' ends leave CUs
// idle. A large bf16 product of the library runs at 1070.
struct Flash {
  int pre;     // 1: every row over the prefix's keys
  int virt;    // 1: the prefix's tiles come before each sequence's own
  int few;     // sequences of at most as many rows are k_attend's
  int tiles;   // row tiles, at most
  int splits;  // parts that a row tile's keys are cut into
  int fold;    // row tiles whose workgroups take one place on every CU
  float* o;    // partial results [tiles][kv_heads][splits][128][hd], and m, l
  float* ml;
};
constexpr int kFlashRows = 128, kFlashKeys = 64;

__device__ __forceinline__ int flash_tiles(const CacheArgs& c, const Flash& f, int prefix_len, int b) {
  const Seq s = pass_seq(c, f.pre, prefix_len, b);
  const int rows = s.n * c.group;
  return !f.pre && rows <= f.few ? 0 : (rows + kFlashRows - 1) / kFlashRows;
}
__device__ __forceinline__ int64_t flash_slot(const CacheArgs& c, const Flash& f, int tile, int h, int split) {
  return (((int64_t)tile * c.kv_heads + h) * f.splits + split) * kFlashRows;
}

typedef float f32x16_t __attribute__((ext_vector_type(16)));
template <class T> __device__ __forceinline__ f32x16_t mma32(const i32x4_t& a, const i32x4_t& b, const f32x16_t& c) {
  if constexpr (T::code == SY_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c,
                                                   0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0,
                                                  0, 0);
}

// 16 bytes a lane from memory to LDS, lane i's at byte `at` + 16 i of the workgroup's LDS;
// done when vmcnt says so. (The builtin's loads are waited for before the next read of any
// LDS, the other buffer included. There is no output register that could be reused while
// the load is under way. The compiler does not count these loads: a wait of its own for an
// earlier load would wait for them too, so there must be none behind them. m0 is declared as
// written, so that the compiler's own uses of it, in indexed registers and LDS, set it anew; its
// warning that the register is a reserved one is of no use here.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_to_lds(const void* from, uint32_t at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(at), "v"(from)
               : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ __forceinline__ uint32_t lds_byte(void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)p;
}
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// LDS: two tiles of keys, two of values; whether all keys of a wave's rows are there, of
// either tile; and of an edge tile's keys, 1 it is there, 2 its value holds an infinity or NaN.
template <int HD> constexpr int flash_lds() { return 4 * kFlashKeys * HD * 2 + 2 * kWaves * 4 + kFlashKeys * 4; }

template <class T, int HD, bool EXACT, bool TWO>
__device__ __forceinline__ void flash(const AttendArgs& a, const Flash& f, const int direct, float* const row_o,
                                      float* const row_ml, const int block, char* const shared) {
  using S = typename T::storage;
  constexpr int KT = kFlashKeys;
  constexpr int CPR = HD / 8;      // 16-byte chunks of a row
  constexpr int RB = HD * 2;       // bytes of a row in LDS, without padding: chunks are swizzled instead
  constexpr int RPI = 64 / CPR;    // rows a wave loads at a time
  constexpr int NP = KT / (RPI * kWaves);
  constexpr int KC = HD / 16, MD = HD / 32;
  char* const kl = shared;
  char* const vl = kl + 2 * KT * RB;
  const auto whole = reinterpret_cast<int (*)[kWaves]>(vl + 2 * KT * RB);
  int* const flags = reinterpret_cast<int*>(whole + 2);
  const CacheArgs& c = a.c;
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
  const int col = lane & 31, half = lane >> 5;
  const int plen = (int)a.prefix_len;
  const int hd = EXACT ? HD : c.hd;

  const int h = block % c.kv_heads;
  const int rest = block / c.kv_heads;
  const int split = rest % f.splits, tile_id = rest / f.splits;
  int b, rtile;
  if (!locate_last(f.pre ? 1 : c.n_seq, tile_id, f.tiles, f.fold,
                   [&](int x) { return flash_tiles(c, f, plen, x); }, &b, &rtile))
    return;
  const Seq s = pass_seq(c, f.pre, plen, b);
  const int rows = s.n * c.group;
  const int r0 = rtile * kFlashRows;
  const int last = min(r0 + kFlashRows, rows) - 1;
  const int past = f.pre ? plen : s.len - s.n + 1;  // keys the first token sees
  const int most = f.pre ? plen : min(past + last / c.group, s.keys);
  const int pre_tiles = f.virt ? (plen + KT - 1) / KT : 0;
  const int tiles = pre_tiles + (most > 0 ? (most + KT - 1) / KT : 0);
  const int t0 = (int)((int64_t)tiles * split / f.splits), t1 = (int)((int64_t)tiles * (split + 1) / f.splits);

  // This wave's rows, a lane's own among them.
  const int w0 = r0 + 32 * wave;
  const bool active = w0 <= last;
  const int r = min(w0 + col, last);
  const int tok = r / c.group;
  const int limit = f.pre ? plen : min(past + tok, s.keys);
  const int least = f.pre ? plen : min(past + w0 / c.group, s.keys);
  const int wmost = f.pre ? plen : min(past + min(w0 + 31, last) / c.group, s.keys);
  const int64_t out_row = (int64_t)(s.row0 + tok) * c.heads + h * c.group + (r - tok * c.group);
  i32x4_t q[KC];
  {
    const S* const qp = static_cast<const S*>(a.q) + (s.row0 + tok) * a.q_tok_stride +
                        (h * c.group + (r - tok * c.group)) * a.q_head_stride;
#pragma unroll
    for (int k = 0; k < KC; ++k) {
      const int ch = (2 * k + half) * 8;
      q[k] = i32x4_t{0, 0, 0, 0};
      if (EXACT || ch < hd) q[k] = *reinterpret_cast<const i32x4_t*>(qp + ch);
    }
  }
  // Scores in base 2; a negative scale turns the queries' signs, so that the largest
  // product is the largest score. A scale of zero goes into the queries (those of infinities
  // and NaN become NaN, as their products would): hidden scores are -inf before the scale.
  float sl = a.scale * 1.44269504088896340736f;
  if (sl == 0.0f) {
    sl = 1.0f;
#pragma unroll
    for (int k = 0; k < KC; ++k) {
      float z[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) z[e] = 0.0f * elem<T>(q[k], e);
      q[k] = pack<T>(z);
    }
  } else if (sl < 0.0f) {
    sl = -sl;
#pragma unroll
    for (int k = 0; k < KC; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) q[k][e] ^= (int)0x80008000;
  }

  // Loading: a wave's rows of load p are (4 p + wave) RPI + lane / CPR, a lane's place in a
  // row lane % CPR. Chunk ch of row r lies at place ch ^ key_swizzle(r) (keys: 16 rows of
  // one chunk then lie in 16 different groups of banks) or ch ^ value_swizzle(r) (values: 4
  // rows of one 64-byte group in 4 different ones).
  const auto key_swizzle = [](int r) { return HD == 64 ? (r >> 1) & 7 : r & 15; };
  const auto value_swizzle = [](int r) { return (HD == 64 ? (r >> 1) & 1 : r & 3) << 2; };
  const S* const kb = static_cast<const S*>(c.k) + h * c.head_stride;
  const S* const vb = static_cast<const S*>(c.v) + h * c.head_stride;
  const int32_t* const own_pages = f.pre ? a.prefix_pages : c.table + b * c.table_stride;
  const int own_last = f.pre ? (plen - 1) >> c.page_shift : (int)(c.cap >> c.page_shift) - 1;
  const int wg_least = f.pre ? plen : min(past + r0 / c.group, s.keys);
  const uint32_t kl_at = lds_byte(kl), vl_at = lds_byte(vl);
  int id[NP];
  const auto ask_ids = [&](int t) {
    const bool own = t >= pre_tiles;
    const int32_t* const pages = own ? own_pages : a.prefix_pages;
    const int end = own ? own_last : (plen - 1) >> c.page_shift;
    const int j0 = (own ? t - pre_tiles : t) * KT + wave * RPI + lane / CPR;
#pragma unroll
    for (int p = 0; p < NP; ++p) id[p] = pages[min((j0 + p * kWaves * RPI) >> c.page_shift, end)];
  };
  const auto ask = [&](int t) {  // keys with no place read the cache's first row
    const int buf = (t - t0) & 1;
    const bool own = t >= pre_tiles;
    const int j0 = (own ? t - pre_tiles : t) * KT;
    const int end = own ? most : plen;
    bool all = true;
    uint64_t off[NP];
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      asm volatile("" : "+v"(id[p]));  // its wait is here, before the first load to LDS
      const int j = j0 + (p * kWaves + wave) * RPI + lane / CPR;
      const bool ok = (unsigned)id[p] < (unsigned)c.n_pages && j < end;
      all = all && ok;
      off[p] = row_at(c, ok ? id[p] : 0, ok ? j : 0);
    }
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const int first = (p * kWaves + wave) * RPI, row = first + lane / CPR;
      const int kc = (lane % CPR ^ key_swizzle(row)) * 8, vc = (lane % CPR ^ value_swizzle(row)) * 8;
      const uint32_t to = __builtin_amdgcn_readfirstlane(buf * (KT * RB) + first * RB);
      load_to_lds(bytes_on(kb + (EXACT || kc < hd ? kc : 0), off[p]), kl_at + to);
      load_to_lds(bytes_on(vb + (EXACT || vc < hd ? vc : 0), off[p]), vl_at + to);
    }
    all = __all(all);
    if (lane == 0) whole[buf][wave] = all;
  };
  // Where a lane reads: keys of row `col`, chunk 2 k + half, at key_at ^ 32 k; values of row
  // 4 half + (lane & 15) / 4, output tile d, at value_at ^ 64 d.
  const int key_at = col * RB + ((half ^ key_swizzle(col)) << 4);
  const int vrow = 4 * half + ((lane & 15) >> 2);
  const int value_at =
      vrow * RB + (((((lane >> 4) & 1) * 2 + ((lane & 3) >> 1)) ^ value_swizzle(vrow)) << 4) + (lane & 1) * 8;

  // The queries' waits are here: inside the loop they would wait for its loads.
#pragma unroll
  for (int k = 0; k < KC; ++k) asm volatile("" : "+v"(q[k]));
  constexpr int kOnes = T::code == SY_BF16 ? 0x3f803f80 : 0x3c003c00;
  constexpr float kLag = T::code == SY_F16 ? 15.0f : 8.0f;  // of the reference behind the maximum: 7 and 8
  const i32x4_t ones = {kOnes, kOnes, kOnes, kOnes};
  float m = -INFINITY, l = 0.0f;
  f32x16_t o[MD];
#pragma unroll
  for (int d = 0; d < MD; ++d) o[d] = f32x16_t{};

  if (t0 < t1) {
    ask_ids(t0);
    ask(t0);
    ask_ids(min(t0 + 1, t1 - 1));
  }
  for (int t = t0; t < t1; ++t) {
    const int buf = (t - t0) & 1;
    const bool own = t >= pre_tiles;
    const int j0 = (own ? t - pre_tiles : t) * KT;
    wait_loads();  // tile t, which was asked for a whole tile ago
    __syncthreads();
    if (t + 1 < t1) {
      ask(t + 1);  // into the buffer that was read before the barrier
      ask_ids(min(t + 2, t1 - 1));
    }
    uint64_t there = ~0ull, odd = 0;
    const i32x4_t w4 = *reinterpret_cast<const i32x4_t*>(whole[buf]);
    if ((w4[0] & w4[1] & w4[2] & w4[3]) == 0 || (own && j0 + KT > wg_least)) {
      // Values of keys that are not there become zero, and so do those that some rows must
      // not see and that hold an infinity or NaN (0 times one is none): the rows that see
      // them add them on their own. Four threads a row.
      const int row = tid / 4, j = j0 + row;
      const int32_t* const pages = own ? own_pages : a.prefix_pages;
      const int page = pages[min(j >> c.page_shift, own ? own_last : (plen - 1) >> c.page_shift)];
      const bool ok = (unsigned)page < (unsigned)c.n_pages && j < (own ? most : plen);
      i32x4_t* const at = reinterpret_cast<i32x4_t*>(vl + buf * (KT * RB) + row * RB + tid % 4 * (RB / 4));
      bool bad = false;
#pragma unroll
      for (int x = 0; x < CPR / 4; ++x) bad = bad || nonfinite<T>(at[x]);
      bad = (__ballot(bad) >> (lane & ~3) & 15) != 0;
      if (bad || !ok) {
#pragma unroll
        for (int x = 0; x < CPR / 4; ++x) at[x] = i32x4_t{0, 0, 0, 0};
      }
      if (tid % 4 == 0) flags[row] = (ok ? 1 : 0) | (ok && bad ? 2 : 0);
      __syncthreads();
      const int flag = flags[lane];
      there = __ballot(flag & 1);
      odd = __ballot(flag & 2);
    }
    if (active && (!own || j0 < wmost)) {
      f32x16_t st[2] = {f32x16_t{}, f32x16_t{}};
#pragma unroll
      for (int k = 0; k < KC; ++k) {
        if (!EXACT && k * 16 >= hd) continue;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          i32x4_t w = *reinterpret_cast<const i32x4_t*>(kl + buf * (KT * RB) + x * 32 * RB + (key_at ^ (k * 32)));
          if (!EXACT && (2 * k + half) * 8 >= hd) w = i32x4_t{0, 0, 0, 0};
          st[x] = mma32<T>(w, q[k], st[x]);
        }
      }
      const bool full = ~there == 0 && (!own || j0 + KT <= least);
      if (__builtin_expect(!full, 0)) {
        asm volatile("" ::: "memory");  // a branch: selects would cost every tile
        const int lim = own ? limit - j0 : KT;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const uint32_t bits = (uint32_t)(there >> (32 * x)) >> (4 * half);
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int at = 8 * (e / 4) + e % 4;
            const bool see = ((bits >> at) & 1u) != 0 && x * 32 + at + 4 * half < lim;
            st[x][e] = see ? st[x][e] : -INFINITY;
          }
        }
      }
      float top = fmaxf(st[0][0], st[1][0]);
#pragma unroll
      for (int e = 1; e < 16; ++e) top = fmaxf(fmaxf(top, st[0][e]), st[1][e]);
      {
        const uint32_t v = __float_as_uint(top);
        const auto sw = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        top = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])) * sl;
      }
      if (__any(top > m + kLag)) {
        const float mn = fmaxf(m, reference_of<T, 7>(top));
        const float sc = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.0f : mn));
        m = mn;
        l *= sc;
#pragma unroll
        for (int d = 0; d < MD; ++d) o[d] *= sc;
      }
      const float mu = m == -INFINITY ? 0.0f : m;
      // A product that is not rounded before the reference is taken off it may pass a rounded
      // one: by an eighth where that is below 2^22, by more than the weights' room above.
      // (The branch costs nothing at widths of 64 and 128 and 1 to 2 % at 256. Padded widths
      // round every product instead, 2 to 4 %: the branch's registers cost 72 to 248 20 to 50 %.)
      float sx = sl;
      if (EXACT && __builtin_expect(__any(fabsf(mu) >= kWholeScores), 0)) {
        asm volatile("" ::: "memory");
        sx = 1.0f;
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int e = 0; e < 16; ++e) st[x][e] *= sl;
      }
      i32x4_t p16[4];
      [[maybe_unused]] i32x4_t p16r[4];
      float sum = 0.0f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float pf[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = st[k / 2][(k % 2) * 8 + e];
          pf[e] = __builtin_amdgcn_exp2f(EXACT ? fmaf(x, sx, -mu) : product(x, sl) - mu);
        }
        // Weights are rounded to the values' dtype for the product (at most half a step,
        // independent of one another), and their sum is of the rounded ones: two a
        // v_dot2, half the additions. As two numbers (TWO) they would make three products
        // of the two that bound this kernel: error 2.0e-3 or 1.64e-3 in bf16, 2.9e-4 or
        // 2.1e-4 in fp16, and prompts 76 or 93 us, pieces of them 198 or 272. A prefix's
        // pass, whose rows are few, takes them as k_attend does: there the products wait
        // for memory (64 rows behind 4096 tokens 38.1 and 39.0 us, 16 of 4 heads each
        // behind 30011 47.4 and 50.9), and a token's result does not depend on how many
        // others share the prefix.
        p16[k] = pack<T>(pf);
        if constexpr (TWO) {
          float rest[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            rest[e] = pf[e] - elem<T>(p16[k], e);
            sum += pf[e];
          }
          p16r[k] = pack<T>(rest);
        } else {
          sum = dot<T>(p16[k], ones, sum);
        }
      }
      l += sum;
      if (__builtin_expect(odd != 0, 0)) {
        asm volatile("" ::: "memory");
#pragma unroll 1
        for (int j = 0; j < KT; ++j) {
          if ((odd >> j & 1) == 0) continue;
          const int e = 8 * (j >> 4) + 4 * ((j >> 3) & 1) + (j & 3);  // of the 32 weights of a lane
          const auto weight = [&](const i32x4_t (&p)[4]) {
            int word = p[0][0];
#pragma unroll
            for (int x = 1; x < 16; ++x) word = e >> 1 == x ? p[x / 4][x % 4] : word;
            word = __shfl(word, col + 32 * ((j >> 2) & 1));
            const i32x4_t w4 = {word, 0, 0, 0};
            return (e & 1) ? elem<T>(w4, 1) : elem<T>(w4, 0);
          };
          float pv = weight(p16);
          if constexpr (TWO) pv += weight(p16r);
          const int id = (own ? own_pages : a.prefix_pages)[(j0 + j) >> c.page_shift];
          const S* const vr = bytes_on(vb, row_at(c, id, j0 + j));
          if (own && j0 + j >= limit) continue;
#pragma unroll
          for (int d = 0; d < MD; ++d)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int ch = d * 32 + 8 * x + 4 * half;
              if (!EXACT && ch >= hd) continue;
              i32x4_t v4 = {0, 0, 0, 0};
              __builtin_memcpy(&v4, vr + ch, 8);
#pragma unroll
              for (int i = 0; i < 4; ++i) o[d][4 * x + i] = fmaf(pv, elem<T>(v4, i), o[d][4 * x + i]);
            }
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        i32x4_t w[MD];
#pragma unroll
        for (int d = 0; d < MD; ++d) {
          if (!EXACT && d * 32 >= hd) continue;
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            char* const from = vl + buf * (KT * RB) + (16 * k + 8 * x) * RB + (value_at ^ (d * 64));
            const i16x4_t v4 =
                __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4_t*)from);
            const i32x2_t v2 = __builtin_bit_cast(i32x2_t, v4);
            w[d][2 * x] = v2[0];
            w[d][2 * x + 1] = v2[1];
          }
          o[d] = mma32<T>(w[d], p16[k], o[d]);
        }
        if constexpr (TWO) {  // (no product next to the one whose sum it adds to)
#pragma unroll
          for (int d = 0; d < MD; ++d) {
            if (!EXACT && d * 32 >= hd) continue;
            o[d] = mma32<T>(w[d], p16r[k], o[d]);
          }
        }
      }
    }
  }

  {
    const uint32_t v = __float_as_uint(l);
    const auto sw = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    l = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
  }
  const int base = f.splits == 1 || f.pre ? 0 : total_of(b, [&](int x) { return flash_tiles(c, f, plen, x); });
  if (w0 + col > last) return;
  // Sequences that overlap have more tiles than there are places for.
  if (f.splits > 1 && base + rtile >= f.tiles) return;
  if (direct) {
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    S* const op = static_cast<S*>(a.out) + out_row * hd;
#pragma unroll
    for (int d = 0; d < MD; ++d)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int ch = d * 32 + 8 * x + 4 * half;
        if (!EXACT && ch >= hd) continue;
        float y[8] = {};
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = l == 0.0f ? 0.0f : o[d][4 * x + i] * inv;
        const i32x4_t v4 = pack<T>(y);
        *reinterpret_cast<i32x2_t*>(op + ch) = i32x2_t{v4[0], v4[1]};
      }
    return;
  }
  const bool uncut = f.splits == 1;
  const int64_t slot = uncut ? out_row : flash_slot(c, f, base + rtile, h, split) + (w0 - r0) + col;
  float* const po = (uncut ? row_o : f.o) + slot * hd;
#pragma unroll
  for (int d = 0; d < MD; ++d)
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int ch = d * 32 + 8 * x + 4 * half;
      if (EXACT || ch < hd)
        *reinterpret_cast<f32x4_t*>(po + ch) =
            f32x4_t{o[d][4 * x], o[d][4 * x + 1], o[d][4 * x + 2], o[d][4 * x + 3]};
    }
  if (half == 0) {
    float* const pm = (uncut ? row_ml : f.ml) + slot * 2;
    pm[0] = m;
    pm[1] = l;
  }
}

template <class T, int HD, bool EXACT>
__global__ void __launch_bounds__(kBlock, HD <= 128 ? 2 : 1)
k_flash(const AttendArgs a, const Flash f, const int direct, const int zero, float* const row_o, float* const row_ml) {
  __shared__ __align__(16) char shared[flash_lds<HD>()];
  flash<T, HD, EXACT, false>(a, f, direct, row_o, row_ml, blockIdx.x, shared);
  if (zero) zero_outside<T>(a);
}

// Where whole results of rows go that are yet to be joined: [n_tok][heads][hd], and m, l.
struct Rows {
  float *o, *ml;
};

// Both in one launch, where a call may bring sequences of either kind, or the pass over a
// shared prefix goes with that over the sequences' own keys (PRE): the many rows' long
// workgroups first, the equal runs of the few rows fill up behind them.
template <class T, int HD, bool EXACT, bool PRE>
__global__ void __launch_bounds__(kBlock, HD <= 128 ? 2 : 1)
k_both(const AttendArgs a, const Cut u, const Flash f, const int direct_u, const int direct_f, const int zero,
       const Rows ru, const Rows rf) {
  __shared__ __align__(16) char shared[flash_lds<HD>() > attend_lds<T, HD>() ? flash_lds<HD>() : attend_lds<T, HD>()];
  const int many = f.tiles * a.c.kv_heads * f.splits;
  if ((int)blockIdx.x < many)
    flash<T, HD, EXACT, PRE>(a, f, direct_f, rf.o, rf.ml, blockIdx.x, shared);
  else
    attend<T, HD, 1, EXACT>(a, u, direct_u, ru.o, ru.ml, blockIdx.x - many, shared);
  if (zero) zero_outside<T>(a);
}

// ---------------------------------------------------------------------- merge
//
// Joins the partial results of rows that several workgroups worked on, and those of a
// prefix with a sequence's own: out = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i. A
// workgroup takes some heads of one token; hd / 4 threads read a partial result, so many
// results are read at once, and every thread's sum runs in the order of the keys. Rows
// that one workgroup finished are left alone. Bound by latency: lengths, statistics and
// the first results are loads one after another (32 tokens of 16 heads, one to three results
// each, 6.4 us, of 7.3 with the sums and results asked for one by one).
struct Parts {  // `count` results, number k at row at + k step (+ second at k = 0); one: the row's own
  int count;
  int64_t at, step, second;
};
struct Shares {
  int per_head, base, share;
};

__device__ __forceinline__ Shares shares_of(const CacheArgs& c, const Cut& u, int plen, int b) {
  const auto count = [&](int x) { return units_of(c, u, plen, x); };
  Shares x;
  x.per_head = total_of(u.pre ? 1 : c.n_seq, count);
  x.base = u.pre ? 0 : total_of(b, count);
  x.share = share_of(u, x.per_head * c.kv_heads);
  return x;
}
// Row r of sequence s and kv head h as k_attend left it: in the second slot of the worker
// in whose run the segment begins and the first slots of the next ones, or whole.
// (Workers past the last are those of sequences that overlap, whose numbers of units may be
// past all bounds: then results are some numbers, but read from where there are any.)
__device__ __forceinline__ Parts parts_of(const CacheArgs& c, const Cut& u, const Shares& x, const Seq& s, int h,
                                          int r) {
  const int rtile = r / u.rt, k = tiles_of(u, c.group, s).key_tiles;
  const int at = h * x.per_head + x.base + rtile * k;
  const int first = u.least != 0 ? clamp(at / x.share, 0, u.workers - 1) : 0;
  const int count = u.least != 0 ? clamp((at + k - 1) / x.share - first + 1, 1, u.workers - first) : 1;
  Parts p;
  p.count = __builtin_amdgcn_readfirstlane(count);
  p.at = 2 * (int64_t)first * u.rs + (r - rtile * u.rt);
  p.step = 2 * u.rs;
  p.second = u.rs;
  return p;
}
// The same as k_flash left it.
__device__ __forceinline__ Parts flash_parts(const CacheArgs& c, const Flash& f, int base, int h, int r) {
  const int rtile = r / kFlashRows;
  Parts p;
  p.count = f.splits;
  p.at = flash_slot(c, f, base + rtile, h, 0) + (r - rtile * kFlashRows);
  p.step = kFlashRows;
  p.second = 0;
  return p;
}

constexpr int kMostParts = 1024;  // of a row, of one pass

// The prefix's pass is one of pre (k_attend's) and fpre (k_flash's), by which has splits.
struct JoinArgs {
  Cut own, pre;
  Flash fown, fpre;
  int has_pre;  // 0, 1: k_attend's, 2: k_flash's
  int per_wg;   // heads a workgroup
  int few;      // tokens a sequence to look at, where only k_attend's rows are left; else 0
  int many;     // workgroups for k_flash's cut rows, where there is no prefix to join
  float *row_o, *row_ml, *pre_o, *pre_ml;
};

template <class T>
__device__ __forceinline__ void merge(const AttendArgs& a, const JoinArgs& g, const int block) {
  using S = typename T::storage;
  const CacheArgs& c = a.c;
  __shared__ float weight[2 * kMostParts], mass[2 * kMostParts];
  __shared__ f32x4_t fold[kBlock];
  __shared__ float tops[kWaves], sums[kWaves];
  const int tid = threadIdx.x;
  const int plen = (int)a.prefix_len;
  const int slices = (c.heads + g.per_wg - 1) / g.per_wg;
  int tok = block / slices, b;
  const int slice = block - tok * slices;
  Seq s;
  if (g.few != 0) {
    b = tok / g.few;
    s = seq_of(c, b);
    const int i = tok - b * g.few;
    if (i >= s.n || s.n * c.group > g.own.few) return;
    tok = s.row0 + i;
  } else {
    b = find_seq(c, tok);
    if (b < 0) return;
    s = seq_of(c, b);
  }
  const bool flash = s.n * c.group > g.own.few;
  Shares xo{}, xp{};
  int fbase = 0;
  if (flash)
    fbase = total_of(b, [&](int x) { return flash_tiles(c, g.fown, plen, x); });
  else if (g.own.least != 0)
    xo = shares_of(c, g.own, 0, b);
  Seq ps{};
  if (g.has_pre != 0) ps = pass_seq(c, 1, plen, 0);
  if (g.has_pre == 1) xp = shares_of(c, g.pre, plen, 0);
  const int lpr = c.hd / 4, groups = kBlock / lpr;
  const int grp = tid / lpr, ch = (tid - grp * lpr) * 4;
  for (int hq = slice * g.per_wg; hq < min((slice + 1) * g.per_wg, c.heads); ++hq) {
    const int64_t row = (int64_t)tok * c.heads + hq;
    const int h = hq / c.group, gi = hq - h * c.group;
    const int r = (tok - s.row0) * c.group + gi;
    const Parts mine = flash ? flash_parts(c, g.fown, fbase, h, r) : parts_of(c, g.own, xo, s, h, r);
    if (g.has_pre == 0 && mine.count == 1) continue;
    if (flash && g.fown.splits > 1 && fbase + r / kFlashRows >= g.fown.tiles) continue;
    Parts front{};
    const int rp = (tok - ps.row0) * c.group + gi;
    if (g.has_pre == 1) front = parts_of(c, g.pre, xp, ps, h, rp);
    else if (g.has_pre == 2) front = flash_parts(c, g.fpre, 0, h, rp);
    const float* const mo = mine.count == 1 ? g.row_o : flash ? g.fown.o : g.own.o;
    const float* const mm = mine.count == 1 ? g.row_ml : flash ? g.fown.ml : g.own.ml;
    const float* const fo = front.count == 1 ? g.pre_o : g.has_pre == 2 ? g.fpre.o : g.pre.o;
    const float* const fm = front.count == 1 ? g.pre_ml : g.has_pre == 2 ? g.fpre.ml : g.pre.ml;
    const int n = front.count + mine.count;  // the prefix's first
    const auto at = [&](int i) -> int64_t {
      const bool f = i < front.count;
      if ((f ? front.count : mine.count) == 1) return row;
      const int k = f ? i : i - front.count;
      return (f ? front.at : mine.at) + k * (f ? front.step : mine.step) +
             (k == 0 ? (f ? front.second : mine.second) : 0);
    };
    // The first result is on its way while its weight is worked out.
    const auto part = [&](int i) {
      return *reinterpret_cast<const f32x4_t*>((i < front.count ? fo : mo) + at(i) * c.hd + ch);
    };
    f32x4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
    const bool mine_too = grp < groups && grp < n;
    if (mine_too) o = part(grp);
    float m = -INFINITY;
    for (int i = tid; i < n; i += kBlock) {
      const float* const x = (i < front.count ? fm : mm) + at(i) * 2;
      weight[i] = x[0];
      mass[i] = x[1];
      m = fmaxf(m, x[0]);
    }
#pragma unroll
    for (int k = 32; k >= 1; k /= 2) m = fmaxf(m, __shfl_xor(m, k));
    if ((tid & 63) == 0) tops[wave_id()] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) m = fmaxf(m, tops[w]);
    const float mu = m == -INFINITY ? 0.0f : m;
    float sum = 0.0f;
    for (int i = tid; i < n; i += kBlock) {
      const float l = mass[i];
      // NaN scores leave no maximum, but the row is not an empty one.
      const float w = l != l ? 1.0f : __builtin_amdgcn_exp2f(weight[i] - mu);
      weight[i] = w;
      sum = fmaf(l, w, sum);
    }
#pragma unroll
    for (int k = 32; k >= 1; k /= 2) sum += __shfl_xor(sum, k);
    if ((tid & 63) == 0) sums[wave_id()] = sum;
    __syncthreads();
    sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) sum += sums[w];
    if (mine_too) {
      o *= weight[grp];
#pragma unroll 4
      for (int i = grp + groups; i < n; i += groups) o += weight[i] * part(i);
    }
    fold[tid] = o;
    __syncthreads();
    if (tid < lpr) {
      for (int k = 1; k < min(groups, n); ++k) o += fold[k * lpr + tid];
      float f[T::ce] = {};
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = sum == 0.0f ? 0.0f : o[e] / sum;
      const i32x4_t x4 = pack<T>(f);
      __builtin_memcpy(static_cast<S*>(a.out) + row * c.hd + ch, &x4, 4 * sizeof(S));
    }
    __syncthreads();
  }
}

// The same for k_flash's cut rows where there is no prefix to join: a workgroup takes 32
// rows of a tile and kv head, hd / 4 threads one row's few results, without LDS or barriers.
// Bound by reading the partial results once, with enough workgroups to hide that the
// statistics come first (64 tiles of 8 kv heads, all 128 rows in one workgroup and the few
// rows' merge in a launch of its own: 36 us; together in this one 18).
constexpr int kMergeRows = 32;
template <class T>
__device__ __forceinline__ void merge_flash(const AttendArgs& a, const Flash& f, const int block) {
  using S = typename T::storage;
  const CacheArgs& c = a.c;
  constexpr int kParts = kFlashRows / kMergeRows;
  const int i0 = block % kParts * kMergeRows, rest = block / kParts;
  const int h = rest % c.kv_heads, tile = rest / c.kv_heads;
  int b, base;
  if (!locate(c.n_seq, tile, [&](int x) { return flash_tiles(c, f, 0, x); }, &b, &base)) return;
  const Seq s = seq_of(c, b);
  const int r0 = (tile - base) * kFlashRows;
  const int rows = min(kFlashRows, s.n * c.group - r0);
  const int64_t slot = flash_slot(c, f, tile, h, 0);
  const int lpr = c.hd / 4, groups = kBlock / lpr;
  const int grp = threadIdx.x / lpr, ch = (threadIdx.x - grp * lpr) * 4;
  if (grp >= groups) return;
  for (int i = i0 + grp; i < min(rows, i0 + kMergeRows); i += groups) {
    const float* const ml = f.ml + (slot + i) * 2;
    float m = -INFINITY;
    for (int k = 0; k < f.splits; ++k) m = fmaxf(m, ml[k * (2 * kFlashRows)]);
    const float mu = m == -INFINITY ? 0.0f : m;
    float sum = 0.0f;
    f32x4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int k = 0; k < f.splits; ++k) {
      const float l = ml[k * (2 * kFlashRows) + 1];
      const float w = l != l ? 1.0f : __builtin_amdgcn_exp2f(ml[k * (2 * kFlashRows)] - mu);
      sum = fmaf(l, w, sum);
      o += w * *reinterpret_cast<const f32x4_t*>(f.o + (slot + i + (int64_t)k * kFlashRows) * c.hd + ch);
    }
    const int r = r0 + i, t = r / c.group;
    const int64_t row = (int64_t)(s.row0 + t) * c.heads + h * c.group + (r - t * c.group);
    float y[T::ce] = {};
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = sum == 0.0f ? 0.0f : o[e] / sum;
    const i32x4_t x4 = pack<T>(y);
    __builtin_memcpy(static_cast<S*>(a.out) + row * c.hd + ch, &x4, 4 * sizeof(S));
  }
}

template <class T>
__global__ void __launch_bounds__(kBlock) k_merge(const AttendArgs a, const JoinArgs g) {
  if ((int)blockIdx.x < g.many) merge_flash<T>(a, g.fown, blockIdx.x);
  else merge<T>(a, g, (int)blockIdx.x - g.many);
}

// ----------------------------------------------------------------------- host

// Tokens at most of a sequence that one workgroup reads whole, by the number of workgroups
// that gives. One takes 8 us for 256 tokens, 12 for 512, 19 for 1024 and 33 for 2048 (37
// GB/s, which is what a CU's loads reach: eight waves take as long as four); shared out, 16
// for any of them, 8 of which are the second launch. More of them share memory's rate: 128
// over 1024 tokens 19.4 us whole, 22 shared out, over 2048 33 and 31; 256 over 2048 tokens
// 43 and 49 to 53, over any lengths up to 2048 34 and 36, or 35 and 41 (8 kv heads of 32).
// With more than two a CU the long ones among sequences of any lengths may start last: 1024
// over up to 2048 tokens 130 us whole, 116 shared out (180 and 190 where all are as long),
// 2048 over up to 1024 125 and 129. Next to a prefix's pass they start behind it anyway: 128
// over up to 1024 tokens behind 30011 shared ones 52.0 us whole, 51.3 shared out.
int whole_tokens(int64_t workgroups, bool beside) {
  return beside || workgroups < 128 ? 512 : workgroups >= 256 && workgroups < 512 ? 2048 : 1024;
}

constexpr int64_t kMost = 0x7fffffff;
constexpr int64_t kMostGroups = 0xffffff;  // workgroups of a launch, which has less than 2^32 threads

// What a call launches: k_attend over the sequences of few rows, k_flash over the others,
// one of them over a shared prefix, and the merge of what was cut.
struct Plan {
  bool ok;
  bool attend, flash;  // the sequences' own keys
  int pre;             // a pass over the prefix: 0 none, 1 k_attend, 2 k_flash
  int direct_attend, direct_flash;
  bool merge, merge_flash;
  int merge_few;
  Cut own, cpre;
  Flash fown, fpre;
  int64_t bytes;
  int64_t row_o, row_ml, pre_o, pre_ml;  // float offsets, as the o and ml of the passes
};

bool cut(const CacheArgs& c, int dtype, bool pre, bool beside, int64_t len, int few, int nt, int cus, Cut* u) {
  u->pre = pre;
  u->few = few;
  u->kt = dtype == SY_F32 ? 16 : 32;
  u->rt = 16 * nt;
  const int64_t rows = (int64_t)c.n_tok * c.group;
  const int64_t keys = std::max<int64_t>(1, (len + u->kt - 1) / u->kt);
  const bool even = !pre && c.starts == nullptr;
  int64_t tiles;  // row tiles, at most
  if (pre) tiles = (rows + u->rt - 1) / u->rt;
  else if (even) tiles = c.n_seq * (((int64_t)c.each * c.group + u->rt - 1) / u->rt);
  else if (few <= u->rt) tiles = std::min<int64_t>(c.n_seq, rows);
  else tiles = rows / u->rt + std::min<int64_t>(c.n_seq, rows);
  if (tiles > kMost / 2 / keys || tiles * keys > kMost / 2 / c.kv_heads) return false;
  u->rs = (int)std::min<int64_t>(u->rt, even ? (int64_t)c.each * c.group : rows);
  if (even && keys * u->kt <= whole_tokens(tiles * c.kv_heads, beside)) {
    u->least = 0;
    u->workers = (int)(tiles * c.kv_heads);
    return true;
  }
  u->least = 2 * kWaves;
  const int64_t units = tiles * keys * c.kv_heads;
  const int64_t full = std::min<int64_t>(kMostParts, (int64_t)cus * (nt == 1 && c.hd <= 128 ? 2 : 1));
  u->workers = (int)std::max<int64_t>(1, std::min(full, (units + u->least - 1) / u->least));
  return true;
}

// Parts of a row tile's keys: the number that promises the shortest time. A CU works
// through its workgroups' tiles at a rate (measured: 1.45 us a tile of 64 keys and 128 rows
// of 128, 0.72 of 64, 3.2 of 256), a workgroup alone no faster than 1.2 us a tile; the last
// workgroups leave CUs idle for part of their time; cut rows are written, read and joined.
// Prompts see half of their own tokens on average, and sequences are rarely of one length.
// A prefix's parts are all as long, and the sequences' own keys fill what they leave idle:
// there the CU with the most of them counts (30011 tokens behind 8 kv heads: 32 parts, one a
// CU, 53.3 us; 24 58.0; 48, two on half of the CUs, 54.8).
bool flash_cut(const CacheArgs& c, bool pre, bool virt, int64_t prefix_len, int few, int cus, Flash* f) {
  f->pre = pre;
  f->virt = virt;
  f->few = few;
  const int64_t rows = (int64_t)c.n_tok * c.group;
  if (pre) f->tiles = (int)((rows + kFlashRows - 1) / kFlashRows);
  else if (c.starts == nullptr)
    f->tiles = (int)std::min<int64_t>(kMost, c.n_seq * (((int64_t)c.each * c.group + kFlashRows - 1) / kFlashRows));
  else f->tiles = (int)(rows / kFlashRows + std::min<int64_t>(c.n_seq, rows / (few + 1)));
  const int64_t grid = (int64_t)f->tiles * c.kv_heads;
  const int64_t keys = (pre ? prefix_len : c.cap + (virt ? prefix_len : 0));
  const double longest = (double)keys / kFlashKeys;
  const double mean = 0.8 * std::max(longest / 2, longest - 0.5 * c.n_tok / c.n_seq / kFlashKeys);
  const int places = c.hd <= 64 ? 3 : c.hd <= 128 ? 2 : 1;
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>(64, keys / (2 * kFlashKeys)));
  const double tile_us = c.hd <= 64 ? 0.72 : c.hd <= 128 ? 1.45 : 3.2;
  const double row_us = (double)rows * c.kv_heads * c.hd * 8 / 4e6;  // fp32 results out and in again at 4 TB/s
  f->splits = 1;
  double best = 0.0;
  for (int n = 1; n <= most; ++n) {
    const double work = pre ? (double)((grid * n + cus - 1) / cus) * longest / n * tile_us
                            : std::max(grid * mean * tile_us / cus, longest / n * 1.2) +
                                  0.25 * longest / n * tile_us * places;
    const double cost = work + (n > 1 ? 6.0 + n * row_us : 0.0);
    if (n == 1 || cost < best) {
      best = cost;
      f->splits = n;
    }
  }
  f->fold = cus / (c.kv_heads * f->splits);
  return grid * f->splits <= kMost / kFlashRows;  // (of rows, and so of the merge's workgroups)
}

// Workgroups of the merge's launch, and the heads that one of them takes: one, until there
// are far more rows than fit the device at once.
int64_t merge_groups(const CacheArgs& c, const Plan& p, int* per_wg) {
  const int64_t toks = p.merge_few ? (int64_t)c.n_seq * p.merge_few : c.n_tok;
  const int heads = (int)std::min<int64_t>(c.heads, std::max<int64_t>(1, toks * c.heads / 8192));
  if (per_wg != nullptr) *per_wg = heads;
  return (p.merge_flash ? (int64_t)p.fown.tiles * c.kv_heads * (kFlashRows / kMergeRows) : 0) +
         (p.merge ? toks * ((c.heads + heads - 1) / heads) : 0);
}

Plan plan_attend(const CacheArgs& c, int64_t prefix_len, int dtype) {
  Plan p{};
  int cus = 0;
  if (cu_count(&cus) != hipSuccess || cus < 1) cus = 1;
  const int64_t rows = (int64_t)c.n_tok * c.group;  // of a kv head
  if (rows * c.kv_heads > kMost / 2) return p;
  const int64_t avg = (rows + c.n_seq - 1) / c.n_seq;
  p.ok = true;
  if (dtype == SY_F32) {
    const int nt = avg <= 16 ? 1 : c.hd > 128 ? 1 : 2;
    p.attend = true;
    p.pre = prefix_len > 0 ? 1 : 0;
    p.ok = cut(c, dtype, false, false, c.cap, (int)kMost, nt, cus, &p.own);
    const int nt_pre = rows <= 16 || c.hd > 128 ? 1 : 2;
    if (p.ok && p.pre) p.ok = cut(c, dtype, true, false, prefix_len, (int)kMost, nt_pre, cus, &p.cpre);
  } else {
    // Up to 16 rows are k_attend's. A prefix has a pass of its own where sequences bring
    // few rows, so that it is read once for all; else its keys are part of every
    // sequence's, whose rows share them anyway.
    const bool shared = prefix_len > 0 && avg <= 16;
    const bool virt = prefix_len > 0 && !shared;
    const int few = virt ? 0 : 16;
    p.attend = !virt && (c.starts != nullptr || avg <= 16);
    p.flash = c.starts != nullptr ? rows > few : avg > few;
    p.own.few = few;
    if (p.attend) p.ok = cut(c, dtype, false, shared && rows > 16, c.cap, few, 1, cus, &p.own);
    if (p.ok && p.flash) p.ok = flash_cut(c, false, virt, prefix_len, few, cus, &p.fown);
    p.pre = !shared ? 0 : rows <= 16 ? 1 : 2;
    if (p.ok && p.pre == 1) p.ok = cut(c, dtype, true, false, prefix_len, (int)kMost, 1, cus, &p.cpre);
    if (p.ok && p.pre == 2) p.ok = flash_cut(c, true, false, prefix_len, 0, cus, &p.fpre);
  }
  if (!p.ok) return p;
  p.direct_attend = p.pre == 0;
  p.direct_flash = p.pre == 0 && p.fown.splits == 1;
  const bool cut_attend = p.attend && p.own.least != 0 && c.cap > p.own.kt;
  p.merge = p.pre != 0 || cut_attend;
  p.merge_flash = p.pre == 0 && p.flash && p.fown.splits > 1;
  p.merge_few = p.pre == 0 && p.flash ? std::max(1, 16 / c.group) : 0;
  const auto flash_groups = [&](const Flash& f) { return (int64_t)f.tiles * c.kv_heads * f.splits; };
  const int64_t own_groups = p.attend ? p.own.workers : 0;
  p.ok = own_groups + std::max(p.flash ? flash_groups(p.fown) : 0, p.pre == 2 ? flash_groups(p.fpre) : 0) <= kMostGroups &&
         (int64_t)p.cpre.workers <= kMostGroups && merge_groups(c, p, nullptr) <= kMostGroups;
  if (!p.ok) return p;
  int64_t at = 0;
  const auto take = [&](int64_t n) {
    const int64_t was = at;
    at += (n + 3) / 4 * 4;
    return was;
  };
  const auto slots = [&](auto& u, int64_t n) {
    u.o = reinterpret_cast<float*>(take(n * c.hd) * sizeof(float));
    u.ml = reinterpret_cast<float*>(take(n * 2) * sizeof(float));
  };
  if (p.attend && p.own.least != 0) slots(p.own, 2 * (int64_t)p.own.workers * p.own.rs);
  if (p.flash && p.fown.splits > 1)
    slots(p.fown, (int64_t)p.fown.tiles * c.kv_heads * p.fown.splits * kFlashRows);
  if (p.pre == 1) slots(p.cpre, 2 * (int64_t)p.cpre.workers * p.cpre.rs);
  if (p.pre == 2 && p.fpre.splits > 1)
    slots(p.fpre, (int64_t)p.fpre.tiles * c.kv_heads * p.fpre.splits * kFlashRows);
  if (p.pre != 0) {
    const int64_t n = (int64_t)c.n_tok * c.heads;
    p.row_o = take(n * c.hd);
    p.row_ml = take(n * 2);
    p.pre_o = take(n * c.hd);
    p.pre_ml = take(n * 2);
  }
  p.bytes = at * (int64_t)sizeof(float);
  return p;
}

template <class T, int HD, int NT>
hipError_t attend_t(const AttendArgs& a, const Cut& u, int direct, int zero, const Rows& r, hipStream_t s) {
  const dim3 grid((unsigned)u.workers);
  if (a.c.hd == HD)
    hipLaunchKernelGGL((k_attend<T, HD, NT, true>), grid, dim3(kBlock), 0, s, a, u, direct, zero, r.o, r.ml);
  else
    hipLaunchKernelGGL((k_attend<T, HD, NT, false>), grid, dim3(kBlock), 0, s, a, u, direct, zero, r.o, r.ml);
  return hipGetLastError();
}

template <class T>
hipError_t attend_pass(const AttendArgs& a, const Cut& u, int direct, int zero, const Rows& r, hipStream_t s) {
  constexpr int two = T::code == SY_F32 ? 2 : 1;  // fp32 rows in two groups of 16, up to 128 wide
  const bool one = u.rt == 16;
  if (a.c.hd <= 64)
    return one ? attend_t<T, 64, 1>(a, u, direct, zero, r, s) : attend_t<T, 64, two>(a, u, direct, zero, r, s);
  if (a.c.hd <= 128)
    return one ? attend_t<T, 128, 1>(a, u, direct, zero, r, s) : attend_t<T, 128, two>(a, u, direct, zero, r, s);
  return attend_t<T, 256, 1>(a, u, direct, zero, r, s);
}

template <class T, int HD>
hipError_t flash_t(const AttendArgs& a, const Flash& f, int direct, int zero, const Rows& r, hipStream_t s) {
  const dim3 grid((unsigned)(f.tiles * a.c.kv_heads * f.splits));
  if (a.c.hd == HD)
    hipLaunchKernelGGL((k_flash<T, HD, true>), grid, dim3(kBlock), 0, s, a, f, direct, zero, r.o, r.ml);
  else
    hipLaunchKernelGGL((k_flash<T, HD, false>), grid, dim3(kBlock), 0, s, a, f, direct, zero, r.o, r.ml);
  return hipGetLastError();
}

template <class T>
hipError_t flash_pass(const AttendArgs& a, const Flash& f, int direct, int zero, const Rows& r, hipStream_t s) {
  if constexpr (T::code == SY_F32) {
    return hipErrorInvalidConfiguration;
  } else {
    if (a.c.hd <= 64) return flash_t<T, 64>(a, f, direct, zero, r, s);
    if (a.c.hd <= 128) return flash_t<T, 128>(a, f, direct, zero, r, s);
    return flash_t<T, 256>(a, f, direct, zero, r, s);
  }
}

// k_attend's pass u and k_flash's pass f.
struct Both {
  const Cut& u;
  const Flash& f;
  int direct_u, direct_f, zero;
  Rows ru, rf;
};

template <class T, int HD, bool PRE>
hipError_t both_t(const AttendArgs& a, const Both& b, hipStream_t s) {
  const dim3 grid((unsigned)(b.u.workers + b.f.tiles * a.c.kv_heads * b.f.splits));
  if (a.c.hd == HD)
    hipLaunchKernelGGL((k_both<T, HD, true, PRE>), grid, dim3(kBlock), 0, s, a, b.u, b.f, b.direct_u, b.direct_f, b.zero,
                       b.ru, b.rf);
  else
    hipLaunchKernelGGL((k_both<T, HD, false, PRE>), grid, dim3(kBlock), 0, s, a, b.u, b.f, b.direct_u, b.direct_f, b.zero,
                       b.ru, b.rf);
  return hipGetLastError();
}

template <class T, bool PRE>
hipError_t both_pass(const AttendArgs& a, const Both& b, hipStream_t s) {
  if constexpr (T::code == SY_F32) {
    return hipErrorInvalidConfiguration;
  } else {
    if (a.c.hd <= 64) return both_t<T, 64, PRE>(a, b, s);
    if (a.c.hd <= 128) return both_t<T, 128, PRE>(a, b, s);
    return both_t<T, 256, PRE>(a, b, s);
  }
}

template <class T>
hipError_t attend_dt(const AttendArgs& a, hipStream_t s) {
  Plan p = plan_attend(a.c, a.prefix_len, T::code);
  char* const ws = static_cast<char*>(a.workspace);
  const auto place = [&](auto& u) {  // offsets -> addresses (unused where nothing is cut)
    u.o = reinterpret_cast<float*>(ws + reinterpret_cast<uintptr_t>(u.o));
    u.ml = reinterpret_cast<float*>(ws + reinterpret_cast<uintptr_t>(u.ml));
  };
  place(p.own);
  place(p.cpre);
  place(p.fown);
  place(p.fpre);
  float* const wf = static_cast<float*>(a.workspace);
  const Rows own{wf + p.row_o, wf + p.row_ml}, pre{wf + p.pre_o, wf + p.pre_ml};
  hipError_t e = hipSuccess;
  const int zero = a.fill && a.c.starts != nullptr;
  bool attend = p.attend, flash = p.flash;
  if (p.pre == 1) {
    e = attend_pass<T>(a, p.cpre, 0, 0, pre, s);
  } else if (p.pre == 2) {
    e = both_pass<T, true>(a, Both{p.own, p.fpre, p.direct_attend, 0, zero, own, pre}, s);
    attend = false;
  }
  if (e == hipSuccess && attend && flash)
    e = both_pass<T, false>(a, Both{p.own, p.fown, p.direct_attend, p.direct_flash, zero, own, own}, s), attend = flash = false;
  if (e == hipSuccess && flash) e = flash_pass<T>(a, p.fown, p.direct_flash, zero && !p.attend, own, s);
  if (e == hipSuccess && attend) e = attend_pass<T>(a, p.own, p.direct_attend, zero, own, s);
  if (e != hipSuccess) return e;
  if (!p.merge && !p.merge_flash) return e;
  const int many = p.merge_flash ? p.fown.tiles * a.c.kv_heads * (kFlashRows / kMergeRows) : 0;
  JoinArgs g{p.own, p.cpre, p.fown, p.fpre, p.pre, 1, p.merge_few, many, own.o, own.ml, pre.o, pre.ml};
  const unsigned grid = (unsigned)merge_groups(a.c, p, &g.per_wg);
  hipLaunchKernelGGL((k_merge<T>), dim3(grid), dim3(kBlock), 0, s, a, g);
  return hipGetLastError();
}

template <class T, int VE>
hipError_t append_t(const AppendArgs& a, hipStream_t s) {
  const unsigned grid = (unsigned)std::min(a.c.n_tok, 1 << 20);
  hipLaunchKernelGGL((k_append<T, VE>), dim3(grid), dim3(kBlock), 0, s, a);
  return hipGetLastError();
}

template <class T, int VE, int L>
hipError_t append_norm_t(const AppendArgs& a, hipStream_t s) {
  // A workgroup for a token, or where they are many a wave.
  const int split = a.c.n_tok < 1024 ? kWaves : 1;
  constexpr int kTokens = 1 << 23;  // of a launch
  for (int at = 0; at < a.c.n_tok; at += kTokens) {
    const int n = std::min(kTokens, a.c.n_tok - at);
    hipLaunchKernelGGL((k_append_norm<T, VE, L>), dim3((unsigned)((n + kWaves / split - 1) / (kWaves / split))),
                       dim3(kBlock), 0, s, a, split, at);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (a.c.n_tok - at <= kTokens) break;
  }
  return hipSuccess;
}

template <class T, int VE>
hipError_t append_norm_lanes(const AppendArgs& a, hipStream_t s) {
  int lanes = 1;
  while (lanes * VE < a.c.hd / 2) lanes *= 2;
  switch (lanes) {
    case 1: return append_norm_t<T, VE, 1>(a, s);
    case 2: return append_norm_t<T, VE, 2>(a, s);
    case 4: return append_norm_t<T, VE, 4>(a, s);
    case 8: return append_norm_t<T, VE, 8>(a, s);
    case 16: return append_norm_t<T, VE, 16>(a, s);
    case 32: return append_norm_t<T, VE, 32>(a, s);
    default: return hipErrorInvalidConfiguration;
  }
}

template <class T>
hipError_t append_dt(const AppendArgs& a, hipStream_t s) {
  // The widest access that the projection's rows and half a head allow.
  constexpr int CE = T::ce;
  const int64_t es = sizeof(typename T::storage);
  const auto fits = [&](int ve) {
    const int64_t w = ve * es;
    return (uintptr_t)a.qkv % w == 0 && a.tok_stride * es % w == 0 && a.head_stride * es % w == 0 &&
           a.c.hd / 2 % ve == 0;
  };
  if (a.q_gain != nullptr) {  // (the checks have seen that four elements fit)
    if constexpr (CE == 8) {
      if (!fits(8)) return append_norm_lanes<T, 4>(a, s);
    }
    return append_norm_lanes<T, CE>(a, s);
  }
  if (fits(CE)) return append_t<T, CE>(a, s);
  if (CE == 8 && fits(4)) return append_t<T, 4>(a, s);
  return append_t<T, 1>(a, s);
}

}  // namespace

hipError_t launch_append(const AppendArgs& a, int dtype, hipStream_t s) {
  if (dtype == SY_BF16) return append_dt<BF16>(a, s);
  if (dtype == SY_F16) return append_dt<F16>(a, s);
  return append_dt<F32>(a, s);
}

int64_t attend_workspace(const CacheArgs& c, int64_t prefix_len, int dtype) {
  const Plan p = plan_attend(c, prefix_len, dtype);
  return p.ok ? p.bytes : -1;
}

hipError_t launch_attend(const AttendArgs& a, int dtype, hipStream_t s) {
  if (dtype == SY_BF16) return attend_dt<BF16>(a, s);
  if (dtype == SY_F16) return attend_dt<F16>(a, s);
  return attend_dt<F32>(a, s);
}

}  // namespace sy
