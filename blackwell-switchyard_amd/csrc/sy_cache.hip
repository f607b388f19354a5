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

// One sequence's rows of the packed tensors and its keys. The prefix pass takes every
// row as one sequence over the prefix's keys.
struct Seq {
  int row0, n, len;
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
  s.len = (int)clamp(c.lengths[b], 0, (int)c.cap);
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

// Element offset of the row of token j in the cache (head 0), or -1 where a page id names no page.
__device__ __forceinline__ int64_t row_offset(const CacheArgs& c, const int32_t* pages, int j) {
  const int id = pages[j >> c.page_shift];
  if ((unsigned)id >= (unsigned)c.n_pages) return -1;
  return id * c.page_stride + (j & ((1 << c.page_shift) - 1)) * c.row_stride;
}

// --------------------------------------------------------------------- append
//
// A workgroup per token, a thread per two chunks of VE elements that turn together
// (channel i of a head's first half with channel i of its second). Bound by memory:
// every byte is read once and written once. The projection's chunks and the tables' are
// asked for before the token's sequence is looked up.
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
    int64_t dst = -1;
    if (j >= 0 && j < c.cap && at < a.n_pos) dst = row_offset(c, c.table + b * c.table_stride, j);
    for (int i = threadIdx.x; i < items; i += kBlock) {
      const int head = i / per_head;
      const int ch = (i - head * per_head) * VE;
      const S* const src = row + head * a.head_stride + ch;
      Chunk<T, VE> lo = ld_chunk<T, VE>(src);
      Chunk<T, VE> hi = ld_chunk<T, VE>(src + half);
      if (head < c.heads + c.kv_heads && dst >= 0) {
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
        if (dst < 0) {
#pragma unroll
          for (int e = 0; e < VE; ++e) lo.f[e] = hi.f[e] = __int_as_float(0x7fc00000);
        }
        out = q + ((int64_t)tok * c.heads + head) * c.hd + ch;
      } else {
        if (dst < 0) continue;
        const bool key = head < c.heads + c.kv_heads;
        const int h = head - c.heads - (key ? 0 : c.kv_heads);
        out = static_cast<S*>(key ? c.k : c.v) + dst + h * c.head_stride + ch;
      }
      st_chunk<T, VE>(out, lo);
      st_chunk<T, VE>(out + half, hi);
    }
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
// the segment's end. A run begins and ends inside at most one segment each, so two
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

template <class T> constexpr int tokens_of() { return T::code == SY_F32 ? 16 : 32; }

// How a pass over the keys is cut, the same for the kernel, the merge and the host.
struct Cut {
  int pre;      // 1: every row over the prefix's keys
  int rt;       // rows a tile
  int kt;       // tokens a tile
  int workers;  // workgroups
  int least;    // fewest units a worker takes; 0: every worker takes one whole segment
  int rs;       // rows a partial result holds
  float* o;     // partial results [2 workers][rs][hd], and m, l
  float* ml;
};

struct Tiles {
  int row_tiles, key_tiles;
};
__device__ __forceinline__ Tiles tiles_of(const Cut& u, int group, const Seq& s) {
  if (s.n == 0) return {0, 0};
  const int k = (s.len + u.kt - 1) / u.kt;  // rows that see nothing still have to be written
  return {(int)(((int64_t)s.n * group + u.rt - 1) / u.rt), k < 1 ? 1 : k};
}

__device__ __forceinline__ Seq pass_seq(const CacheArgs& c, const Cut& u, int prefix_len, int b) {
  if (!u.pre) return seq_of(c, b);
  Seq s;
  s.row0 = c.starts != nullptr ? clamp(c.starts[0], 0, c.n_tok) : 0;
  s.n = (c.starts != nullptr ? clamp(c.starts[c.n_seq], s.row0, c.n_tok) : c.n_tok) - s.row0;
  s.len = prefix_len;
  return s;
}

__device__ __forceinline__ int scan_add(int x) {  // inclusive over the lanes
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int k = 1; k < 64; k *= 2) {
    const int y = __shfl_up(x, k);
    if (lane >= k) x += y;
  }
  return x;
}

// The units of one kv head before sequence b (b < 0: not asked for), and of all
// sequences; and the sequence that holds unit `unit`, with the units before it.
struct Place {
  int total, before, seq, base;
};
__device__ __forceinline__ int units_of(const CacheArgs& c, const Cut& u, int prefix_len, int b) {
  const Tiles t = tiles_of(u, c.group, pass_seq(c, u, prefix_len, b));
  return t.row_tiles * t.key_tiles;
}
__device__ __forceinline__ int total_units(const CacheArgs& c, const Cut& u, int prefix_len, int upto) {
  const int lane = threadIdx.x & 63;
  int x = 0;
  for (int b = lane; b < upto; b += 64) x += units_of(c, u, prefix_len, b);
  return __builtin_amdgcn_readlane(scan_add(x), 63);
}
__device__ __forceinline__ void locate(const CacheArgs& c, const Cut& u, int prefix_len, int n_seq, int unit,
                                       int* seq, int* base) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int b0 = 0; b0 < n_seq; b0 += 64) {
    const int mine = b0 + lane < n_seq ? units_of(c, u, prefix_len, b0 + lane) : 0;
    const int incl = scan_add(mine);
    const uint64_t hit = __ballot(before + incl > unit);
    if (hit != 0) {
      const int l = __ffsll((unsigned long long)hit) - 1;
      *seq = b0 + l;
      *base = before + __builtin_amdgcn_readlane(incl - mine, l);
      return;
    }
    before += __builtin_amdgcn_readlane(incl, 63);
  }
  *seq = n_seq - 1;  // not reached: unit < the total
  *base = before;
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

template <class T, int HD, int NT, bool EXACT>
__global__ void __launch_bounds__(kBlock, NT == 1 && HD <= 128 ? 2 : 1)
k_attend(const AttendArgs a, const Cut u, const int direct, float* const row_o, float* const row_ml) {
  using S = typename T::storage;
  constexpr int CE = T::ce;
  constexpr int KT = tokens_of<T>();
  constexpr int MT = KT / 16;
  constexpr int KC = HD / (4 * CE);  // chunks a lane holds of a row
  constexpr int MD = HD / 16;        // output tiles
  constexpr bool kF32 = T::code == SY_F32;
  // A row's start moves by 32 (fp32: 16) bytes from row to row modulo all banks.
  constexpr int LS = HD * (int)sizeof(S) + (kF32 ? 16 : 32);
  constexpr int OS = HD * 4 + 16;  // stride of a row of results in the same space
  static_assert(16 * OS <= KT * LS, "results fit the values' space");
  __shared__ __align__(16) char lds[kWaves][KT * LS];
  __shared__ float stats[kWaves][16][2];
  const CacheArgs& c = a.c;
  const int lane = threadIdx.x & 63;
  const int col = lane & 15, grp = lane >> 4;
  const int wave = wave_id();
  char* const vt = lds[wave];
  const int worker = blockIdx.x;
  const int n_seq = u.pre ? 1 : c.n_seq;
  const int plen = (int)a.prefix_len;
  const int hd = EXACT ? HD : c.hd;
  const float sl = a.scale * 1.44269504088896340736f;

  int h, b, rtile, tile;
  Seq s;
  Tiles ti;
  int64_t unit = 0, end = 0;
  bool some;
  if (u.least == 0) {
    // Equal row tiles for every sequence: no search.
    const int per_seq = (c.each * c.group + u.rt - 1) / u.rt;
    h = worker / (per_seq * n_seq);
    b = worker / per_seq - h * n_seq;
    rtile = worker - (h * n_seq + b) * per_seq;
    tile = 0;
    s = pass_seq(c, u, plen, b);
    ti = tiles_of(u, c.group, s);
    end = ti.key_tiles;
    some = true;
  } else {
    const int per_head = total_units(c, u, plen, n_seq);
    const int64_t units = (int64_t)per_head * c.kv_heads;
    const int64_t share = max((units + u.workers - 1) / u.workers, (int64_t)u.least);
    unit = worker * share;
    end = min(unit + share, units);
    some = unit < end;
    if (some) {
      h = (int)(unit / per_head);
      const int at = (int)(unit - (int64_t)h * per_head);
      int base;
      locate(c, u, plen, n_seq, at, &b, &base);
      s = pass_seq(c, u, plen, b);
      ti = tiles_of(u, c.group, s);
      rtile = (at - base) / ti.key_tiles;
      tile = at - base - rtile * ti.key_tiles;
    }
  }

  if (some) {
    while (true) {
      const int count = (int)min((int64_t)(ti.key_tiles - tile), end - unit);
      const bool begins = tile == 0, whole = begins && count == ti.key_tiles;

      // ---- this segment: kv head h, row tile rtile of sequence b, key tiles [tile, tile + count)
      const int rows = s.n * c.group;
      const int r0 = rtile * 16 * NT;
      const int past = u.pre ? plen : s.len - s.n + 1;  // keys the first token sees
      const int last = min(r0 + 16 * NT, rows) - 1;
      const int least = u.pre ? plen : past + r0 / c.group;
      const int most = u.pre ? plen : past + last / c.group;
      int limit[NT];
      i32x4_t q[NT][KC];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int r = min(r0 + 16 * n + col, last);  // rows past the last repeat it and are not stored
        const int t = r / c.group;
        limit[n] = u.pre ? plen : past + t;
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
      int64_t off[MT];
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
          off[x] = okn[x] ? id[x] * c.page_stride + (j & ((1 << c.page_shift) - 1)) * c.row_stride : 0;
        }
      };
      const auto ask = [&](const S* base_p, i32x4_t (&dst)[MT][KC]) {
#pragma unroll
        for (int x = 0; x < MT; ++x)
#pragma unroll
          for (int k = 0; k < KC; ++k) {
            const int ch = (k * 4 + grp) * CE;
            dst[x][k] = *reinterpret_cast<const i32x4_t*>(base_p + off[x] + (EXACT || ch < hd ? ch : 0));
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
        i32x4_t p16[NT];
        float pf[NT][MT * 4];
        bool any_new = false;
        float scale_o[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float y[MT * 4];
#pragma unroll
          for (int x = 0; x < MT; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) y[x * 4 + e] = st[n][x][e] * sl;
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
          const float mn = fmaxf(m[n], group_max(top));
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
          // The weights are rounded to the values' dtype for the product (at most half a
          // step each, independent of one another; the sum keeps them unrounded).
          if constexpr (!kF32) p16[n] = pack<T>(pf[n]);
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
              for (int n = 0; n < NT; ++n) o[n][d] = Mma<T>::run(w, p16[n], o[n][d]);
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
            x += f * *reinterpret_cast<const f32x4_t*>(lds[w] + row * OS + ch * 4);
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
          s = pass_seq(c, u, plen, b);
        } while (s.n == 0);
        ti = tiles_of(u, c.group, s);
      }
    }
  }
  if (a.fill && !u.pre && c.starts != nullptr) {
    const int lo = clamp(c.starts[0], 0, c.n_tok), hi = clamp(c.starts[c.n_seq], lo, c.n_tok);
    const int64_t width = (int64_t)c.heads * hd;
    S* const out = static_cast<S*>(a.out);
    const int64_t step = (int64_t)gridDim.x * kBlock;
    for (int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x; i < lo * width; i += step) out[i] = S(0);
    for (int64_t i = hi * width + (int64_t)blockIdx.x * kBlock + threadIdx.x; i < c.n_tok * width; i += step)
      out[i] = S(0);
  }
}

// ---------------------------------------------------------------------- merge
//
// Joins the partial results of rows that several workgroups worked on, and those of a
// prefix with a sequence's own: out = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i. A
// workgroup takes some heads of one token; hd / 4 threads read a partial result, so many
// results are read at once, and every thread's sum runs in the order of the keys. Rows
// that one workgroup finished are left alone.
struct Parts {
  int first, count, row;  // workers first .. first + count - 1; row of the tile
};
struct Shares {
  int per_head, base;
  int64_t share;
};

__device__ __forceinline__ Shares shares_of(const CacheArgs& c, const Cut& u, int plen, int b) {
  Shares x;
  x.per_head = total_units(c, u, plen, u.pre ? 1 : c.n_seq);
  x.base = u.pre ? 0 : total_units(c, u, plen, b);
  const int64_t units = (int64_t)x.per_head * c.kv_heads;
  x.share = max((units + u.workers - 1) / u.workers, (int64_t)u.least);
  return x;
}
__device__ __forceinline__ Parts parts_of(const CacheArgs& c, const Cut& u, const Shares& x, const Seq& s, int h, int r) {
  Parts p;
  const int rtile = r / u.rt;
  p.row = r - rtile * u.rt;
  if (u.least == 0) {
    p.first = 0;
    p.count = 1;
    return p;
  }
  const int k = tiles_of(u, c.group, s).key_tiles;
  const int64_t at = (int64_t)h * x.per_head + x.base + (int64_t)rtile * k;
  p.first = (int)(at / x.share);
  p.count = (int)((at + k - 1) / x.share) - p.first + 1;
  return p;
}

constexpr int kMostWorkers = 1024;

template <class T>
__global__ void __launch_bounds__(kBlock)
k_merge(const AttendArgs a, const Cut own, const Cut pre, const int has_pre, const int per_wg, float* const row_o,
        float* const row_ml, float* const pre_o, float* const pre_ml) {
  using S = typename T::storage;
  const CacheArgs& c = a.c;
  __shared__ float weight[2 * kMostWorkers];
  __shared__ f32x4_t fold[kBlock];
  __shared__ float tops[kWaves], sums[kWaves];
  const int tid = threadIdx.x;
  const int slices = (c.heads + per_wg - 1) / per_wg;
  const int tok = blockIdx.x / slices, slice = blockIdx.x - tok * slices;
  const int b = find_seq(c, tok);
  if (b < 0) return;
  const Seq s = seq_of(c, b);
  const Shares xo = own.least == 0 ? Shares{} : shares_of(c, own, 0, b);
  Shares xp{};
  Seq ps{};
  if (has_pre) {
    ps = pass_seq(c, pre, (int)a.prefix_len, 0);
    xp = shares_of(c, pre, (int)a.prefix_len, 0);
  }
  const int lpr = c.hd / 4, groups = kBlock / lpr;
  const int grp = tid / lpr, ch = (tid - grp * lpr) * 4;
  for (int hq = slice * per_wg; hq < min((slice + 1) * per_wg, c.heads); ++hq) {
    const int64_t row = (int64_t)tok * c.heads + hq;
    const int h = hq / c.group, g = hq - h * c.group;
    const Parts mine = parts_of(c, own, xo, s, h, (tok - s.row0) * c.group + g);
    if (!has_pre && mine.count == 1) continue;
    Parts front{};
    if (has_pre) front = parts_of(c, pre, xp, ps, h, (tok - ps.row0) * c.group + g);
    // Partial result i, the prefix's first: worker first + k's second slot where the segment
    // begins (k = 0), its first slot otherwise, or one whole result.
    const auto slot = [&](int i) -> int64_t {
      const bool f = i < front.count;
      const Parts& p = f ? front : mine;
      if (p.count == 1) return row;
      const int k = f ? i : i - front.count;
      return (2 * (int64_t)(p.first + k) + (k == 0 ? 1 : 0)) * (f ? pre.rs : own.rs) + p.row;
    };
    const float* const fo = front.count == 1 ? pre_o : pre.o;
    const float* const fm = front.count == 1 ? pre_ml : pre.ml;
    const float* const mo = mine.count == 1 ? row_o : own.o;
    const float* const mm = mine.count == 1 ? row_ml : own.ml;
    const int n = front.count + mine.count;
    float m = -INFINITY;
    for (int i = tid; i < n; i += kBlock) {
      const float x = (i < front.count ? fm : mm)[slot(i) * 2];
      weight[i] = x;
      m = fmaxf(m, x);
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
      const float l = (i < front.count ? fm : mm)[slot(i) * 2 + 1];
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
    f32x4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
    if (grp < groups) {
#pragma unroll 4
      for (int i = grp; i < n; i += groups)
        o += weight[i] * *reinterpret_cast<const f32x4_t*>((i < front.count ? fo : mo) + slot(i) * c.hd + ch);
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

// ----------------------------------------------------------------------- host

// Tiles a wave at most of a segment that is not cut.
constexpr int kShort = 4;

// Row groups of 16 that a tile takes: one where a sequence brings at most 16 rows (a
// decoded token of up to 16 heads a kv head), else as many as the registers hold.
int row_groups(int64_t rows, int hd, int dtype) {
  if (rows <= 16) return 1;
  return dtype == SY_F32 ? (hd > 128 ? 1 : 2) : (hd > 128 ? 2 : 4);
}

struct Plan {
  Cut own, pre;
  int nt_own, nt_pre;
  int64_t bytes;
  int64_t row_o, row_ml, pre_o, pre_ml;  // float offsets
  bool ok;
};

bool cut(const CacheArgs& c, int dtype, bool pre, int64_t len, int nt, int cus, Cut* u) {
  u->pre = pre;
  u->kt = dtype == SY_F32 ? 16 : 32;
  u->rt = 16 * nt;
  const int64_t rows = (int64_t)c.n_tok * c.group;
  const int64_t keys = std::max<int64_t>(1, (len + u->kt - 1) / u->kt);
  const bool even = !pre && c.starts == nullptr;
  int64_t tiles;  // row tiles, at most
  if (pre) tiles = (rows + u->rt - 1) / u->rt;
  else if (even) tiles = c.n_seq * (((int64_t)c.each * c.group + u->rt - 1) / u->rt);
  else tiles = rows / u->rt + std::min<int64_t>(c.n_seq, rows);
  const int64_t most = 0x7fffffff;
  if (rows * c.kv_heads > most || tiles > most / keys || tiles * keys > most / c.kv_heads) return false;
  u->rs = (int)std::min<int64_t>(u->rt, even ? (int64_t)c.each * c.group : rows);
  // Whole segments where the longest takes a wave few tiles.
  if (even && keys <= kShort * kWaves) {
    u->least = 0;
    u->workers = (int)(tiles * c.kv_heads);
    return true;
  }
  u->least = 2 * kWaves;
  const int64_t units = tiles * keys * c.kv_heads;
  const int64_t full = std::min<int64_t>(kMostWorkers, (int64_t)cus * (nt == 1 && c.hd <= 128 ? 2 : 1));
  u->workers = (int)std::max<int64_t>(1, std::min(full, (units + u->least - 1) / u->least));
  return true;
}

Plan plan_attend(const CacheArgs& c, int64_t prefix_len, int dtype) {
  Plan p{};
  int cus = 0;
  if (cu_count(&cus) != hipSuccess || cus < 1) cus = 1;
  const int64_t rows = (int64_t)c.n_tok * c.group;
  p.nt_own = row_groups((rows + c.n_seq - 1) / c.n_seq, c.hd, dtype);
  p.nt_pre = row_groups(rows, c.hd, dtype);
  p.ok = cut(c, dtype, false, c.cap, p.nt_own, cus, &p.own);
  if (p.ok && prefix_len > 0) p.ok = cut(c, dtype, true, prefix_len, p.nt_pre, cus, &p.pre);
  if (!p.ok) return p;
  int64_t at = 0;
  const auto take = [&](int64_t n) {
    const int64_t was = at;
    at += (n + 3) / 4 * 4;
    return was;
  };
  const auto slots = [&](Cut& u) {
    const int64_t n = 2 * (int64_t)u.workers * u.rs;
    u.o = reinterpret_cast<float*>(take(n * c.hd) * sizeof(float));
    u.ml = reinterpret_cast<float*>(take(n * 2) * sizeof(float));
  };
  if (p.own.least != 0) slots(p.own);
  if (prefix_len > 0) {
    slots(p.pre);
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
hipError_t attend_t(const AttendArgs& a, const Cut& u, int direct, float* row_o, float* row_ml, hipStream_t s) {
  const dim3 grid((unsigned)u.workers);
  if (a.c.hd == HD)
    hipLaunchKernelGGL((k_attend<T, HD, NT, true>), grid, dim3(kBlock), 0, s, a, u, direct, row_o, row_ml);
  else
    hipLaunchKernelGGL((k_attend<T, HD, NT, false>), grid, dim3(kBlock), 0, s, a, u, direct, row_o, row_ml);
  return hipGetLastError();
}

template <class T>
hipError_t attend_pass(const AttendArgs& a, const Cut& u, int direct, float* row_o, float* row_ml, hipStream_t s) {
  constexpr bool f = T::code == SY_F32;
  const bool one = u.rt == 16;
  if (a.c.hd <= 64)
    return one ? attend_t<T, 64, 1>(a, u, direct, row_o, row_ml, s)
               : attend_t<T, 64, f ? 2 : 4>(a, u, direct, row_o, row_ml, s);
  if (a.c.hd <= 128)
    return one ? attend_t<T, 128, 1>(a, u, direct, row_o, row_ml, s)
               : attend_t<T, 128, f ? 2 : 4>(a, u, direct, row_o, row_ml, s);
  return one ? attend_t<T, 256, 1>(a, u, direct, row_o, row_ml, s)
             : attend_t<T, 256, f ? 1 : 2>(a, u, direct, row_o, row_ml, s);
}

template <class T>
hipError_t attend_dt(const AttendArgs& a, hipStream_t s) {
  Plan p = plan_attend(a.c, a.prefix_len, T::code);
  float* const ws = static_cast<float*>(a.workspace);
  const auto at = [&](float* off) { return reinterpret_cast<float*>((char*)ws + reinterpret_cast<uintptr_t>(off)); };
  p.own.o = at(p.own.o);  // (not used where nothing is cut)
  p.own.ml = at(p.own.ml);
  const bool pre = a.prefix_len > 0;
  if (pre) {
    p.pre.o = at(p.pre.o);
    p.pre.ml = at(p.pre.ml);
    const hipError_t e = attend_pass<T>(a, p.pre, 0, ws + p.pre_o, ws + p.pre_ml, s);
    if (e != hipSuccess) return e;
  }
  hipError_t e = attend_pass<T>(a, p.own, pre ? 0 : 1, ws + p.row_o, ws + p.row_ml, s);
  if (e != hipSuccess) return e;
  if (!pre && (p.own.least == 0 || a.c.cap <= p.own.kt)) return hipSuccess;  // nothing was cut
  // Heads a workgroup: one, until there are far more tokens than fit the device at once.
  const int per_wg = (int)std::min<int64_t>(a.c.heads, std::max<int64_t>(1, (int64_t)a.c.n_tok * a.c.heads / 8192));
  const int64_t grid = (int64_t)a.c.n_tok * ((a.c.heads + per_wg - 1) / per_wg);
  hipLaunchKernelGGL((k_merge<T>), dim3((unsigned)grid), dim3(kBlock), 0, s, a, p.own, p.pre, pre ? 1 : 0, per_wg,
                     ws + p.row_o, ws + p.row_ml, ws + p.pre_o, ws + p.pre_ml);
  return hipGetLastError();
}

template <class T, int VE>
hipError_t append_t(const AppendArgs& a, hipStream_t s) {
  const unsigned grid = (unsigned)std::min(a.c.n_tok, 1 << 20);
  hipLaunchKernelGGL((k_append<T, VE>), dim3(grid), dim3(kBlock), 0, s, a);
  return hipGetLastError();
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
