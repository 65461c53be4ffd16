// Attention of new tokens over a paged KV cache on gfx950.
//
//   out[i,h] = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(scale q_i.k_j - m_i)
//
// for the packed rows i of a ragged batch, over the pages of each sequence;
// causal: row t of a chunk of n new tokens sees the first len - n + t + 1 of
// the sequence's len keys. One pass over the keys with the running maximum
// and sum. Statistics, scores and the sum over p v are 32 bits; p is rounded
// to the rows' 16-bit type for the matrix product (half a step of 2^-8 or
// 2^-11 each, independent over the keys), the result once more. The sum of a
// row is taken over the rounded p, so that its weights add up to one. That is a
// choice: p in 32 bits would need a second product of its lower half with V,
// half as much again on the matrix pipe, which bounds prompts. Against 64
// bits the result is off by 2.2e-3 of its norm in bf16 and 2.9e-4 in fp16, of
// which its own rounding is 1.7e-3 and 2.2e-4.
//
// Rows: the G = Hq / Hk query heads that share a kv head are rows of one
// tile, row r = t * G + g, so that a key is fetched once for all of them.
// Both kernels work on S^T = K Q^T and O^T = V^T P^T: a column of the
// result is a query row, so a lane keeps one row's statistics, and what S^T
// leaves in a lane's registers is, with the keys of a step permuted in V
// likewise, what P^T takes: p never leaves the registers.
//
//   few:  tiles of 16 rows, 4 or 8 waves that each take every fourth or
//         eighth tile of 32 keys by themselves and are joined at the end. K
//         goes from memory to registers, V through the wave's own LDS and
//         comes back by transposing reads. An item (a tile of rows and a kv
//         head) is a workgroup's, or all items are shared out evenly. Bound by
//         HBM where there is enough to read: 64 sequences of 700 to 8191 keys,
//         64 / 8 heads, D = 128, 8 bits: 594 MB in 116 us, 5.1 TB/s with the
//         launches (a large copy reads 6.3); one of 131071 at 16 bits: 537 MB
//         in 99 us, 5.4 TB/s. Below that by a launch and one way to memory:
//         8 sequences of 560 keys take 9.2 us, of 128 keys 5.4.
//   many: tiles of 128 rows, 4 waves of 32 rows over shared tiles of 64
//         keys in LDS, two of them in turn. Bound by what the matrix and the
//         vector pipe issue together: a prompt of 8192 tokens, 32 / 8 heads,
//         D = 128: 550 GFLOP in 515 to 535 us, 1030 to 1070 TFLOP/s; the
//         matrix pipe is busy for 54 % and the vector pipe for 43 % of the
//         time, and a large library product reaches 1180.
//
// Where that leaves units idle the keys are split: the few kernel's shares
// end anywhere in an item, the many kernel's in equal parts, and a second
// kernel joins the parts. How many splits work is settled on the device, by
// the sequence's own length.
//
// Keys that a row does not see have p = 0 by selection; V rows past the end
// enter as 0. Where rows of a tile see different keys, a V value that is NaN
// or infinite enters the product as 0 and is added by itself to the rows that
// see it. A page number outside of the pool makes the scores of its keys NaN;
// a length that the table cannot hold makes its rows NaN. Nothing outside of
// the tensors is read.

#include "paged_common.h"

namespace {

using namespace paged;

typedef float f16v __attribute__((ext_vector_type(16)));
typedef short s4 __attribute__((ext_vector_type(4)));

struct Args {
  const void* q;
  const void* k;
  const void* v;
  const uint8_t* k_scale;
  const uint8_t* v_scale;
  const int* q_starts;
  const int* kv_lens;
  const int* table;
  void* out;
  // [part][row][D]: sums over p v; [part][row][2]: maximum, sum of p. Parts:
  // 2 of each worker, or [tile][h][split]
  float* parts;
  float* stats;
  long long q_row, q_head, table_row;
  int cols;  // of the table
  int T, B, Hq, Hk, G, pages, page_log2;
  uint32_t inv_group;  // 2^32 / G, rounded up
  float scale;  // times log2(e): exponentials are of base 2
  int causal, splits;
  int sorted;     // the many kernel's tiles
  int workers;    // of the few kernel, where they share the work
  int unit_log2;  // of their line: 32 << unit_log2 keys
};

// ---- what is where ----------------------------------------------------

struct Span {
  int seq = -1;
  int row0, rows;  // the tile's first row, the sequence's rows
  int t0, g0;      // of row0: its token, and head of the group
  int q0, n, len;  // first packed token, new tokens, keys
  bool broken;     // a length that the table cannot hold
};

// a row of a tile: its token of the sequence, and head of the kv head's group
struct Row {
  int t, g;
};

__device__ inline Row row_at(const Args& a, const Span& s, int i) {
  // i and g0 are small: the product with 2^32 / G, rounded up, is exact
  const int x = s.g0 + i;
  const int q = a.G == 1 ? x : (int)__umulhi((uint32_t)x, a.inv_group);
  return Row{s.t0 + q, x - q * a.G};
}

// how many of the sequence's keys row i of the tile sees
__device__ inline int seen_by(const Args& a, const Span& s, int i) {
  if (s.row0 + i >= s.rows) return 0;
  if (!a.causal) return s.len;
  return min(max(s.len - s.n + row_at(a, s, i).t + 1, 0), s.len);
}
// the last row's, of the first `rows`
__device__ inline int most_seen(const Args& a, const Span& s, int rows) {
  return seen_by(a, s, min(rows, s.rows - s.row0) - 1);
}

// tiles of keys: what a workgroup takes of `all`, and how many splits work
struct Share {
  int first, last, active = 1;
};

// keys of a tile of the many kernel, and the fewest tiles of a split
constexpr int MANY_KEYS = 64, MANY_LEAST = 4;

__device__ inline Share share_of(int all, int splits, int split, int least) {
  int each = max((all + splits - 1) / splits, least);
  Share s;
  s.active = max((all + each - 1) / each, 1);
  s.first = min(split * each, all);
  s.last = min(s.first + each, all);
  return s;
}

// a load by the scalar unit: the address is the wave's, and nothing in the
// kernel writes there. It is not counted with the vector loads in flight.
__device__ inline int uniform_load(const int* p) {
  return *(const __attribute__((address_space(4))) int*)(uintptr_t)p;
}

// ---- small pieces ------------------------------------------------------

__device__ inline float lane_xor16_max(float x) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x),
                                            __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ inline float lane_xor32_max(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x),
                                            __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ inline float lane_xor16_add(float x) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x),
                                            __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ inline float lane_xor32_add(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x),
                                            __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ inline float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ inline float minus_inf() { return __uint_as_float(0xff800000u); }
__device__ inline float plus_inf() { return __uint_as_float(0x7f800000u); }
// a maximum to subtract: nothing has been seen where it is -inf
__device__ inline float base_of(float m) {
  return m == minus_inf() ? 0.0f : m;
}

// The maximum that is subtracted is not looked for at every step: p and its
// sum over a lane's keys are worked out with the one there is, and only where
// a sum comes out at 2^8 or more (or not as a number: at first the maximum is
// -inf) is it found and p worked out again. So p is at most 2^8 instead of 1:
// fp16 and 32 bits hold that and the sums with room to spare, and its rounding
// is relative as before; the maximum itself is always some score's, never too
// high. Of 88 vector instructions for 32 keys this saves 20, and the wait for
// them before the first exponential (2 sequences of 2048 new tokens over 6000
// keys, 32 / 8 heads, D = 128: 400.7 us before, 392 with it).
constexpr float MOST = 256.0f;

__device__ inline f4 mfma16(Bf16::V8 a, Bf16::V8 b, f4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ inline f4 mfma16(Fp16::V8 a, Fp16::V8 b, f4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ inline f16v mfma32(Bf16::V8 a, Bf16::V8 b, f16v c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ inline f16v mfma32(Fp16::V8 a, Fp16::V8 b, f16v c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// sum + the two values of pair j: what is summed is what is multiplied
__device__ inline float add_pair(const Oct<Bf16>& p, int j, float sum) {
  const Bf16::V2 one = {(__bf16)1.0f, (__bf16)1.0f};
  return __builtin_amdgcn_fdot2_f32_bf16(Bf16::V2{p.v[2 * j], p.v[2 * j + 1]},
                                         one, sum, false);
}
__device__ inline float add_pair(const Oct<Fp16>& p, int j, float sum) {
  const Fp16::V2 one = {(_Float16)1.0f, (_Float16)1.0f};
  return __builtin_amdgcn_fdot2(Fp16::V2{p.v[2 * j], p.v[2 * j + 1]}, one,
                                sum, false);
}

// 8 codes times their scale, rounded to 16 bits: exact, but for fp16 where
// the value is not one of fp16's
__device__ inline void widen(Oct<Bf16>& o, u2 codes, float scale) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    auto lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes[j], scale, false);
    auto hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes[j], scale, true);
    o.h[4 * j] = lo[0];
    o.h[4 * j + 1] = lo[1];
    o.h[4 * j + 2] = hi[0];
    o.h[4 * j + 3] = hi[1];
  }
}
__device__ inline void widen(Oct<Fp16>& o, u2 codes, float scale) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    auto lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes[j], scale, false);
    auto hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes[j], scale, true);
    o.h[4 * j] = lo[0];
    o.h[4 * j + 1] = lo[1];
    o.h[4 * j + 2] = hi[0];
    o.h[4 * j + 3] = hi[1];
  }
}

__device__ inline bool strange(const Oct<Bf16>& o) {
  bool s = false;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    s |= (o.raw[j] & 0x7f80u) == 0x7f80u ||
         (o.raw[j] & 0x7f800000u) == 0x7f800000u;
  return s;
}
__device__ inline bool strange(const Oct<Fp16>& o) {
  bool s = false;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    s |= (o.raw[j] & 0x7c00u) == 0x7c00u ||
         (o.raw[j] & 0x7c000000u) == 0x7c000000u;
  return s;
}

// its values, with 0 for those
template <typename K>
__device__ inline u4 finite_only(Oct<K> o) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (!(fabsf((float)o.h[j]) < plus_inf())) o.h[j] = (typename K::T)0.0f;
  return o.raw;
}

// Calls add(d, v) for each value v = at(d) of a key's V row that is NaN or
// infinite, d and v the wave's.
template <int D, typename P, typename F>
__device__ inline void each_strange(P at, F add) {
  const int lane = threadIdx.x & 63;
#pragma unroll 1
  for (int d0 = 0; d0 < D; d0 += 64) {
    const int d = d0 + lane;
    float v = d < D ? at(d) : 0.0f;
    unsigned long long found = __ballot(!(fabsf(v) < plus_inf()));
    while (found) {
      const int i = __ffsll(found) - 1;
      found &= found - 1;
      add(d0 + i, __uint_as_float(__builtin_amdgcn_readlane(
                      __float_as_uint(v), i)));
    }
  }
}

typedef __attribute__((address_space(3))) s4* lds_s4;

// 4 keys by 16 values, transposed: a lane of 16 names 4 values of key
// (lane >> 2), and gets the 4 keys of value (lane & 15)
__device__ inline u2 transposed(const void* p) {
  s4 r = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (lds_s4)(const __attribute__((address_space(3))) void*)p);
  return __builtin_bit_cast(u2, r);
}

__device__ inline void wave_fence() {
  // LDS of one wave: its accesses are done in order, the compiler is told
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// ---- the few rows' work ----------------------------------------------------

// Shared out, the work is one line: for each kv head, each sequence, each of its tiles of
// rows, an item of OWN + (its keys / unit keys) units. Worker w takes the
// units from edge(w) to edge(w + 1): w * per, moved to an item's start or end
// where that is less than near(item) away. So workers end together however
// ragged the batch is, items of less than WHOLE units are never split, and of
// a worker's items at most two are split: one that it starts (its part is in
// place 1), and one that it goes on with (place 0). A unit is 32 keys, or
// more where the line would pass 2^30 units.
//
// WHOLE: a workgroup of 4 waves takes 128 keys in 1.1 us, and the kernel that
// joins two parts takes 4.5 us: a part of less than 512 keys does not pay.
// LEAST: a share holds one of the shortest items at least (8 sequences of 200
// keys in tables for 8192 take 11.3 us; with 8, by which two came to one
// workgroup while others had none, 13.3).
constexpr int OWN = 4, NEAR = 4, LEAST = 5, WHOLE = 32;

__device__ inline int near(int units) {
  return units < WHOLE ? units / 2 + 1 : NEAR;
}

struct Item {
  int seq, tile;  // tile of the sequence's rows
  int first;      // unit of its head's line
  int units;
};

// 64 sequences, one a lane: its tokens and keys (-1: a length that the table
// cannot hold), the units of one of its items, and of all up to its last;
// `before`: of the sequences before these
struct Chunk {
  int base, before, q0, n, len, one, own, upto;
};

struct Line {
  int head, per;  // units of a head's line, of a worker
};

__device__ inline int length_of(const Args& a, int len) {
  return len > ((long long)a.cols << a.page_log2) ? -1 : max(len, -1);
}

__device__ inline Chunk chunk_of(const Args& a, int base, int before,
                                 int BM) {
  const int lane = threadIdx.x & 63, i = base + lane;
  Chunk c{base, before, 0, 0, 0, 0, 0, 0};
  if (i < a.B) {
    c.q0 = min(max(a.q_starts[i], 0), a.T);
    c.n = min(max(a.q_starts[i + 1], 0), a.T) - c.q0;
    c.len = length_of(a, a.kv_lens[i]);
    if (c.n > 0) {
      // at most 2^30 keys: the sum stays below 2^31
      const int log2 = 5 + a.unit_log2;
      c.one = OWN + ((max(c.len, 0) + (1 << log2) - 1) >> log2);
      c.own = (c.n * a.G + BM - 1) / BM * c.one;
    }
  }
  c.upto = c.own;
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) {
    const int y = __shfl_up(c.upto, x, 64);
    if (lane >= x) c.upto += y;
  }
  return c;
}

// the first sequences, and the line of all
__device__ inline Line line_of(const Args& a, Chunk& c, int BM) {
  c = chunk_of(a, 0, 0, BM);
  Line l;
  l.head = __builtin_amdgcn_readlane(c.upto, 63);
  bool falls = c.n < 0;
  for (int base = 64; base < a.B; base += 64) {
    const Chunk x = chunk_of(a, base, 0, BM);
    l.head += __builtin_amdgcn_readlane(x.upto, 63);
    falls |= x.n < 0;
  }
  // starts that fall could make the line longer than the host knows: no work
  if (__ballot(falls)) l.head = 0;
  l.per = max((int)((uint32_t)(l.head * a.Hk + a.workers - 1) /
                    (uint32_t)a.workers), LEAST);
  return l;
}

// the item of unit `at` of a head's line; at < line.head
__device__ inline Item item_at(const Args& a, Chunk& c, int at, int BM) {
  if (at < c.before) c = chunk_of(a, 0, 0, BM);
  while (true) {
    const unsigned long long over = __ballot(c.before + c.upto > at);
    if (over) {
      const int l = __ffsll(over) - 1;
      Item r;
      r.seq = c.base + l;
      r.units = __builtin_amdgcn_readlane(c.one, l);
      const int start = c.before + __builtin_amdgcn_readlane(c.upto, l) -
                        __builtin_amdgcn_readlane(c.own, l);
      r.tile = at == start ? 0 : (at - start) / r.units;
      r.first = start + r.tile * r.units;
      return r;
    }
    if (c.base + 64 >= a.B) return Item{-1, 0, 0, 1};
    c = chunk_of(a, c.base + 64,
                 c.before + __builtin_amdgcn_readlane(c.upto, 63), BM);
  }
}

// where the parts of an item that starts at unit `first` of the whole line
// lie: part 0, and part i + 1 `stride` after part i from the second on
struct Parts {
  long long part0, part1;
  int count, stride;
};

__device__ inline Parts parts_of(const Line& l, int first, int units) {
  Parts p{0, 0, 1, 2};
  if (units < WHOLE) return p;
  // the edges inside of the item
  const int w0 = (int)((uint32_t)(first + NEAR + l.per - 1) / (uint32_t)l.per);
  const int w1 = (int)((uint32_t)(first + units - NEAR) / (uint32_t)l.per);
  p.count = max(w1 - w0 + 2, 1);
  p.part0 = 2LL * (w0 - 1) + 1;
  p.part1 = 2LL * w0;
  return p;
}

// the rows from row0 of sequence `seq`, one of the chunk's
__device__ inline Span span_of(const Args& a, const Chunk& c, int seq,
                               int row0) {
  const int l = seq - c.base;
  Span s;
  s.seq = seq;
  s.q0 = __builtin_amdgcn_readlane(c.q0, l);
  s.n = __builtin_amdgcn_readlane(c.n, l);
  s.rows = s.n * a.G;
  s.row0 = row0;
  s.t0 = row0 ? row0 / a.G : 0;
  s.g0 = row0 - s.t0 * a.G;
  s.len = __builtin_amdgcn_readlane(c.len, l);
  s.broken = s.len < 0;
  s.len = max(s.len, 0);
  return s;
}

// Places for the tiles of BM rows: sequence i's may start at
// floor(starts[i] * G / BM) + i, which leaves each at least its own number and
// needs no sum over the sequences before it; without their first tiles
// (FIRST = 0), and without the i, it is as much. The 64 sequences that have
// `place` among theirs:
template <int BM, int FIRST>
__device__ inline Chunk chunk_at(const Args& a, int place) {
  int base = 0;
  for (int above = (a.B + 63) / 64; above - base > 1;) {
    const int mid = (base + above) / 2;
    const int q0 = min(max(uniform_load(a.q_starts + mid * 64), 0), a.T);
    if (q0 * a.G / BM + FIRST * mid * 64 <= place)
      base = mid;
    else
      above = mid;
  }
  return chunk_of(a, base * 64, 0, BM);
}

// A tile in the many kernel's order. Where the units get more than two
// workgroups each, the tiles of the longest of 64 sequences come first, from
// its last one on: what starts late is short (16 sequences of 52 to 400 new
// tokens on 498 to 4052 keys, 32 / 8 heads, D = 128: as they come 192 us, like
// this 173). Otherwise all start at once, the last one first, and are spared
// the search (12 of 3 to 7 tokens on up to 4000 keys: 37.3 us, with it 38.4).
template <int BM>
__device__ inline Span find(const Args& a, int place) {
  if (!a.sorted) place = a.T * a.G / BM + a.B - 1 - place;
  const Chunk c = chunk_at<BM, 1>(a, place);
  const int lane = threadIdx.x & 63;
  const int tiles = c.n > 0 ? (c.n * a.G + BM - 1) / BM : 0;
  int first = c.q0 * a.G / BM + c.base + lane;
  if (a.sorted) {
    first = __builtin_amdgcn_readfirstlane(first);
    for (int i = 0; i < min(a.B - c.base, 64); ++i) {
      const int len = __builtin_amdgcn_readlane(c.len, i);
      if (len > c.len || (len == c.len && i < lane))
        first += __builtin_amdgcn_readlane(tiles, i);
    }
  }
  const unsigned long long at =
      __ballot(first <= place && place - first < tiles);
  if (at == 0) return Span();
  const int l = __ffsll(at) - 1;
  const int back = place - __builtin_amdgcn_readlane(first, l);
  return span_of(
      a, c, c.base + l,
      (a.sorted ? __builtin_amdgcn_readlane(tiles, l) - 1 - back : back) * BM);
}

// All first tiles, then the others: where no sequence has others, the tiles
// at the end are those without work, and every unit gets as many with.
template <int BM>
__device__ inline Span find_first(const Args& a, int tile) {
  if (tile >= a.B) {
    tile -= a.B;
    const Chunk c = chunk_at<BM, 0>(a, tile);
    const int lane = threadIdx.x & 63;
    const int first = c.q0 * a.G / BM;
    const unsigned long long at =
        __ballot(c.base + lane < a.B && first <= tile);
    if (at == 0) return Span();
    const int l = 63 - __clzll(at);
    const Span s =
        span_of(a, c, c.base + l,
                (tile - __builtin_amdgcn_readlane(first, l) + 1) * BM);
    return s.row0 < s.rows ? s : Span();
  }
  Chunk c{tile, 0, 0, 0, 0, 0, 0, 0};
  c.q0 = min(max(uniform_load(a.q_starts + tile), 0), a.T);
  c.n = min(max(uniform_load(a.q_starts + tile + 1), 0), a.T) - c.q0;
  c.len = length_of(a, uniform_load(a.kv_lens + tile));
  const Span s = span_of(a, c, tile, 0);
  return s.row0 < s.rows ? s : Span();
}

// ---- the splits' parts ------------------------------------------------------

// The sums of a row's parts: D/4 lanes a row (each load is of one run of
// memory: a lane has pairs of the two halves of D); GS groups of them share a
// row's parts, and are joined through LDS.
template <typename K, int D, int GS>
__device__ inline void join_rows(const Args& a, const Span& s, int h,
                                 const Parts& p, int BM, int row0) {
  typedef typename K::T T;
  constexpr int LANES = D / 4, GROUPS = 256 / LANES;
  __shared__ f4 sums[GS > 1 ? GROUPS : 1][LANES];
  __shared__ f2 tops[GROUPS];
  const int group = threadIdx.x / LANES, lane = threadIdx.x % LANES;
  const int row = row0 + group / GS;
  const bool real = row < BM && s.row0 + row < s.rows;

  // parts group % GS, + GS, ...: 4 loads on their way at a time
  f4 x = {0, 0, 0, 0};
  float top = minus_inf(), total = 0.0f;
  if (real)
    for (int i = group % GS; i < p.count; i += 4 * GS) {
      f2 y[4][2], st[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = min(i + j * GS, p.count - 1);
        const long long from =
            (k ? p.part1 + (long long)(k - 1) * p.stride : p.part0) * BM + row;
        const float* at = a.parts + from * D + lane * 2;
        y[j][0] = *reinterpret_cast<const f2*>(at);
        y[j][1] = *reinterpret_cast<const f2*>(at + D / 2);
        st[j] = *reinterpret_cast<const f2*>(a.stats + from * 2);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (i + j * GS >= p.count) continue;
        const float next = fmaxf(top, st[j][0]), base = base_of(next);
        const float old = exp2_of(top - base), now = exp2_of(st[j][0] - base);
        x = x * old + f4{y[j][0][0], y[j][0][1], y[j][1][0], y[j][1][1]} * now;
        total = total * old + st[j][1] * now;
        top = next;
      }
    }
  if constexpr (GS > 1) {
    sums[group][lane] = x;
    if (lane == 0) tops[group] = f2{top, total};
    __syncthreads();
    if (group % GS || !real) return;
    float best = top;
#pragma unroll
    for (int g = 1; g < GS; ++g) best = fmaxf(best, tops[group + g][0]);
    const float base = base_of(best), own = exp2_of(top - base);
    x *= own;
    total *= own;
#pragma unroll
    for (int g = 1; g < GS; ++g) {
      const float now = exp2_of(tops[group + g][0] - base);
      x += sums[group + g][lane] * now;
      total += tops[group + g][1] * now;
    }
  }
  if (!real) return;
  const bool none = seen_by(a, s, row) == 0;
  const float inv = s.broken ? nan_f32() : 1.0f / total;
  const Row at = row_at(a, s, row);
  T* dst = (T*)a.out +
           ((long long)(s.q0 + at.t) * a.Hq + h * a.G + at.g) * D + lane * 2;
#pragma unroll
  for (int j = 0; j < 4; j += 2) {
    const T y[2] = {none && !s.broken ? (T)0.0f : (T)(x[j] * inv),
                    none && !s.broken ? (T)0.0f : (T)(x[j + 1] * inv)};
    __builtin_memcpy(dst + j / 2 * (D / 2), y, sizeof y);
  }
}

// ---- few rows ------------------------------------------------------------

// Where 16-byte piece c of a wave's V row lies: the 32-byte blocks that a
// transposing read takes from 8 neighbouring rows fall on different banks.
template <int D>
__device__ inline int few_piece(int row, int c) {
  if constexpr (D == 128) return c ^ ((row & 7) << 1);
  if constexpr (D == 64) return c ^ (((row >> 1) & 3) << 1);
  return c ^ (((row >> 2) & 1) << 1);
}

template <typename K, int D, int DV, bool Q8, int WAVES>
__device__ inline void
few_part(const Args& a, char* lds, float (*stat)[WAVES][16], const Span& s, int h,
         int dv, const Share& mine, bool whole, long long part) {
  typedef typename K::T T;
  constexpr int BM = 16, BN = 32;
  constexpr int NF = D / 32;              // steps of the product over D
  constexpr int NT = DV / 16;             // tiles of 16 values of O^T
  constexpr int EB = Q8 ? 1 : 2;          // bytes of a cached value
  constexpr int LPR = DV * EB / 16;       // lanes for one V row
  constexpr int VROWS = 64 / LPR;         // V rows of one load
  constexpr int NV = BN / VROWS;          // loads for a tile of V
  constexpr int KB = NF * 8 * EB >= 16 ? 16 : 8;  // bytes of a K load
  constexpr int NK = NF * 8 * EB / KB;    // K loads of a lane for 16 keys
  constexpr int JS = DV + 4;              // a row of what the waves join

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int lane = threadIdx.x & 63;
  // What goes by the lane is worked out for each item anew: kept over the
  // items it would take the registers that the tiles need.
  asm volatile("" : "+v"(lane));
  const int col = lane & 15, grp = lane >> 4;

  const int seen_min = seen_by(a, s, 0), seen_max = most_seen(a, s, BM);

  // Q: a lane holds 8 values of row `col` for each step
  Oct<K> q[NF];
  const int seen = seen_by(a, s, col);
  {
    const bool real = s.row0 + col < s.rows;
    const Row r = row_at(a, s, real ? col : 0);
    const T* src = (const T*)a.q + (s.q0 + r.t) * a.q_row +
                   (long long)(h * a.G + r.g) * a.q_head;
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      const int d0 = KB == 16 && Q8 ? 64 * (f >> 1) + grp * 16 + (f & 1) * 8
                                    : 32 * f + grp * 8;
      q[f].raw = real ? *reinterpret_cast<const u4*>(src + d0)
                      : u4{0, 0, 0, 0};
      // scores grow with the product below: a negative scale turns q
      if (a.scale < 0.0f) q[f].raw ^= u4{0x80008000u, 0x80008000u,
                                         0x80008000u, 0x80008000u};
    }
  }
  const float scale = fabsf(a.scale);

  const int* pages = a.table + s.seq * a.table_row;
  const uint8_t* kc = (const uint8_t*)a.k;
  const uint8_t* vc = (const uint8_t*)a.v;
  const int in_page = (1 << a.page_log2) - 1;

  // the page of 16 keys; those past the last are not looked up
  auto page_of = [&](int key) {
    return key < seen_max ? uniform_load(pages + (key >> a.page_log2)) : 0;
  };

  struct Arrival {
    u4 kr[2][NK], vr[NV];
    uint32_t ksr[2], vsr[NV];
    bool bad0, bad1;  // halves without a page
  };
  int id[2];  // pages of the tile to come
  const uint32_t k_off = col * (D * EB) + grp * KB;
  const uint32_t v_off = lane / LPR * (D * EB) + lane % LPR * 16 + dv * EB;

  auto row_of = [&](int id, int key) {
    const bool bad = (unsigned)id >= (unsigned)a.pages;
    return (((long long)(bad ? 0 : id) * a.Hk + h) << a.page_log2) +
           (key & in_page);
  };
  auto fetch_k = [&](Arrival& to, int kt) {
    to.bad0 = (unsigned)id[0] >= (unsigned)a.pages;
    to.bad1 = (unsigned)id[1] >= (unsigned)a.pages;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const long long row = row_of(id[half], kt * BN + half * 16);
      const uint8_t* src = kc + row * (D * EB);
      if constexpr (Q8) to.ksr[half] = (a.k_scale + row)[col];
#pragma unroll
      for (int i = 0; i < NK; ++i) {
        if constexpr (KB == 16) {
          to.kr[half][i] = *reinterpret_cast<const u4*>(src + k_off + i * 64);
        } else {
          u2 x = *reinterpret_cast<const u2*>(src + k_off);
          to.kr[half][i] = u4{x[0], x[1], 0, 0};
        }
      }
    }
  };
  auto fetch_v = [&](Arrival& to, int kt) {
    const long long row0 = row_of(id[0], kt * BN);
    const long long row1 = row_of(id[1], kt * BN + 16);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if constexpr (VROWS <= 16) {
        constexpr int PER16 = 16 / (VROWS > 16 ? 16 : VROWS);
        const long long row =
            (i / PER16 ? row1 : row0) + (i % PER16) * VROWS;
        if constexpr (Q8) to.vsr[i] = (a.v_scale + row)[lane / LPR];
        to.vr[i] = *reinterpret_cast<const u4*>(vc + row * (D * EB) + v_off);
      } else {  // one load takes both halves
        const int vrow = lane / LPR;
        const long long row = (vrow < 16 ? row0 : row1) + (vrow & 15);
        if constexpr (Q8) to.vsr[i] = a.v_scale[row];
        to.vr[i] = *reinterpret_cast<const u4*>(
            vc + row * (D * EB) + lane % LPR * 16 + dv * EB);
      }
    }
  };

  f4 o[NT];
  float m = seen ? minus_inf() : 0.0f, sum = 0.0f;
#pragma unroll
  for (int t = 0; t < NT; ++t) o[t] = f4{0, 0, 0, 0};

  char* mine_v = lds + wave * (BN * DV * 2);
  uint32_t v_at[NT];  // a lane's 4 keys by 4 values of transposing reads
  {
    const int row = grp * 4 + (col >> 2);
#pragma unroll
    for (int t = 0; t < NT; ++t)
      v_at[t] = row * (DV * 2) +
                few_piece<DV>(row, t * 2 + ((col >> 1) & 1)) * 16 +
                (col & 1) * 8;
  }
  // 8-bit tiles: two on their way in turn, since widening one takes long
  constexpr int AHEAD = Q8 ? 1 : 0;
  Arrival arrivals[1 + AHEAD];
  int kt = mine.first + wave;
  if (kt < mine.last) {
    id[0] = page_of(kt * BN);
    id[1] = page_of(kt * BN + 16);
    fetch_k(arrivals[0], kt);
    fetch_v(arrivals[0], kt);
    id[0] = page_of((kt + WAVES) * BN);
    id[1] = page_of((kt + WAVES) * BN + 16);
  }
  auto next_k = [&](Arrival& to) {
    if (kt + WAVES < mine.last) fetch_k(to, kt + WAVES);
  };
  auto next_v = [&](Arrival& to) {
    if (kt + WAVES < mine.last) {
      fetch_v(to, kt + WAVES);
      id[0] = page_of((kt + 2 * WAVES) * BN);
      id[1] = page_of((kt + 2 * WAVES) * BN + 16);
    }
  };
  // The next tile's loads start as soon as there are registers for them.
  auto take = [&](Arrival& now, Arrival& next) {
    if constexpr (AHEAD) {
      next_k(next);
      next_v(next);
    }
    const int key0 = kt * BN;
    const bool none0 = now.bad0, none1 = now.bad1;

    // S^T: 2 tiles of 16 keys
    f4 sc[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      sc[half] = f4{0, 0, 0, 0};
      float scale = 1.0f;
      if constexpr (Q8) scale = scale_of(now.ksr[half]);
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        Oct<K> x;
        if constexpr (Q8) {
          const u4 w = now.kr[half][KB == 16 ? f >> 1 : f];
          widen(x, (KB == 16 && (f & 1)) ? u2{w[2], w[3]} : u2{w[0], w[1]},
                scale);
        } else {
          x.raw = now.kr[half][f];
        }
        sc[half] = mfma16(x.v, q[f].v, sc[half]);
      }
    }

    if constexpr (!AHEAD) next_k(next);

    // V to the wave's LDS; rows past the end, or without a page, as 0
    const bool past = key0 + BN > seen_max || none0 || none1;
    const bool cut = key0 + BN > seen_min || none0 || none1;
    const bool look = cut && seen_min < seen_max;
    bool odd_v = false;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int vrow = i * VROWS + lane / LPR;
      if (past) {
        if (key0 + vrow >= seen_max || (vrow < 16 ? none0 : none1)) {
          now.vr[i] = u4{0, 0, 0, 0};
          now.vsr[i] = 127;
        }
      }
      if constexpr (Q8) {
        const float scale = scale_of(now.vsr[i]);
        Oct<K> x, y;
        widen(x, u2{now.vr[i][0], now.vr[i][1]}, scale);
        widen(y, u2{now.vr[i][2], now.vr[i][3]}, scale);
        if (look) odd_v |= strange(x) || strange(y);
        const int c = (lane % LPR) * 2;
        char* row = mine_v + vrow * (DV * 2);
        *reinterpret_cast<u4*>(row + few_piece<DV>(vrow, c) * 16) = x.raw;
        *reinterpret_cast<u4*>(row + few_piece<DV>(vrow, c + 1) * 16) = y.raw;
      } else {
        Oct<K> x;
        x.raw = now.vr[i];
        if (look) odd_v |= strange(x);
        *reinterpret_cast<u4*>(mine_v + vrow * (DV * 2) +
                               few_piece<DV>(vrow, lane % LPR) * 16) = x.raw;
      }
    }
    wave_fence();

    if constexpr (!AHEAD) next_v(next);

    Oct<K> p;
    if (cut) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int key = key0 + (j >> 2) * 16 + grp * 4 + (j & 3);
        if ((j >> 2) ? none1 : none0) sc[j >> 2][j & 3] = nan_f32();
        if (key >= seen) sc[j >> 2][j & 3] = minus_inf();
      }
    }
    auto weigh = [&](float base) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        p.h[j] = (T)exp2_of(__builtin_fmaf(sc[j >> 2][j & 3], scale, -base));
      float part = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) part = add_pair(p, j, part);
      return part;
    };
    float part = weigh(m);
    if (__ballot(!(part < MOST))) {
      float top = sc[0][0];
#pragma unroll
      for (int j = 1; j < 8; ++j) top = fmaxf(top, sc[j >> 2][j & 3]);
      const float higher =
          fmaxf(m, lane_xor32_max(lane_xor16_max(top)) * scale);
      const float keep = exp2_of(m - base_of(higher));
      m = higher;
      sum *= keep;
#pragma unroll
      for (int t = 0; t < NT; ++t) o[t] *= keep;
      part = weigh(base_of(m));
    }
    sum += part;

    if (look && __ballot(odd_v)) {
      // what is not finite goes to the rows that see it, then gives way
#pragma unroll 1
      for (int key = 0; key < BN; ++key)
        each_strange<DV>(
            [&](int d) {
              return (float)*(const T*)(mine_v + key * (DV * 2) +
                                        few_piece<DV>(key, d >> 3) * 16 +
                                        (d & 7) * 2);
            },
            [&](int d, float v) {
#pragma unroll
              for (int i = 0; i < NT * 4; ++i)
                if (d == (i >> 2) * 16 + grp * 4 + (i & 3) &&
                    key0 + key < seen)
                  o[i >> 2][i & 3] += v;
            });
      wave_fence();
#pragma unroll 1
      for (int i = lane; i < BN * DV / 8; i += 64) {
        Oct<K>* x = reinterpret_cast<Oct<K>*>(mine_v + i * 16);
        x->raw = finite_only<K>(*x);
      }
      wave_fence();
    }

    // O^T += V^T P^T: step j of a lane's 8 keys is 4 grp + j of the first
    // 16, then of the last 16
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const u2 lo = transposed(mine_v + v_at[t]);
      const u2 up = transposed(mine_v + v_at[t] + 16 * (DV * 2));
      Oct<K> x;
      x.raw = u4{lo[0], lo[1], up[0], up[1]};
      o[t] = mfma16(x.v, p.v, o[t]);
    }
    wave_fence();
  };
  while (kt < mine.last) {
    take(arrivals[0], arrivals[AHEAD]);
    kt += WAVES;
    if constexpr (AHEAD) {
      if (kt >= mine.last) break;
      take(arrivals[1], arrivals[0]);
      kt += WAVES;
    }
  }

  // join the waves
  float(*all)[16][JS] = reinterpret_cast<float(*)[16][JS]>(lds);
  __syncthreads();
  const float l = lane_xor32_add(lane_xor16_add(sum));
  if (grp == 0) {
    stat[0][wave][col] = m;
    stat[1][wave][col] = l;
  }
#pragma unroll
  for (int t = 0; t < NT; ++t)
    *reinterpret_cast<f4*>(&all[wave][col][t * 16 + grp * 4]) = o[t];
  __syncthreads();
  constexpr int LANES = WAVES * 4;  // for a row
  const int row = threadIdx.x / LANES;
  if (s.row0 + row >= s.rows) return;
  float top = minus_inf();
#pragma unroll
  for (int w = 0; w < WAVES; ++w) top = fmaxf(top, stat[0][w][row]);
  const float base = base_of(top);
  float keep[WAVES], total = 0.0f;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    keep[w] = exp2_of(stat[0][w][row] - base);
    total += stat[1][w][row] * keep[w];
  }
  // pairs of values: stores of one run of memory
  const int d0 = threadIdx.x % LANES * 2;
  const Row r = row_at(a, s, row);
  const bool none = seen_by(a, s, row) == 0;
  const float inv = s.broken ? nan_f32() : none ? 0.0f : 1.0f / total;
  T* dst =
      (T*)a.out + ((long long)(s.q0 + r.t) * a.Hq + h * a.G + r.g) * D + dv;
  const long long at = part * BM + row;
#pragma unroll
  for (int d = d0; d < DV; d += 2 * LANES) {
    float x = 0.0f, y = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const f2 v = *reinterpret_cast<const f2*>(&all[w][row][d]);
      x += v[0] * keep[w];
      y += v[1] * keep[w];
    }
    if (whole) {
      const T z[2] = {none && !s.broken ? (T)0.0f : (T)(x * inv),
                      none && !s.broken ? (T)0.0f : (T)(y * inv)};
      __builtin_memcpy(dst + d, z, sizeof z);
    } else {
      *reinterpret_cast<f2*>(a.parts + at * D + d) = f2{x, y};
    }
  }
  if (!whole && d0 == 0)
    *reinterpret_cast<f2*>(a.stats + at * 2) = f2{top, total};
}

template <typename K, int D, int DV, bool Q8, int WAVES, bool SHARED>
__global__ void __launch_bounds__(WAVES * 64, 2) few_kernel(Args a) {
  constexpr int BM = 16, BN = 32;
  constexpr int JOIN = WAVES * 16 * (DV + 4) * 4, TILES = WAVES * BN * DV * 2;
  // V tiles while the keys pass, then the waves' sums
  __shared__ __attribute__((aligned(16))) char
      lds[JOIN > TILES ? JOIN : TILES];
  __shared__ float stat[2][WAVES][16];

  if constexpr (!SHARED) {
    // an item a workgroup, or D / DV of them, on one XCD, for its values
    const int item = blockIdx.x / (8 * D / DV) * 8 + blockIdx.x % 8;
    const Span s = find_first<BM>(a, item / a.Hk);
    if (s.seq < 0) return;
    Share mine;
    mine.first = 0;
    mine.last = (most_seen(a, s, BM) + BN - 1) / BN;
    few_part<K, D, DV, Q8, WAVES>(a, lds, stat, s, item % a.Hk,
                                  blockIdx.x / 8 % (D / DV) * DV, mine, true,
                                  0);
    return;
  }
  Chunk c;
  const Line line = line_of(a, c, BM);
  if (line.head == 0) return;
  // neighbouring shares go to one XCD: they read the same sequence
  const int w = a.workers % 8 ? blockIdx.x
                              : blockIdx.x % 8 * (a.workers / 8) +
                                    blockIdx.x / 8;
  const int total = line.head * a.Hk;
  int end = w * line.per;
  if (end >= total) return;
  int h = (int)((uint32_t)end / (uint32_t)line.head);
  Item it = item_at(a, c, end - h * line.head, BM);
  if (it.seq < 0) return;
  int from = end - h * line.head - it.first;
  end += line.per;
  bool next = false;
  if (from < near(it.units))
    from = 0;
  else if (it.units - from < near(it.units))
    next = true;
  while (true) {
    if (next) {
      int at = it.first + it.units;
      if (at == line.head) {
        at = 0;
        if (++h == a.Hk) return;
      }
      it = item_at(a, c, at, BM);
      if (it.seq < 0) return;
      from = 0;
    }
    // the next worker's edge, if it is in this item
    int to = it.units;
    if (end < total) {
      const int e = end - h * line.head - it.first;
      if (e < it.units) {
        if (e < near(it.units)) return;
        if (it.units - e >= near(it.units)) to = e;
      }
    }
    const Span s = span_of(a, c, it.seq, it.tile * BM);
    // an item's last units may hold no key that its rows see
    const int all = (most_seen(a, s, BM) + BN - 1) / BN;
    Share mine;
    mine.first = min(max(from - OWN, 0) << a.unit_log2, all);
    mine.last = min(max(to - OWN, 0) << a.unit_log2, all);
    few_part<K, D, D, Q8, WAVES>(a, lds, stat, s, h, 0, mine,
                       from == 0 && to == it.units,
                       2LL * w + (from == 0 ? 1 : 0));
    if (to < it.units) return;
    next = true;
    __syncthreads();
  }
}

// ---- many rows -----------------------------------------------------------

// 16-byte pieces of K rows: 16 neighbouring rows' same piece on different
// banks; of V rows: 4 neighbouring rows' same 64 bytes
template <int D>
__device__ inline int k_piece(int row, int c) {
  return c ^ ((row / (128 / D)) & (D / 8 - 1));
}
template <int D>
__device__ inline int v_piece_at(int row, int c) {
  if constexpr (D == 128) return c ^ ((row & 3) << 2);
  if constexpr (D == 64) return c ^ (((row >> 1) & 1) << 2);
  return c;
}

// 16 bytes a lane from memory to LDS, at `to` + 16 * lane, without a register
// between; `base` and `to` are the wave's, `off` the lane's. Nothing but
// landed() waits for it.
__device__ inline void to_lds(const void* base, uint32_t off, uint32_t to) {
  asm volatile(
      "s_mov_b32 m0, %2\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %0, %1"
      :
      : "v"(off), "s"(base), "s"(to)
      : "memory");
}
template <int LATER>  // loads that were issued later
__device__ inline void landed() {
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(LATER) : "memory");
}
__device__ inline uint32_t lds_address(const void* p) {
  return (uint32_t)(size_t)(const __attribute__((address_space(3))) char*)p;
}

template <typename K, int D, bool Q8>
__global__ void __launch_bounds__(256, 2) many_kernel(Args a) {
  typedef typename K::T T;
  constexpr int BM = 128, BN = MANY_KEYS;
  constexpr int NF = D / 16;            // steps of the product over D
  constexpr int NT = D / 32;            // tiles of 32 values of O^T
  constexpr int EB = Q8 ? 1 : 2;
  constexpr int LPR = D * EB / 16;      // lanes for one row
  constexpr int ROWS = 64 / LPR;        // rows of one load of a wave
  constexpr int NL = ROWS >= 16 ? 1 : 16 / ROWS;  // loads for its 16 rows
  constexpr int TILE = BN * D * 2;      // bytes of a tile in LDS

  // One object, so that the tiles come first: loads to LDS name their place
  // in 16 bits.
  static_assert(4 * TILE <= 65536, "tiles past what a load to LDS can name");
  __shared__ struct {
    __attribute__((aligned(1024))) char tiles[4 * TILE];  // K of two, V of two
    int odd_v;  // whether a V value was not finite where it matters
  } shared;
  char* const lds = shared.tiles;
  int& odd_v = shared.odd_v;

  // Sorted, a tile's splits come one after the other: the longest tiles' before
  // the next, and the places without a tile at the end. Otherwise all first
  // splits, then the second ones. (15 sequences of 13 new tokens, 64 / 8 heads,
  // D = 64: sorted with the splits outermost 34.6 us, so 30.4; 183 tokens of
  // one sequence, not sorted: 15.0, with the splits innermost 16.5.)
  const int h = blockIdx.x % a.Hk;
  int place = blockIdx.x / a.Hk, split = 0;
  if (a.splits > 1) {
    const int per = a.sorted ? a.splits : a.T * a.G / BM + a.B;
    const int major = place / per, minor = place % per;
    split = a.sorted ? minor : major;
    place = a.sorted ? major : minor;
  }
  const Span s = find<BM>(a, place);
  if (s.seq < 0) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int col = lane & 31, hi = lane >> 5;

  const int seen_min = seen_by(a, s, 0), seen_max = most_seen(a, s, BM);
  const Share mine = share_of((seen_max + BN - 1) / BN, a.splits, split,
                              MANY_LEAST);
  if (split >= mine.active) return;
  if (threadIdx.x == 0) odd_v = 0;
  __syncthreads();

  // this wave's rows
  const int w0 = wave * 32;
  const bool real = s.row0 + w0 + col < s.rows;
  const Row my = row_at(a, s, real ? w0 + col : 0);
  const int seen = seen_by(a, s, w0 + col);
  const bool full = s.row0 + w0 + 31 < s.rows;
  const int wave_min = full ? seen_by(a, s, w0) : 0;  // past the end: none
  const int wave_max = s.row0 + w0 < s.rows ? most_seen(a, s, w0 + 32) : 0;
  Oct<K> q[NF];
  {
    const T* src = (const T*)a.q + (s.q0 + my.t) * a.q_row +
                   (long long)(h * a.G + my.g) * a.q_head;
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      q[f].raw = real ? *reinterpret_cast<const u4*>(src + f * 16 + hi * 8)
                      : u4{0, 0, 0, 0};
      // scores grow with the product below: a negative scale turns q
      if (a.scale < 0.0f) q[f].raw ^= u4{0x80008000u, 0x80008000u,
                                         0x80008000u, 0x80008000u};
    }
  }
  const float scale = fabsf(a.scale);

  // Wave w brings keys 16 w .. 16 w + 15 of a tile: they lie in one page.
  const int* pages = a.table + s.seq * a.table_row;
  const int in_page = (1 << a.page_log2) - 1;
  const int lrow = lane / LPR, lpos = lane % LPR;
  auto page_of = [&](int kt) {
    const int key = kt * BN + wave * 16;
    return kt < mine.last && key < seen_max
               ? uniform_load(pages + (key >> a.page_log2)) : 0;
  };
  auto row_of = [&](int id, int kt) {
    const bool bad = (unsigned)id >= (unsigned)a.pages;
    const int key = kt * BN + wave * 16;
    return (((long long)(bad ? 0 : id) * a.Hk + h) << a.page_log2) +
           (key & in_page);
  };
  uint32_t k_off[NL], v_off[NL];  // 16 bits: what a lane brings of 16 rows
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int row = i * ROWS + lrow;
    k_off[i] = row * (D * 2) + k_piece<D>(wave * 16 + row, lpos) * 16;
    v_off[i] = row * (D * 2) + v_piece_at<D>(wave * 16 + row, lpos) * 16;
  }
  u4 kr[NL], vr[NL];  // 8 bits: codes on their way
  uint32_t ksr[NL], vsr[NL];
  const bool loads = lrow < 16;
  const uint32_t lds0 = lds_address(lds) + wave * (TILE / 4);
  // tile kt's K at (kt & 1) * TILE, its V behind both K's; this wave's rows
  auto k_tile = [&](int kt) { return lds + (kt & 1) * TILE; };
  auto v_tile = [&](int kt) { return lds + (2 + (kt & 1)) * TILE; };

  auto fetch_k = [&](int id, int kt) {
    const long long row = row_of(id, kt);
    const char* src = (const char*)a.k + row * (D * EB);
    if constexpr (Q8) {
      if (loads)
#pragma unroll
        for (int i = 0; i < NL; ++i) {
          const int at = i * ROWS + lrow;
          kr[i] = *reinterpret_cast<const u4*>(src + at * D + lpos * 16);
          ksr[i] = a.k_scale[row + at];
        }
    } else {
#pragma unroll
      for (int i = 0; i < NL; ++i)
        to_lds(src, k_off[i], lds0 + (kt & 1) * TILE + i * 1024);
    }
  };
  auto fetch_v = [&](int id, int kt) {
    const long long row = row_of(id, kt);
    const char* src = (const char*)a.v + row * (D * EB);
    if constexpr (Q8) {
      if (loads)
#pragma unroll
        for (int i = 0; i < NL; ++i) {
          const int at = i * ROWS + lrow;
          vr[i] = *reinterpret_cast<const u4*>(src + at * D + lpos * 16);
          vsr[i] = a.v_scale[row + at];
        }
    } else {
#pragma unroll
      for (int i = 0; i < NL; ++i)
        to_lds(src, v_off[i], lds0 + (2 + (kt & 1)) * TILE + i * 1024);
    }
  };
  // What was fetched becomes the tile, but for the barrier. `more`: NL loads
  // to LDS that were issued later may still be on their way. A key without
  // a page scores NaN: its K row is NaN, its V row 0. V rows past the end
  // are 0, and where rows of the tile see different keys, values that are
  // not finite are 0 too: they are seen to behind the loop.
  auto put_k = [&](int id, int kt, bool more) {
    const bool bad = (unsigned)id >= (unsigned)a.pages;
    char* to = k_tile(kt) + wave * (TILE / 4);
    if constexpr (Q8) {
      if (!loads) return;
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int row = i * ROWS + lrow, c = lpos * 2, at = wave * 16 + row;
        if (bad) kr[i] = u4{0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu,
                            0x7f7f7f7fu};
        Oct<K> x, y;
        const float sc = scale_of(ksr[i]);
        widen(x, u2{kr[i][0], kr[i][1]}, sc);
        widen(y, u2{kr[i][2], kr[i][3]}, sc);
        char* r = to + row * (D * 2);
        *reinterpret_cast<u4*>(r + k_piece<D>(at, c) * 16) = x.raw;
        *reinterpret_cast<u4*>(r + k_piece<D>(at, c + 1) * 16) = y.raw;
      }
    } else {
      if (more) landed<NL>(); else landed<0>();
      if (!bad) return;
#pragma unroll
      for (int i = 0; i < NL; ++i)
        *reinterpret_cast<u4*>(to + i * 1024 + lane * 16) =
            u4{0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu};
    }
  };
  auto put_v = [&](int id, int kt, bool more) {
    const bool bad = (unsigned)id >= (unsigned)a.pages;
    char* to = v_tile(kt) + wave * (TILE / 4);
    const int key0 = kt * BN + wave * 16;
    const bool past = key0 + 16 > seen_max;
    const bool cut = (kt + 1) * BN > seen_min;
    bool odd = false;
    if constexpr (Q8) {
      if (!loads) return;
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int row = i * ROWS + lrow, c = lpos * 2, at = wave * 16 + row;
        Oct<K> x, y;
        const float sc = scale_of(vsr[i]);
        widen(x, u2{vr[i][0], vr[i][1]}, sc);
        widen(y, u2{vr[i][2], vr[i][3]}, sc);
        if (bad || (past && key0 + row >= seen_max))
          x.raw = y.raw = u4{0, 0, 0, 0};
        if (cut && (strange(x) || strange(y))) {
          odd = true;
          x.raw = finite_only<K>(x);
          y.raw = finite_only<K>(y);
        }
        char* r = to + row * (D * 2);
        *reinterpret_cast<u4*>(r + v_piece_at<D>(at, c) * 16) = x.raw;
        *reinterpret_cast<u4*>(r + v_piece_at<D>(at, c + 1) * 16) = y.raw;
      }
    } else {
      if (more) landed<NL>(); else landed<0>();
      if (!bad && !cut) return;
#pragma unroll 1
      for (int i = 0; i < NL; ++i) {
        Oct<K>* x = reinterpret_cast<Oct<K>*>(to + i * 1024 + lane * 16);
        if (bad || (past && key0 + i * ROWS + lrow >= seen_max)) {
          x->raw = u4{0, 0, 0, 0};
        } else if (strange(*x)) {
          odd = true;
          x->raw = finite_only<K>(*x);
        }
      }
    }
    if (odd) odd_v = 1;
  };

  f16v o[NT];
  float m = seen ? minus_inf() : 0.0f, sum = 0.0f;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int j = 0; j < 16; ++j) o[t][j] = 0.0f;

  // a lane's places in a tile: of K the row `col`, of V the 4 keys by 4
  // values of its transposing reads. They change over to the other tile by a
  // bit of theirs, once a tile: worked out for every 32 keys they took a tenth
  // of the vector instructions (2 sequences of 2048 new tokens over 6000 keys,
  // 32 / 8 heads, D = 128: 400.9 us, so 393).
  uint32_t k_at[NF], v_at[NT];
  const int first = (mine.first & 1) * TILE;
#pragma unroll
  for (int f = 0; f < NF; ++f)
    k_at[f] = first + col * (D * 2) + k_piece<D>(col, f * 2 + hi) * 16;
  {
    const int row = hi * 4 + ((lane & 15) >> 2);
    const int c = ((lane >> 4) & 1) * 2 + ((lane >> 1) & 1);
#pragma unroll
    for (int t = 0; t < NT; ++t)
      v_at[t] = 2 * TILE + first + row * (D * 2) +
                v_piece_at<D>(row, t * 4 + c) * 16 + (lane & 1) * 8;
  }

  auto other_k = [&] {
#pragma unroll
    for (int f = 0; f < NF; ++f) k_at[f] ^= TILE;
  };
  auto other_v = [&] {
#pragma unroll
    for (int t = 0; t < NT; ++t) v_at[t] ^= TILE;
  };

  // S^T of the 32 keys from row `row` of the tile
  auto scores = [&](int row, f16v& sc) {
#pragma unroll
    for (int j = 0; j < 16; ++j) sc[j] = 0.0f;
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      Oct<K> x;
      x.raw = *reinterpret_cast<const u4*>(lds + k_at[f] + row * (D * 2));
      sc = mfma32(x.v, q[f].v, sc);
    }
  };
  // The 32 keys from key0 join the sums, while the scores of the next 32 are
  // worked out: what one needs of the vector pipe, the other does not. (Those
  // of no keys at the end, from what lies there, are not used.)
  auto step = [&](int key0, f16v& sc, int row, int next_row, f16v& next) {
    if (key0 + 32 > wave_min) {
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int key = key0 + (j & 3) + 8 * (j >> 2) + 4 * hi;
        if (key >= seen) sc[j] = minus_inf();
      }
    }
    scores(next_row, next);
    Oct<K> p[2];
    auto weigh = [&](float base) {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        p[j >> 3].h[j & 7] =
            (T)exp2_of(__builtin_fmaf(sc[j], scale, -base));
      float part = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) part = add_pair(p[j >> 2], j & 3, part);
      return part;
    };
    float part = weigh(m);
    if (__ballot(!(part < MOST))) {
      float top = sc[0];
#pragma unroll
      for (int j = 1; j < 16; ++j) top = fmaxf(top, sc[j]);
      const float higher = fmaxf(m, lane_xor32_max(top) * scale);
      const float keep = exp2_of(m - base_of(higher));
      m = higher;
      sum *= keep;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < 16; ++j) o[t][j] *= keep;
      part = weigh(base_of(m));
    }
    sum += part;
    // While this wave feeds the matrix pipe with nothing else to do, the
    // unit's other wave waits with its own products, and takes the vector
    // pipe (8192 tokens: 515 us against 530).
    __builtin_amdgcn_s_setprio(1);
    // a lane's 8 keys of a step of 16: 4 hi + 0..3, then 8 + 4 hi + 0..3
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const char* at = lds + v_at[t] + (row + half * 16) * (D * 2);
        const u2 lo = transposed(at), up = transposed(at + 8 * (D * 2));
        Oct<K> x;
        x.raw = u4{lo[0], lo[1], up[0], up[1]};
        o[t] = mfma32(x.v, p[half].v, o[t]);
      }
    __builtin_amdgcn_s_setprio(0);
  };
  // K runs one tile ahead of its use, V half a tile less: each load to LDS
  // has the time of a tile. Two barriers a tile: behind the first, K(kt + 1)
  // is there and K(kt) is free; behind the second, V(kt + 1), and V(kt).
  f16v s0, s1;
  int kt = mine.first;
  int id1 = page_of(kt), id2 = page_of(kt + 1);  // of the next V, the next K
  if (kt < mine.last) {
    fetch_k(id1, kt);
    fetch_v(id1, kt);
    put_k(id1, kt, true);
    put_v(id1, kt, false);
    if (kt + 1 < mine.last) fetch_k(id2, kt + 1);
  }
  __syncthreads();
  if (kt < mine.last && kt * BN < wave_max) scores(0, s0);
  for (; kt < mine.last; ++kt) {
    const bool more = kt + 1 < mine.last, more2 = kt + 2 < mine.last;
    const int key0 = kt * BN;
    id1 = id2;
    id2 = page_of(kt + 2);
    if constexpr (Q8) {
      if (more) put_k(id1, kt + 1, false);
    }
    if (more) fetch_v(id1, kt + 1);
    if (key0 < wave_max)
      step(key0, s0, 0, 32, s1);
    other_k();
    if constexpr (!Q8) {
      if (more) put_k(id1, kt + 1, true);
    }
    __syncthreads();
    if constexpr (Q8) {
      if (more) put_v(id1, kt + 1, false);
    }
    if (more2) fetch_k(id2, kt + 2);
    if (key0 + 32 < wave_max)
      step(key0 + 32, s1, 32, 0, s0);
    other_v();
    if constexpr (!Q8) {
      if (more) put_v(id1, kt + 1, more2);
    }
    __syncthreads();
  }

  if (odd_v) {
    // What is not finite, from memory again, to the rows that see it.
#pragma unroll 1
    for (int key = max(seen_min / BN, mine.first) * BN;
         key < min(mine.last * BN, seen_max); ++key) {
      const int id = uniform_load(pages + (key >> a.page_log2));
      if ((unsigned)id >= (unsigned)a.pages) continue;
      const long long row =
          (((long long)id * a.Hk + h) << a.page_log2) + (key & in_page);
      each_strange<D>(
          [&](int d) {
            if constexpr (Q8)
              return (float)(T)(e4m3_values(((const uint8_t*)a.v)[row * D + d],
                                            scale_of(a.v_scale[row]))[0]);
            else
              return (float)((const T*)a.v)[row * D + d];
          },
          [&](int d, float v) {
#pragma unroll
            for (int i = 0; i < NT * 16; ++i)
              if (d == (i >> 4) * 32 + (i & 3) + 8 * ((i & 15) >> 2) +
                           4 * hi &&
                  key < seen)
                o[i >> 4][i & 15] += v;
          });
    }
  }

  sum = lane_xor32_add(sum);
  if (!real) return;
  if (mine.active == 1) {
    const bool none = seen == 0;
    const float inv = s.broken ? nan_f32() : none ? 0.0f : 1.0f / sum;
    T* dst = (T*)a.out +
             ((long long)(s.q0 + my.t) * a.Hq + h * a.G + my.g) * D;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int j = 0; j < 16; j += 4) {
        T y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          y[i] = none && !s.broken ? (T)0.0f : (T)(o[t][j + i] * inv);
        __builtin_memcpy(dst + t * 32 + 2 * j + 4 * hi, y, sizeof y);
      }
  } else {
    const long long at =
        (((long long)place * a.Hk + h) * a.splits + split) * BM + wave * 32 +
        col;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int j = 0; j < 16; j += 4)
        *reinterpret_cast<f4*>(a.parts + at * D + t * 32 + 2 * j + 4 * hi) =
            f4{o[t][j], o[t][j + 1], o[t][j + 2], o[t][j + 3]};
    if (hi == 0) *reinterpret_cast<f2*>(a.stats + at * 2) = f2{m, sum};
  }
}

// Up to 4 workgroups for the rows of an item of the few kernel: that in which
// worker w > 0 has its edge, if it is the first edge in it.
template <typename K, int D, int GS>
__global__ void __launch_bounds__(256) join_few_kernel(Args a) {
  constexpr int BM = 16, ROWS = 256 / (D / 4) / GS;
  const int w = blockIdx.x + 1;
  Chunk c;
  const Line line = line_of(a, c, BM);
  const int at = w * line.per;
  if (at >= line.head * a.Hk) return;
  const int h = (int)((uint32_t)at / (uint32_t)line.head);
  const Item it = item_at(a, c, at - h * line.head, BM);
  if (it.seq < 0 || it.units < WHOLE) return;
  const int first = h * line.head + it.first;
  if (at - first < NEAR || first + it.units - at < NEAR ||
      at - line.per - first >= NEAR)
    return;
  const Span s = span_of(a, c, it.seq, it.tile * BM);
  const Parts p = parts_of(line, first, it.units);
  for (int row = blockIdx.y * ROWS; row < BM && s.row0 + row < s.rows;
       row += gridDim.y * ROWS) {
    join_rows<K, D, GS>(a, s, h, p, BM, row);
    __syncthreads();
  }
}

// Some workgroups for the rows of a tile of the many kernel.
template <typename K, int D, int GS>
__global__ void __launch_bounds__(256) join_many_kernel(Args a) {
  constexpr int BM = 128, ROWS = 256 / (D / 4) / GS;
  const Span s = find<BM>(a, blockIdx.x / a.Hk);
  if (s.seq < 0) return;
  Parts p;
  p.count = share_of((most_seen(a, s, BM) + MANY_KEYS - 1) / MANY_KEYS,
                     a.splits, 0, MANY_LEAST).active;
  if (p.count == 1) return;
  p.part0 = (long long)blockIdx.x * a.splits;
  p.part1 = p.part0 + 1;
  p.stride = 1;
  for (int row = blockIdx.y * ROWS; row < BM && s.row0 + row < s.rows;
       row += gridDim.y * ROWS) {
    join_rows<K, D, GS>(a, s, blockIdx.x % a.Hk, p, BM, row);
    __syncthreads();
  }
}

// ---- launching ------------------------------------------------------------

template <int D, int GS>
dim3 join_grid(int items, int BM) {
  constexpr int ROWS = 256 / (D / 4) / GS;
  const int n = (BM + ROWS - 1) / ROWS;
  // 4 for an item's rows where there are items for all units, so that the
  // search for the item counts less (9 prompts and steps, 12 heads, D = 64:
  // 48.2 us with one for each 16 rows, 47.1 so); otherwise one for each ROWS
  // (4 sequences of 62 tokens, 15 / 3 heads, D = 128: 33.9 with 4, 27.1)
  return dim3(items, n > 4 && (BM == 16 || items >= 256) ? 4 : n);
}

// Many parts of few rows: 8 groups of lanes for a row, or one (us, 32 / 8
// heads, D = 128; one token on 131000 keys, 32 parts an item: 99.9/103.8; one
// each of 4 sequences on 30000, 8 parts: 93.1/93.3, of 8 on 4000, 4 parts:
// 32.7/32.2; many kernel, 8 tokens on 30000 keys, 64 parts: 31.5/41.6, 64
// tokens, 32 parts: 63.6/65.5).
template <typename K, int D>
int join_few(Args& a, hipStream_t stream) {
  void* args[] = {&a};
  const long long items =
      (long long)a.Hk * max((long long)a.B, (long long)a.T * a.G / 16);
  if (a.workers == 1) return 0;
  return (int)(a.workers / items >= 16
      ? hipLaunchKernel(
            reinterpret_cast<const void*>(&join_few_kernel<K, D, 8>),
            join_grid<D, 8>(a.workers - 1, 16), dim3(256), args, 0, stream)
      : hipLaunchKernel(
            reinterpret_cast<const void*>(&join_few_kernel<K, D, 1>),
            join_grid<D, 1>(a.workers - 1, 16), dim3(256), args, 0, stream));
}

template <typename K, int D>
int join_many(Args& a, int tiles, hipStream_t stream) {
  void* args[] = {&a};
  return (int)(a.splits >= 16 && tiles * a.Hk <= 32
      ? hipLaunchKernel(
            reinterpret_cast<const void*>(&join_many_kernel<K, D, 8>),
            join_grid<D, 8>(tiles * a.Hk, 128), dim3(256), args, 0, stream)
      : hipLaunchKernel(
            reinterpret_cast<const void*>(&join_many_kernel<K, D, 1>),
            join_grid<D, 1>(tiles * a.Hk, 128), dim3(256), args, 0, stream));
}

// workers: 0 where the many kernel runs; of the few kernel otherwise, of 4 or
// 8 waves each. join: they share all items out, and a second kernel joins what
// they split; otherwise an item is a workgroup's. splits: of the many kernel.
struct Plan {
  int workers, waves, join, splits;
};

template <typename K, int D, int DV, bool Q8, int WAVES, bool SHARED>
int few(Args& a, int workgroups, hipStream_t stream) {
  void* args[] = {&a};
  return (int)hipLaunchKernel(
      reinterpret_cast<const void*>(&few_kernel<K, D, DV, Q8, WAVES, SHARED>),
      dim3(workgroups), dim3(WAVES * 64), args, 0, stream);
}

// Whole items. Where they are half of the units or less, two or four workgroups
// take an item: each all of K, and its part of V and of the result, which leaves
// nothing to join (us, 32 / 8 heads, D = 128, one, two, four: 8 sequences of 700
// keys 11.6, 11.1, 10.6, at 8 bits 10.1, 8.5, 8.5; 16 of 560 at 8 bits 9.5, 8.2;
// 1 of 128 6.1, 5.6, 5.2).
template <typename K, int D, bool Q8>
int whole(Args& a, const Plan& p, int tiles, hipStream_t stream) {
  const int items = (tiles * a.Hk + 7) / 8 * 8;  // of each 8, one an XCD
  const int busy = a.Hk * max(a.B, (int)((long long)a.T * a.G / 16));
  constexpr int W = Q8 ? 8 : 4;
  if constexpr (D == 128)
    if (busy <= 64) return few<K, D, 32, Q8, W, false>(a, items * 4, stream);
  if constexpr (D >= 64)
    if (busy <= 128)
      return few<K, D, D / 2, Q8, W, false>(a, items * 2, stream);
  return Q8 && p.waves == 8 ? few<K, D, D, Q8, W, false>(a, items, stream)
                            : few<K, D, D, Q8, 4, false>(a, items, stream);
}

template <typename K, int D, bool Q8>
int run(Args a, const Plan& p, hipStream_t stream) {
  const int BM = p.workers ? 16 : 128;
  const int tiles = (int)((long long)a.T * a.G / BM) + a.B;
  if (p.workers) {
    a.workers = p.workers;
    a.stats = a.parts + 2LL * a.workers * BM * D;
    const int rc =
        !p.join ? whole<K, D, Q8>(a, p, tiles, stream)
        : p.waves == 8 ? few<K, D, D, Q8, 8, true>(a, a.workers, stream)
                       : few<K, D, D, Q8, 4, true>(a, a.workers, stream);
    return rc || !p.join ? rc : join_few<K, D>(a, stream);
  }
  a.splits = p.splits;
  a.sorted = (long long)tiles * a.Hk * a.splits > 768;
  a.stats = a.parts + (long long)tiles * a.Hk * a.splits * BM * D;
  void* args[] = {&a};
  int rc = (int)hipLaunchKernel(
      reinterpret_cast<const void*>(&many_kernel<K, D, Q8>),
      dim3(tiles * a.Hk * a.splits), dim3(256), args, 0, stream);
  return rc || a.splits == 1 ? rc : join_many<K, D>(a, tiles, stream);
}

template <typename K, bool Q8>
int run_d(const Args& a, const Plan& p, int D, hipStream_t stream) {
  switch (D) {
    case 32: return run<K, 32, Q8>(a, p, stream);
    case 64: return run<K, 64, Q8>(a, p, stream);
    case 128: return run<K, 128, Q8>(a, p, stream);
  }
  return (int)hipErrorInvalidValue;
}

}  // namespace

extern "C" {

// parts: 32-bit floats, 2 * workers * 16 * (D + 2) of them where the few
// kernel's items are shared out (join), tiles * Hk * splits * 128 * (D + 2)
// for the many kernel's splits.
int tf_paged_attention(
    const void* q, const void* k, const void* v, const void* k_scale,
    const void* v_scale, const void* q_starts, const void* kv_lens,
    const void* table, void* out, void* parts, long long q_row,
    long long q_head, long long table_row, int cols, int T, int B, int Hq,
    int Hk, int pages, int page_log2, int D, float scale, int causal,
    int fp16, int workers, int waves, int join,
    int splits, void* stream) {
  if (T < 1 || B < 1 || Hk < 1 || Hq < 1 || Hq % Hk || Hq > 32768 || cols < 0 ||
      pages < 1 || page_log2 < 4 || page_log2 > 10 ||
      workers < 0 || (waves != 4 && waves != 8) || splits < 1 || splits > 65535 ||
      ((join || splits > 1) && !parts) ||
      ((long long)T * (Hq / Hk) / 16 + B) * Hk >= (1LL << 31) ||
      ((long long)T * (Hq / Hk) / 128 + B) * Hk >= (1LL << 31) / splits ||
      (long long)T * (Hq / Hk) + 128LL * B >= (1LL << 31))
    return (int)hipErrorInvalidValue;
  Args a{q, k, v, (const uint8_t*)k_scale, (const uint8_t*)v_scale,
         (const int*)q_starts, (const int*)kv_lens, (const int*)table, out,
         (float*)parts, nullptr, q_row, q_head, table_row, cols, T, B, Hq, Hk,
         Hq / Hk, pages, page_log2,
         (uint32_t)(((1ULL << 32) + Hq / Hk - 1) / (Hq / Hk)),
         // 0 times a masked score would be NaN; this leaves every p 1 too, to
         // 2^-21 for the largest scores (1e-38 did not: they reach 3e38)
         scale == 0.0f ? 0x1p-149f : scale * 1.4426950408889634f, causal, 1, 0, 1, 0};
  // a line of less than 2^30 units, as bounded by what the host knows
  const double items = ((double)T * (Hq / Hk) / 16 + B) * Hk;
  while (items * (OWN + ((double)cols * (1 << page_log2) /
                         (32 << a.unit_log2)) + 1) >= (double)(1 << 30) &&
         a.unit_log2 < 25)
    ++a.unit_log2;
  const Plan p{workers, waves, join, splits};
  const bool q8 = k_scale != nullptr;
  hipStream_t st = (hipStream_t)stream;
  return fp16 ? (q8 ? run_d<Fp16, true>(a, p, D, st)
                    : run_d<Fp16, false>(a, p, D, st))
              : (q8 ? run_d<Bf16, true>(a, p, D, st)
                    : run_d<Bf16, false>(a, p, D, st));
}

}  // extern "C"
