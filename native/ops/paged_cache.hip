// Writing and reading a paged KV cache on gfx950.
//
//   write:       pages[slot] <- k, v                  (16 bits, or e4m3)
//   rope write:  q <- rope(q);  pages[slot] <- rope(k), v
//   read:        k, v <- pages[slot]
//
// A pool is [pages, Hk, page, D]; slot = page * page_size + offset. One row
// is the D values of one token and head; D/8 lanes hold it, 16 bytes each,
// and a workgroup of 256 lanes takes 256/(D/8) neighbouring tokens of ONE
// head: new tokens lie in neighbouring slots of a page, so what a workgroup
// stores is one run of memory, the scales' single bytes among it.
//
// Quantising (e4m3, OCP): e = the smallest whole number with
// max|x| <= 448 * 2^e, code = e4m3(x * 2^-e), to nearest even. max|x| is
// taken on the bits without the sign, where NaN > inf > every number: a row
// that holds either gets NaN codes throughout. 2^-e is exact, so is the
// product, and the only rounding is the code's. fp16 rows are held to
// +-61440 first: at e = 8 the next code stands for 65536, which fp16 lacks.
//
// Bound: HBM. Every byte moves once and there is no reuse; at decode sizes
// it is the launch.

#include "paged_common.h"

namespace {

using namespace paged;

constexpr int BLOCK = 256;

struct Pools {
  uint8_t* k;
  uint8_t* v;
  uint8_t* k_scale;
  uint8_t* v_scale;
  long long slots;  // pages * page_size
  int page_log2;
  int kv_heads;
};

__device__ inline long long row_of(const Pools& p, long long slot, int head) {
  long long page = slot >> p.page_log2;
  long long off = slot & ((1 << p.page_log2) - 1);
  return ((page * p.kv_heads + head) << p.page_log2) + off;
}

template <typename K, int D>
__device__ inline void store_row(uint8_t* pool, uint8_t* scales,
                                 long long row, int lane, const float* x,
                                 const Oct<K>& as_is, bool quantized,
                                 bool keep) {
  // every lane comes here, kept or not: the maximum below crosses lanes
  constexpr int LANES = D / 8;
  if (!quantized) {
    if (keep)
      *reinterpret_cast<u4*>(pool + (row * D + lane * 8) * 2) = as_is.raw;
    return;
  }
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    top = max(top, __float_as_uint(x[j]) & 0x7fffffffu);
#pragma unroll
  for (int m = 1; m < LANES; m <<= 1)
    top = max(top, (uint32_t)__shfl_xor((int)top, m, 64));
  // 448 = 1.75 * 2^8
  int e = (int)(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = max(e, 1);
  const bool broken = top >= 0x7f800000u;
  const float inv = __uint_as_float((uint32_t)(254 - e) << 23);
  float y[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float f = x[j];
    if constexpr (sizeof(typename K::T) == 2 &&
                  __is_same(typename K::T, _Float16))
      f = fminf(fmaxf(f, -61440.0f), 61440.0f);
    y[j] = broken ? nan_f32() : f * inv;
  }
  u2 codes = {e4m3_codes(y[0], y[1], y[2], y[3]),
              e4m3_codes(y[4], y[5], y[6], y[7])};
  if (!keep) return;
  *reinterpret_cast<u2*>(pool + row * D + lane * 8) = codes;
  if (lane == 0) scales[row] = broken ? 127 : (uint8_t)e;
}

// A lane has the same 8 values of HEADS heads of one token: their loads are
// on their way together, and the rotation's cosines and sines, as many bytes
// as a head's values, are loaded once for them.
template <typename K, int D, bool ROPE, bool Q8, int HEADS>
__global__ void __launch_bounds__(BLOCK)
write_kernel(const typename K::T* __restrict__ q,
             const typename K::T* __restrict__ k,
             const typename K::T* __restrict__ v, long long q_row,
             long long k_row, long long k_head, long long v_row,
             long long v_head, const float* __restrict__ cos_t,
             const float* __restrict__ sin_t,
             const long long* __restrict__ pos, int positions,
             const long long* __restrict__ slots, typename K::T* q_out,
             Pools pools, int n, int heads) {
  constexpr int LANES = D / 8, ROWS = BLOCK / LANES;
  const int lane = threadIdx.x % LANES;
  const int t = blockIdx.x * ROWS + threadIdx.x / LANES;
  const int at = min(t, n - 1);  // lanes past the end work on a copy
  const int d0 = lane * 8;
  const int all = heads + 2 * pools.kv_heads;
  const int h0 = blockIdx.y * HEADS;

  Oct<K> in[HEADS];
#pragma unroll
  for (int i = 0; i < HEADS; ++i) {
    const int h = min(h0 + i, all - 1);
    const typename K::T* src =
        h < heads ? q + at * q_row + (long long)h * D
        : h >= heads + pools.kv_heads
            ? v + at * v_row + (h - heads - pools.kv_heads) * v_head
            : k + at * k_row + (h - heads) * k_head;
    // A projection's output is read once: marked so, its large q leaves the
    // caches to the q that is written, which attention reads next.
    in[i].raw = ROPE ? __builtin_nontemporal_load(
                           reinterpret_cast<const u4*>(src + d0))
                     : *reinterpret_cast<const u4*>(src + d0);
  }
  const long long slot = h0 + HEADS > heads ? slots[at] : -1;
  const bool keep = t < n && slot >= 0 && slot < pools.slots;
  f4 c = {1, 1, 1, 1}, s = {0, 0, 0, 0};
  if (ROPE && h0 < heads + pools.kv_heads) {
    // interleaved pairs (2j, 2j+1) against tables [positions, D/2]; a
    // position outside of them answers NaN
    const long long p = pos[at];
    const bool known = p >= 0 && p < positions;
    const long long base = (known ? p : 0) * (D / 2) + d0 / 2;
    c = *reinterpret_cast<const f4*>(cos_t + base);
    s = *reinterpret_cast<const f4*>(sin_t + base);
    if (!known) c = f4{nan_f32(), nan_f32(), nan_f32(), nan_f32()};
  }
#pragma unroll
  for (int i = 0; i < HEADS; ++i) {
    int h = h0 + i;
    if (h >= all) return;
    const bool is_v = h >= heads + pools.kv_heads;
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = (float)in[i].h[j];
    if (ROPE && !is_v) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float a = x[2 * j], b = x[2 * j + 1];
        x[2 * j] = a * c[j] - b * s[j];
        x[2 * j + 1] = b * c[j] + a * s[j];
      }
      // one rounding, from the 32-bit product
#pragma unroll
      for (int j = 0; j < 8; ++j) in[i].h[j] = (typename K::T)x[j];
    }
    if (ROPE && h < heads) {
      if (t < n)
        *reinterpret_cast<u4*>(q_out + ((long long)t * heads + h) * D + d0) =
            in[i].raw;
      continue;
    }
    h -= is_v ? heads + pools.kv_heads : heads;
    const long long row = keep ? row_of(pools, slot, h) : 0;
    store_row<K, D>(is_v ? pools.v : pools.k,
                    is_v ? pools.v_scale : pools.k_scale, row, lane, x, in[i],
                    Q8, keep);
  }
}

template <typename K, int D, bool Q8>
__global__ void __launch_bounds__(BLOCK)
read_kernel(Pools pools, const long long* __restrict__ slots,
            typename K::T* __restrict__ k, typename K::T* __restrict__ v,
            int n) {
  constexpr int LANES = D / 8, ROWS = BLOCK / LANES;
  const int lane = threadIdx.x % LANES;
  const int t = blockIdx.x * ROWS + threadIdx.x / LANES;
  if (t >= n) return;
  int h = blockIdx.y;
  const bool is_v = h >= pools.kv_heads;
  if (is_v) h -= pools.kv_heads;
  const long long slot = slots[t];
  Oct<K> out;
  if (slot < 0 || slot >= pools.slots) {
    // no slot reads 0; one past the pool is a mistake, and reads NaN
    float x = slot < 0 ? 0.0f : nan_f32();
#pragma unroll
    for (int j = 0; j < 8; ++j) out.h[j] = (typename K::T)x;
  } else {
    const uint8_t* pool = is_v ? pools.v : pools.k;
    const long long row = row_of(pools, slot, h);
    if constexpr (Q8) {
      const float s =
          scale_of((is_v ? pools.v_scale : pools.k_scale)[row]);
      u2 codes = *reinterpret_cast<const u2*>(pool + row * D + lane * 8);
      f4 a = e4m3_values(codes[0], s), b = e4m3_values(codes[1], s);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        out.h[j] = (typename K::T)a[j];
        out.h[4 + j] = (typename K::T)b[j];
      }
    } else {
      out.raw = *reinterpret_cast<const u4*>(pool + (row * D + lane * 8) * 2);
    }
  }
  typename K::T* dst = is_v ? v : k;
  *reinterpret_cast<u4*>(
      dst + ((long long)t * pools.kv_heads + h) * D + lane * 8) = out.raw;
}

struct WriteArgs {
  const void *q, *k, *v;
  long long q_row, k_row, k_head, v_row, v_head;
  const float *cos_t, *sin_t;
  const long long* pos;
  int positions;
  const long long* slots;
  void* q_out;
  Pools pools;
  int n, heads;
};

template <typename K, int D, bool ROPE, bool Q8, int HEADS>
int launch_write_by(WriteArgs& a, hipStream_t stream) {
  constexpr int ROWS = BLOCK / (D / 8);
  dim3 grid((a.n + ROWS - 1) / ROWS,
            (a.heads + 2 * a.pools.kv_heads + HEADS - 1) / HEADS);
  void* args[] = {&a.q,       &a.k,      &a.v,         &a.q_row, &a.k_row,
                  &a.k_head,  &a.v_row,  &a.v_head,    &a.cos_t, &a.sin_t,
                  &a.pos,     &a.positions, &a.slots,  &a.q_out, &a.pools,
                  &a.n,       &a.heads};
  return (int)hipLaunchKernel(
      reinterpret_cast<const void*>(&write_kernel<K, D, ROPE, Q8, HEADS>),
      grid, dim3(BLOCK), args, 0, stream);
}

template <typename K, int D, bool ROPE, bool Q8>
int launch_write(WriteArgs& a, hipStream_t stream) {
  // 4 heads a lane once that still fills the card: 8190 tokens of 64 + 2 * 8
  // heads take 57 us against 81 us with one (73 us without the marked loads);
  // 8 tokens take 2.4 us with one.
  const long long rows =
      (long long)a.n * (a.heads + 2 * a.pools.kv_heads) * (D / 8);
  return rows >= 4LL * 2048 * BLOCK
             ? launch_write_by<K, D, ROPE, Q8, 4>(a, stream)
             : launch_write_by<K, D, ROPE, Q8, 1>(a, stream);
}

template <typename K, bool ROPE, bool Q8>
int write_d(WriteArgs& a, int D, hipStream_t stream) {
  switch (D) {
    case 32: return launch_write<K, 32, ROPE, Q8>(a, stream);
    case 64: return launch_write<K, 64, ROPE, Q8>(a, stream);
    case 128: return launch_write<K, 128, ROPE, Q8>(a, stream);
  }
  return (int)hipErrorInvalidValue;
}

template <typename K>
int write_any(WriteArgs& a, int D, bool rope, bool q8, hipStream_t s) {
  return rope ? (q8 ? write_d<K, true, true>(a, D, s)
                    : write_d<K, true, false>(a, D, s))
              : (q8 ? write_d<K, false, true>(a, D, s)
                    : write_d<K, false, false>(a, D, s));
}

template <typename K, int D, bool Q8>
int launch_read(Pools pools, const long long* slots, void* k, void* v, int n,
                hipStream_t stream) {
  constexpr int ROWS = BLOCK / (D / 8);
  dim3 grid((n + ROWS - 1) / ROWS, 2 * pools.kv_heads);
  void* args[] = {&pools, &slots, &k, &v, &n};
  return (int)hipLaunchKernel(
      reinterpret_cast<const void*>(&read_kernel<K, D, Q8>), grid,
      dim3(BLOCK), args, 0, stream);
}

template <typename K>
int read_any(Pools p, const long long* slots, void* k, void* v, int n, int D,
             bool q8, hipStream_t s) {
  switch (D) {
    case 32: return q8 ? launch_read<K, 32, true>(p, slots, k, v, n, s)
                       : launch_read<K, 32, false>(p, slots, k, v, n, s);
    case 64: return q8 ? launch_read<K, 64, true>(p, slots, k, v, n, s)
                       : launch_read<K, 64, false>(p, slots, k, v, n, s);
    case 128: return q8 ? launch_read<K, 128, true>(p, slots, k, v, n, s)
                        : launch_read<K, 128, false>(p, slots, k, v, n, s);
  }
  return (int)hipErrorInvalidValue;
}

// what both entries ask of the numbers that they are given
bool fine(int n, int heads, int kv_heads, int page_log2, long long pages) {
  return n > 0 && heads >= 0 && kv_heads > 0 && pages > 0 &&
         page_log2 >= 4 && page_log2 <= 10 &&
         (long long)heads + 2LL * kv_heads <= 65535;
}

}  // namespace

extern "C" {

// k, v: n rows of [kv_heads, D]; q: n rows of heads * D values, rotated to
// q_out along with k where cos_t is given. fp16: whether the rows are fp16
// (bf16 otherwise). k_scale and v_scale are null for a 16-bit cache.
int tf_paged_write(const void* q, const void* k, const void* v,
                   long long q_row, long long k_row, long long k_head,
                   long long v_row, long long v_head, const void* cos_t,
                   const void* sin_t, const void* pos, int positions,
                   const void* slots, void* q_out, void* k_pool, void* v_pool,
                   void* k_scale, void* v_scale, long long pages,
                   int page_log2, int n, int heads, int kv_heads, int D,
                   int fp16, void* stream) {
  if (!fine(n, heads, kv_heads, page_log2, pages))
    return (int)hipErrorInvalidValue;
  WriteArgs a{q, k, v, q_row, k_row, k_head, v_row, v_head,
              (const float*)cos_t, (const float*)sin_t,
              (const long long*)pos, positions, (const long long*)slots,
              q_out,
              {(uint8_t*)k_pool, (uint8_t*)v_pool, (uint8_t*)k_scale,
               (uint8_t*)v_scale, pages << page_log2, page_log2, kv_heads},
              n, heads};
  const bool rope = cos_t != nullptr, q8 = k_scale != nullptr;
  return fp16 ? write_any<Fp16>(a, D, rope, q8, (hipStream_t)stream)
              : write_any<Bf16>(a, D, rope, q8, (hipStream_t)stream);
}

// k, v: n rows of [kv_heads, D], without gaps
int tf_paged_read(const void* k_pool, const void* v_pool, const void* k_scale,
                  const void* v_scale, long long pages, int page_log2,
                  const void* slots, void* k, void* v, int n, int kv_heads,
                  int D, int fp16, void* stream) {
  if (!fine(n, 0, kv_heads, page_log2, pages))
    return (int)hipErrorInvalidValue;
  Pools p{(uint8_t*)k_pool, (uint8_t*)v_pool, (uint8_t*)k_scale,
          (uint8_t*)v_scale, pages << page_log2, page_log2, kv_heads};
  const bool q8 = k_scale != nullptr;
  return fp16 ? read_any<Fp16>(p, (const long long*)slots, k, v, n, D, q8,
                               (hipStream_t)stream)
              : read_any<Bf16>(p, (const long long*)slots, k, v, n, D, q8,
                               (hipStream_t)stream);
}

}  // extern "C"
