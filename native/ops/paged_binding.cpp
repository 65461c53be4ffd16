// The paged operators' entry from Python: checks, outputs, workspaces and the
// launch in one call of about 5 us, of which the launch itself is 3. (Through
// ctypes, with the checks in Python, rope_kv_write took 15 us a call, five
// times what its kernel takes for a decode step.)
//
// Everything that can be known without waiting for the GPU is checked here,
// before anything is launched: a ValueError, or a RuntimeError where a
// gradient is asked for. No C++ exception leaves a function.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/AutogradState.h>
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <new>
#include <sstream>
#include <stdexcept>
#include <string>

extern "C" {
int tf_paged_write(const void* q, const void* k, const void* v,
                   long long q_row, long long k_row, long long k_head,
                   long long v_row, long long v_head, const void* cos_t,
                   const void* sin_t, const void* pos, int positions,
                   const void* slots, void* q_out, void* k_pool, void* v_pool,
                   void* k_scale, void* v_scale, long long pages,
                   int page_log2, int n, int heads, int kv_heads, int D,
                   int fp16, void* stream);
int tf_paged_read(const void* k_pool, const void* v_pool, const void* k_scale,
                  const void* v_scale, long long pages, int page_log2,
                  const void* slots, void* k, void* v, int n, int kv_heads,
                  int D, int fp16, void* stream);
int tf_paged_attention(
    const void* q, const void* k, const void* v, const void* k_scale,
    const void* v_scale, const void* q_starts, const void* kv_lens,
    const void* table, void* out, void* parts, long long q_row,
    long long q_head, long long table_row, int cols, int T, int B, int Hq,
    int Hk, int pages, int page_log2, int D, float scale, int causal,
    int fp16, int workers, int waves, int join, int splits, void* stream);
}

namespace {

using at::Tensor;

struct NoBackward : std::runtime_error {
  using std::runtime_error::runtime_error;
};

template <typename... A>
[[noreturn]] void refuse(const A&... parts) {
  std::ostringstream s;
  (s << ... << parts);
  throw std::invalid_argument(s.str());
}

struct Shape {
  at::IntArrayRef of;
};
Shape shape(const Tensor& t) { return {t.sizes()}; }
std::ostream& operator<<(std::ostream& s, const Shape& x) {
  s << "(";
  for (size_t i = 0; i < x.of.size(); ++i) s << (i ? ", " : "") << x.of[i];
  return s << ")";
}

// ---- the pools of a cache -----------------------------------------------------

struct Pools {
  Tensor k, v, k_scale, v_scale;
  int64_t pages;
  int kv_heads, page_log2, D;
  bool quantized;
  at::ScalarType dtype;
  at::Device device{at::kCPU};
};

struct PoolsObject {
  PyObject_HEAD
  Pools p;
};

PyTypeObject* pools_type = nullptr;

bool wide(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf; }

// bytes from the first value to the end of the last one; t has values
size_t extent(const Tensor& t) {
  const auto sizes = t.sizes(), strides = t.strides();
  int64_t last = 0;
  for (size_t i = 0; i < sizes.size(); ++i) last += (sizes[i] - 1) * strides[i];
  return (last + 1) * t.itemsize();
}

// A kernel is given addresses: what lies there has to be the tensor's values.
// It is not where a Python class or a function transform stands between (fake,
// distributed and batched tensors), where a sign is still to be applied, or
// where the storage has been taken away.
void check_plain(const char* name, const Tensor& t) {
  using c10::DispatchKey;
  constexpr c10::DispatchKeySet between(
      {DispatchKey::Python, DispatchKey::Functionalize,
       DispatchKey::FuncTorchGradWrapper, DispatchKey::FuncTorchBatched,
       DispatchKey::Batched, DispatchKey::ZeroTensor, DispatchKey::Negative,
       DispatchKey::Conjugate});
  if (t.layout() != at::kStrided || t.is_nested() ||
      t.key_set().has_any(between) ||
      (t.numel() && t.storage_offset() * t.itemsize() + extent(t) >
                        t.storage().nbytes()))
    refuse(name, " is a plain tensor: dense, with its values in its memory");
}

// what is allocated here: under a mode that fakes tensors, so is that
Tensor fresh(Tensor t) {
  check_plain("a result", t);
  return t;
}

Tensor tensor_of(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse(name, " is a tensor");
  Tensor t = THPVariable_Unpack(o);
  check_plain(name, t);
  return t;
}

bool aligned(const Tensor& t) {
  return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
}

void check_pools(Pools& p) {
  const Tensor &k = p.k, &v = p.v;
  check_plain("k", k);
  check_plain("v", v);
  if (p.k_scale.defined()) check_plain("k_scale", p.k_scale);
  if (p.v_scale.defined()) check_plain("v_scale", p.v_scale);
  if (k.dim() != 4 || k.sizes() != v.sizes())
    refuse("k and v pools are [pages, kv_heads, page_size, head_dim], of one "
           "shape: got ", shape(k), " and ", shape(v));
  const int64_t pages = k.size(0), heads = k.size(1), page = k.size(2),
                D = k.size(3);
  if (D != 32 && D != 64 && D != 128)
    refuse("head_dim is one of (32, 64, 128): ", D);
  if (page < 16 || page > 1024 || (page & (page - 1)))
    refuse("page_size is a power of two from 16 to 1024: ", page);
  if (pages < 1 || heads < 1 || heads > 4096)
    refuse("no pool of ", pages, " pages, ", heads, " heads");
  if (pages >= (1LL << 31) / page)
    refuse(pages, " pages of ", page, " tokens: a pool holds less than 2**31 "
           "tokens");
  p.dtype = k.scalar_type();
  p.quantized = p.dtype == at::kFloat8_e4m3fn;
  if ((!p.quantized && !wide(p.dtype)) || v.scalar_type() != p.dtype)
    refuse("pools are both bfloat16, float16 or float8_e4m3fn: got ", p.dtype,
           ", ", v.scalar_type());
  for (const Tensor* s : {&p.k_scale, &p.v_scale}) {
    if (!p.quantized) {
      if (s->defined()) refuse("a ", p.dtype, " pool has no scales");
    } else if (!s->defined() || s->scalar_type() != at::kByte ||
               s->sizes() != k.sizes().slice(0, 3)) {
      refuse("a float8_e4m3fn pool has a uint8 scale of shape ",
             Shape{k.sizes().slice(0, 3)});
    }
  }
  for (const Tensor* x : {&p.k, &p.v, &p.k_scale, &p.v_scale})
    if (x->defined() && (!x->is_contiguous() || !aligned(*x) ||
                         x->device() != k.device()))
      refuse("pools and scales lie on one device, without gaps, at multiples "
             "of 16 bytes");
  p.pages = pages;
  p.kv_heads = (int)heads;
  p.page_log2 = __builtin_ctzll(page);
  p.D = (int)D;
  p.device = k.device();
}

// looked at again at every call: a tensor can be resized, or given other memory
const Pools& pools_of(PyObject* o) {
  if (!PyObject_TypeCheck(o, pools_type)) refuse("a PagedKVCache is wanted");
  Pools& p = reinterpret_cast<PoolsObject*>(o)->p;
  check_pools(p);
  return p;
}

// ---- what the operators ask of their arguments --------------------------------

void on_gpu(const Pools& p, std::initializer_list<const Tensor*> all) {
  for (const Tensor* t : all)
    if (t->device() != p.device)
      refuse("tensors on ", t->device(), " and a cache on ", p.device);
  if (!p.device.is_cuda())
    refuse("the paged operators run on a GPU: got ", p.device);
}

// neither a backward pass nor a tangent
void no_grad(std::initializer_list<const Tensor*> all) {
  const bool backward = at::GradMode::is_enabled(),
             forward = c10::AutogradState::get_tls_state().get_fw_grad_mode();
  for (const Tensor* t : all)
    if (t->defined() && ((backward && t->requires_grad()) ||
                         (forward && t->_fw_grad(0).defined())))
      throw NoBackward("the paged operators have no backward pass and no "
                       "forward mode: call them under torch.no_grad(), and "
                       "without tangents");
}

void check_rows(const Pools& p, std::initializer_list<const Tensor*> all) {
  const at::ScalarType t = (*all.begin())->scalar_type();
  if (!wide(t)) refuse("rows are bfloat16 or float16: got ", t);
  if (!p.quantized && t != p.dtype)
    refuse(t, " rows for a ", p.dtype, " cache");
  for (const Tensor* x : all)
    if (x->scalar_type() != t)
      refuse("rows of one type: got ", t, ", ", x->scalar_type());
}

void check_index(const char* name, const Tensor& x, int64_t n) {
  if (x.scalar_type() != at::kLong || x.dim() != 1 || x.size(0) != n ||
      !x.is_contiguous())
    refuse(name, " is int64 [", n, "] without gaps: got ", x.scalar_type(),
           " ", shape(x));
}

// x, or a copy of it where 16-byte loads do not fit its layout
Tensor rows_of(const Tensor& x) {
  bool fits = x.stride(-1) == 1 && aligned(x);
  for (int64_t i = 0; i + 1 < x.dim(); ++i) fits = fits && x.stride(i) % 8 == 0;
  return fits ? x : fresh(x.clone(at::MemoryFormat::Contiguous));
}

// whether any byte between the first and the last of one lies there of another
bool overlap(const Tensor& a, const Tensor& b) {
  if (!a.defined() || !b.defined() || !a.numel() || !b.numel()) return false;
  auto at = [](const Tensor& t) {
    return reinterpret_cast<uintptr_t>(t.data_ptr());
  };
  return at(a) < at(b) + extent(b) && at(b) < at(a) + extent(a);
}

// rows to be written, and not from under them: rows that lie in the cache are
// copied before
Tensor source_of(const Pools& p, const Tensor& x) {
  for (const Tensor* pool : {&p.k, &p.v, &p.k_scale, &p.v_scale})
    if (overlap(x, *pool)) return fresh(x.clone(at::MemoryFormat::Contiguous));
  return rows_of(x);
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

void* stream_of(const Pools& p) {
  return c10::hip::getCurrentHIPStream(p.device.index()).stream();
}

void launched(const char* name, int rc) {
  if (rc)
    throw std::runtime_error(std::string(name) + " failed: " +
                             std::to_string(rc));
}

// of less than 2^32 lanes in all, in workgroups of 256
constexpr int64_t LAUNCH = 1LL << 24;

// rows of the cache, at 2048 / D a workgroup
void check_count(const Pools& p, int64_t n) {
  if (n > (LAUNCH - 1) * (2048 / p.D)) refuse("too many rows (", n, ")");
}

// written in place: autograd notices where it had kept the values
void changed(const Tensor& t) {
  if (t.defined() && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

void write(const Pools& p, const Tensor& q, const Tensor& k, const Tensor& v,
           int64_t k_head, int64_t v_head, const Tensor& cos,
           const Tensor& sin, const Tensor& pos, const Tensor& slots,
           const Tensor& q_out, int n, int heads) {
  launched("tf_paged_write",
           tf_paged_write(
               ptr(q), ptr(k), ptr(v), q.defined() ? q.stride(0) : 0,
               k.stride(0), k_head, v.stride(0), v_head, ptr(cos), ptr(sin),
               ptr(pos), cos.defined() ? (int)cos.size(0) : 0, ptr(slots),
               ptr(q_out), ptr(p.k), ptr(p.v), ptr(p.k_scale), ptr(p.v_scale),
               p.pages, p.page_log2, n, heads, p.kv_heads, p.D,
               k.scalar_type() == at::kHalf, stream_of(p)));
  for (const Tensor* t : {&p.k, &p.v, &p.k_scale, &p.v_scale}) changed(*t);
}

void kv_write(const Pools& p, Tensor k, Tensor v, const Tensor& slots) {
  const int64_t n = k.dim() ? k.size(0) : 0;
  const int64_t want[] = {n, p.kv_heads, p.D};
  if (k.sizes() != at::IntArrayRef(want) || v.sizes() != at::IntArrayRef(want))
    refuse("k and v are ", Shape{want}, ": got ", shape(k), " and ", shape(v));
  check_rows(p, {&k, &v});
  check_index("slots", slots, n);
  check_count(p, n);
  no_grad({&k, &v, &p.k, &p.v});
  on_gpu(p, {&k, &v, &slots});
  if (n == 0) return;
  const c10::DeviceGuard guard(p.device);
  k = source_of(p, k);
  v = source_of(p, v);
  write(p, Tensor(), k, v, k.stride(1), v.stride(1), Tensor(), Tensor(),
        Tensor(), slots, Tensor(), (int)n, 0);
}

Tensor rope_kv_write(const Pools& p, Tensor q_in, Tensor k_in, Tensor v_in,
                     const Tensor& cos, const Tensor& sin, const Tensor& pos,
                     const Tensor& slots, int64_t heads) {
  const int64_t n = q_in.dim() ? q_in.size(0) : 0, D = p.D;
  if (heads < 1 || heads > 65535 || q_in.dim() != 2 ||
      q_in.size(1) != heads * D)
    refuse("q_in is [n, ", heads, " * ", D, "]: got ", shape(q_in));
  const int64_t want[] = {n, p.kv_heads * D};
  if (k_in.sizes() != at::IntArrayRef(want) ||
      v_in.sizes() != at::IntArrayRef(want))
    refuse("k_in and v_in are ", Shape{want}, ": got ", shape(k_in), " and ",
           shape(v_in));
  check_rows(p, {&q_in, &k_in, &v_in});
  for (const Tensor* x : {&cos, &sin})
    if (x->scalar_type() != at::kFloat || x->dim() != 2 || x->size(0) < 1 ||
        x->size(0) >= (1LL << 31) || x->sizes() != cos.sizes() ||
        x->size(1) != D / 2 || !x->is_contiguous() || !aligned(*x))
      refuse("cos and sin are float32 [positions, ", D / 2, "] without gaps");
  check_index("pos", pos, n);
  check_index("slots", slots, n);
  if (heads + 2 * p.kv_heads > 65535) refuse("too many heads (", heads, ")");
  check_count(p, n);
  no_grad({&q_in, &k_in, &v_in, &cos, &sin, &p.k, &p.v});
  on_gpu(p, {&q_in, &k_in, &v_in, &cos, &sin, &pos, &slots});
  const c10::DeviceGuard guard(p.device);
  Tensor q =
      fresh(at::empty({n, heads, D}, q_in.options().requires_grad(false)));
  if (n == 0) return q;
  q_in = source_of(p, q_in);
  k_in = source_of(p, k_in);
  v_in = source_of(p, v_in);
  write(p, q_in, k_in, v_in, D, D, cos, sin, pos, slots, q, (int)n,
        (int)heads);
  return q;
}

std::pair<Tensor, Tensor> kv_read(const Pools& p, const Tensor& slots,
                                  at::ScalarType dtype) {
  if (!wide(dtype) || !(p.quantized || dtype == p.dtype))
    refuse("a ", p.dtype, " cache is not read as ", dtype);
  if (slots.dim() != 1) refuse("slots is int64 [n]: got ", shape(slots));
  const int64_t n = slots.size(0);
  check_index("slots", slots, n);
  check_count(p, n);
  no_grad({&p.k, &p.v});
  on_gpu(p, {&slots});
  const c10::DeviceGuard guard(p.device);
  const auto options = p.k.options().dtype(dtype);
  Tensor k = fresh(at::empty({n, p.kv_heads, p.D}, options));
  Tensor v = fresh(at::empty({n, p.kv_heads, p.D}, options));
  if (n)
    launched("tf_paged_read",
             tf_paged_read(ptr(p.k), ptr(p.v), ptr(p.k_scale), ptr(p.v_scale),
                           p.pages, p.page_log2, ptr(slots), ptr(k), ptr(v),
                           (int)n, p.kv_heads, p.D, dtype == at::kHalf,
                           stream_of(p)));
  return {k, v};
}

struct Plan {
  int64_t workers, waves, join, splits;
};

// Which kernel attends, and how it shares the keys. What a batch holds lies
// on the device; this goes by the mean number of rows a sequence and by the keys
// that the table could hold, and is right for any batch. It costs time where
// that is far from what the batch holds: 8 steps on 560 keys take 9.5 us in a
// table for 560 and 13.9 in one for 8192, 64 such steps 28.2 and 42.5 (32 / 8
// heads, D = 128, 16 bits); 200 steps on 500 to 4000 keys and 512 tokens over
// 4000 take 466 us in one call and 407 in two. Up to 16
// rows (new tokens * G) a sequence are work for the kernel for few rows, whose
// `workers` share it out among themselves; 0 workers: the kernel for many
// rows, with the keys of each tile of 128 rows in `splits` parts.
//
// Few rows, an item (16 rows or less of a sequence and kv head) a workgroup, or
// all shared out: an item by itself takes `ns` a key, so where items are too
// few for the 256 units, or differ, sharing saves that for its keys times the
// part of the units that idles (taken as a third at least, for lengths that
// differ); it costs 7 us: 4.5 for the joining kernel, the rest for the search
// and the parts. Measured (us, D = 128, 8 kv heads, whole against shared):
// 16 bits, 1 sequence of 700 keys 9.3/14.4, of 1300 14.3/12.7; 8 of 1300
// 16.6/17.4, of 2400 26.7/20.1; 16 of up to 1300 17.2/21.5, of up to 4000
// 44.2/41.4; 32 of 1300 33.1/36.1, of up to 2400 44.8/47.9; 64 of up to 1300
// 45.3/53.9; 8 bits, 8 of 1300 12.0/16.3, of 2400 17.2/17.2; 16 of 2400
// 18.2/22.8; 64 of up to 1300 29.7/40.7; 48 of up to 2400 43.5/41.0.
//
// Waves: a unit holds 8 of the few kernel, as one workgroup or as two. Whole
// items come two to a unit while there are that many, and hide each other's
// latencies (64 sequences of 250 keys at 8 bits: 4 waves 10.9, 8 waves 14.7).
// With no more items than units, 8 waves are through with an 8-bit one sooner
// (8 sequences of 700 keys, a workgroup an item: 13.0/10.1); at 16 bits a unit's
// loads are what it waits for (8 of 560 11.6/11.6, of 256 8.0/8.5). Shared, one workgroup of 8
// has half the parts to join (512 of 4 waves against 256 of 8: 64 sequences
// of 700 to 8191 keys at 8 bits 117.7/115.5, one of 131000 at 16 bits
// 101.1/99.0, 4 of 1000 in a table for 8192 16.2/13.8), but not where the keys
// do not give every unit two (2 of 4000 15.2/15.8, 8 of 1699 18.3/19.4). More
// waves, which D of 32 and 64 have room for, gain nothing (24 sequences of 4000
// keys, D = 64: 512 workers 30.4, 768 31.9).
//
// Splits of the many kernel: a workgroup by itself takes 1.3 us for 64 keys, so
// s parts leave 1/s of 1.3 us * tiles of keys; they cost 4 us for the joining
// kernel, and s times the way of one part of all sums through memory, at 4 TB/s,
// there and back. That is least for an s of its own, and bounded by the places
// for workgroups: two a unit, three for D of 64 and 32. Of few sequences their
// tiles are known, and to fill the places exactly is best (512 tokens over 8000
// keys, 32 / 8 heads, D = 128: 4 parts 86.5, 3 parts 91.1, 6 parts 103.8; 2
// sequences of them: 2 parts 153, 3 parts 178). More sequences are uneven, and
// half more than two a unit balances them (9 of 295 rows on up to 2353 keys: 2
// parts 50.8, 3 parts 44.2; 32 of 64 rows on up to 8000: 2 parts 142, 3 parts
// 112), unless their tiles are mostly empty and memory is what they wait for
// (15 of 22 rows: 5 parts 32.5, 8 parts 37.2). Unsplit against split: 184 rows
// on 272 keys 11.0/13.9, 251 tokens of 64 heads on 288 keys 14.7/20.2, 40
// tokens of 32 heads on 688 keys 20.2/13.7, 65 on 4032 keys 109/32.5; as many
// as fit against the least: 2 of 64 tokens on 4064 keys 39.5/34.5.
Plan plan_of(int64_t T, int64_t B, int64_t G, int64_t Hk, int64_t D,
             int64_t keys, bool quantized) {
  const int64_t rows = T * G;
  // of keys that are worth a workgroup
  const int64_t pieces = std::max<int64_t>(1, (keys + 255) / 256);
  if (rows <= 16 * B) {
    const int64_t items = Hk * std::max(B, rows / 16);
    const int waves = quantized && items <= 256 ? 8 : 4;
    const double ns = !quantized     ? 2 + 0.054 * D
                      : items <= 128 ? std::min(1.8 + 0.034 * D, 4.3)
                      : items <= 256 ? 1.8 + 0.034 * D
                                     : 3.1 + 0.058 * D;
    const double idle = std::max(1 - items / 256.0, 1 / 3.0);
    if (keys * ns * idle <= 7000) return {Hk * (rows / 16 + B), waves, 0, 1};
    if (items * pieces >= 512) return {256, 8, 1, 1};
    // neighbouring workgroups share an XCD of eight
    return {(items * pieces + 7) / 8 * 8, 4, 1, 1};
  }
  const int64_t tiles =
      Hk * std::max(B, B < 4 ? (rows + 127) / 128 : rows / 128);
  const int64_t slots = B < 4 ? (D == 128 ? 512 : 768)
                        : rows < 64 * B ? 512 : 768;
  const double alone = 1.3 * keys / 64;
  const double part = (double)rows * Hk * D * 8 / 4e6;
  const int64_t splits = std::min(
      {pieces, slots / tiles, (int64_t)std::max(1.0, std::sqrt(alone / part))});
  if (splits <= 1 || alone * (1 - 1.0 / splits) <= 4 + part * splits)
    return {0, 4, 0, 1};
  return {0, 4, 0, splits};
}

Tensor attention(const Pools& p, Tensor q, const Tensor& starts,
                 const Tensor& lens, const Tensor& table, double scale,
                 bool causal, Tensor out) {
  if (q.dim() != 3) refuse("q is [tokens, heads, head_dim]: ", shape(q));
  const int64_t T = q.size(0), Hq = q.size(1), D = q.size(2),
                Hk = p.kv_heads;
  if (D != p.D || Hq < 1 || Hq % Hk)
    refuse("q ", shape(q), " for a cache of ", Hk, " heads of ", p.D);
  check_rows(p, {&q});
  if (lens.dim() != 1 || table.dim() != 2 || starts.dim() != 1)
    refuse("q_starts is [B + 1], kv_lens is [B], block_table [B, columns]");
  const int64_t B = table.size(0), cols = table.size(1);
  if (lens.size(0) != B || starts.size(0) != B + 1)
    refuse("for ", B, " sequences of the table: kv_lens ", shape(lens),
           ", q_starts ", shape(starts));
  for (const Tensor* x : {&starts, &lens, &table})
    if (x->scalar_type() != at::kInt)
      refuse("q_starts, kv_lens and block_table are int32");
  if (!starts.is_contiguous() || !lens.is_contiguous() ||
      (cols > 1 && table.stride(1) != 1))
    refuse("q_starts, kv_lens and the table's rows have no gaps");
  if (cols > (1LL << 30) >> p.page_log2)
    refuse(cols, " pages of ", 1 << p.page_log2, " tokens: a sequence has at "
           "most 2**30");
  const int64_t G = Hq / Hk, most = 1LL << 31;
  if (Hq > 32768 || T >= most || B >= most || T * G + 128 * B >= most ||
      (T * G / 16 + B) * Hk >= most)
    refuse(T, " tokens of ", Hq, " heads: too many for a launch");
  Plan plan{0, 4, 0, 1};
  if (T && B) {
    plan = plan_of(T, B, G, Hk, D, cols << p.page_log2, p.quantized);
    // shared, an item has at least 5 of the line's 2^30 units, and one to spare
    const int64_t items = (T * G / (plan.workers ? 16 : 128) + B) * Hk;
    if (plan.join ? items > (1LL << 30) / 6
                  : items * plan.splits > LAUNCH - 8)
      refuse(B, " sequences, ", T, " tokens of ", Hq, " heads: too many for a "
             "launch");
  }
  if (std::isnan(scale)) scale = 1.0 / std::sqrt((double)D);
  no_grad({&q, &out, &p.k, &p.v});
  if (out.defined()) {
    if (out.sizes() != q.sizes() || out.scalar_type() != q.scalar_type() ||
        !out.is_contiguous() || out.device() != q.device() || !aligned(out))
      refuse("out has q's shape, type and device, without gaps");
    for (const Tensor* x :
         {&p.k, &p.v, &p.k_scale, &p.v_scale, &starts, &lens, &table})
      if (overlap(out, *x))
        refuse("out shares memory with the cache, the starts, the lengths or "
               "the table");
  }
  on_gpu(p, {&q, &starts, &lens, &table});
  if (!out.defined())
    out = fresh(at::empty({T, Hq, D}, q.options().requires_grad(false)));
  if (T == 0 || B == 0) return out;
  const c10::DeviceGuard guard(p.device);
  // several workgroups may read a row that one of them answers
  q = overlap(out, q) ? fresh(q.clone(at::MemoryFormat::Contiguous))
                      : rows_of(q);
  Tensor parts;
  if (plan.join || plan.splits > 1) {
    // its own for every call: two captured graphs never share it
    const int64_t rows = plan.workers
                             ? 2 * plan.workers * 16
                             : (T * G / 128 + B) * Hk * plan.splits * 128;
    parts = fresh(at::empty({rows * (D + 2)}, q.options().dtype(at::kFloat)
                                                  .requires_grad(false)));
  }
  launched("tf_paged_attention",
           tf_paged_attention(
               ptr(q), ptr(p.k), ptr(p.v), ptr(p.k_scale), ptr(p.v_scale),
               ptr(starts), ptr(lens), ptr(table), ptr(out), ptr(parts),
               q.stride(0), q.stride(1), table.stride(0), (int)cols, (int)T,
               (int)B, (int)Hq, (int)Hk, (int)p.pages, p.page_log2, (int)D,
               (float)scale, causal, q.scalar_type() == at::kHalf,
               (int)plan.workers, (int)plan.waves, (int)plan.join, (int)plan.splits,
               stream_of(p)));
  changed(out);
  return out;
}

// ---- from and to Python --------------------------------------------------------

template <typename F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (const std::invalid_argument& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const c10::OutOfMemoryError& e) {
    PyObject* torch = PyImport_ImportModule("torch");
    PyObject* type =
        torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
    PyErr_SetString(type ? type : PyExc_RuntimeError,
                    e.what_without_backtrace());
    Py_XDECREF(type);
    Py_XDECREF(torch);
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

void count(Py_ssize_t got, Py_ssize_t want) {
  if (got != want) refuse(want, " arguments are wanted: got ", got);
}

int64_t int_of(PyObject* o, const char* name) {
  const long long x = PyLong_AsLongLong(o);
  if (x == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(name, " is a whole number");
  }
  return x;
}

PyObject* py_pools(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    count(n, 4);
    Pools p;
    p.k = tensor_of(a[0], "k");
    p.v = tensor_of(a[1], "v");
    if (a[2] != Py_None) p.k_scale = tensor_of(a[2], "k_scale");
    if (a[3] != Py_None) p.v_scale = tensor_of(a[3], "v_scale");
    check_pools(p);
    auto* o = reinterpret_cast<PoolsObject*>(
        pools_type->tp_alloc(pools_type, 0));
    if (!o) return nullptr;
    new (&o->p) Pools(std::move(p));
    return reinterpret_cast<PyObject*>(o);
  });
}

void pools_dealloc(PyObject* o) {
  PyTypeObject* type = Py_TYPE(o);
  reinterpret_cast<PoolsObject*>(o)->p.~Pools();
  type->tp_free(o);
  Py_DECREF(type);
}

PyObject* py_kv_write(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    count(n, 4);
    kv_write(pools_of(a[0]), tensor_of(a[1], "k"), tensor_of(a[2], "v"),
             tensor_of(a[3], "slots"));
    Py_RETURN_NONE;
  });
}

PyObject* py_rope_kv_write(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    count(n, 9);
    return THPVariable_Wrap(rope_kv_write(
        pools_of(a[0]), tensor_of(a[1], "q_in"), tensor_of(a[2], "k_in"),
        tensor_of(a[3], "v_in"), tensor_of(a[4], "cos"),
        tensor_of(a[5], "sin"), tensor_of(a[6], "pos"),
        tensor_of(a[7], "slots"), int_of(a[8], "heads")));
  });
}

PyObject* py_kv_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    count(n, 3);
    const Pools& p = pools_of(a[0]);
    at::ScalarType t = p.quantized ? at::kBFloat16 : p.dtype;
    if (a[2] != Py_None) {
      if (!THPDtype_Check(a[2])) refuse("dtype is a torch.dtype");
      t = reinterpret_cast<THPDtype*>(a[2])->scalar_type;
    }
    auto kv = kv_read(p, tensor_of(a[1], "slots"), t);
    PyObject* k = THPVariable_Wrap(kv.first);
    PyObject* v = THPVariable_Wrap(kv.second);
    PyObject* r = k && v ? PyTuple_Pack(2, k, v) : nullptr;
    Py_XDECREF(k);
    Py_XDECREF(v);
    return r;
  });
}

PyObject* py_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    count(n, 8);
    double scale = std::nan("");
    if (a[5] != Py_None) {
      scale = PyFloat_AsDouble(a[5]);
      if (PyErr_Occurred()) return nullptr;
      // the kernels' exponentials are of base 2
      if (!std::isfinite((float)scale * 1.4426950408889634f))
        refuse("scale is a finite number, and times log2(e): got ", scale);
    }
    const int causal = PyObject_IsTrue(a[6]);
    if (causal < 0) return nullptr;
    Tensor out;
    if (a[7] != Py_None) out = tensor_of(a[7], "out");
    return THPVariable_Wrap(attention(
        pools_of(a[0]), tensor_of(a[1], "q"), tensor_of(a[2], "q_starts"),
        tensor_of(a[3], "kv_lens"), tensor_of(a[4], "block_table"), scale,
        causal, out));
  });
}

// sizes of a batch: T, B, G, Hk, D and the table's keys
std::array<int64_t, 6> sizes_of(PyObject* const* a) {
  std::array<int64_t, 6> x;
  for (int i = 0; i < 6; ++i) {
    x[i] = int_of(a[i], "a size");
    if (x[i] < (i < 5) || x[i] > (i < 5 ? 1LL << 18 : 1LL << 30))
      refuse("no plan for a size of ", x[i]);
  }
  return x;
}

// of a 16-bit cache: workers, join, splits
PyObject* py_plan(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    count(n, 6);
    const auto x = sizes_of(a);
    const Plan p = plan_of(x[0], x[1], x[2], x[3], x[4], x[5], false);
    return Py_BuildValue("LLL", (long long)p.workers, (long long)p.join,
                         (long long)p.splits);
  });
}

// of either cache: workers, waves, join, splits
PyObject* py_dispatch(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    count(n, 7);
    const auto x = sizes_of(a);
    const int quantized = PyObject_IsTrue(a[6]);
    if (quantized < 0) return nullptr;
    const Plan p = plan_of(x[0], x[1], x[2], x[3], x[4], x[5], quantized);
    return Py_BuildValue("LLLL", (long long)p.workers, (long long)p.waves,
                         (long long)p.join, (long long)p.splits);
  });
}

#define TF_FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f))
PyMethodDef methods[] = {
    {"pools", TF_FAST(py_pools), METH_FASTCALL, nullptr},
    {"kv_write", TF_FAST(py_kv_write), METH_FASTCALL, nullptr},
    {"rope_kv_write", TF_FAST(py_rope_kv_write), METH_FASTCALL, nullptr},
    {"kv_read", TF_FAST(py_kv_read), METH_FASTCALL, nullptr},
    {"attention", TF_FAST(py_attention), METH_FASTCALL, nullptr},
    {"plan", TF_FAST(py_plan), METH_FASTCALL, nullptr},
    {"dispatch", TF_FAST(py_dispatch), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "tf_paged", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

PyType_Slot pools_slots[] = {{Py_tp_dealloc, (void*)pools_dealloc},
                             {0, nullptr}};
PyType_Spec pools_spec = {"tf_paged.Pools", sizeof(PoolsObject), 0,
                          Py_TPFLAGS_DEFAULT | Py_TPFLAGS_DISALLOW_INSTANTIATION,
                          pools_slots};

}  // namespace

PyMODINIT_FUNC PyInit_tf_paged() {
  PyObject* m = PyModule_Create(&module);
  if (!m) return nullptr;
  pools_type = reinterpret_cast<PyTypeObject*>(PyType_FromSpec(&pools_spec));
  if (!pools_type) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
