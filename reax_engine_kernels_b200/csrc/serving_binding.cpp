// Python binding of libreax_decode for torch tensors (module _serving, used by kernels.py): argument checks, output and
// workspace allocation and the C call.  A serving step is a run of calls of a few microseconds each, and the same checks in
// Python with a ctypes call cost more than that: a 64-token kv_write took 22.2 us a call, with this binding 4.1 us.
//
// Refused arguments raise ValueError before any device is touched; the functions return the C entry point's code.
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include "reax_abi.h"

namespace {
using at::Tensor;
using OptTensor = std::optional<Tensor>;
namespace py = pybind11;

[[noreturn]] void refuse(const std::string& what) { throw py::value_error(what); }

std::string shape_of(at::IntArrayRef s) {
  std::string r = "(";
  for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + (s[i] < 0 ? std::string("*") : std::to_string(s[i]));
  return r + ")";
}

// `t` has that dtype, device and shape (a size of -1: any)
void want(const char* name, const Tensor& t, at::ScalarType dtype, at::IntArrayRef shape, at::Device device) {
  if (t.scalar_type() != dtype) {
    const char* wanted = dtype == at::kBFloat16 ? "bfloat16" : dtype == at::kFloat ? "float32" : dtype == at::kInt ? "int32"
                         : dtype == at::kLong   ? "int64"    : dtype == at::kByte ? "uint8"   : dtype == at::kBool ? "bool"
                                                                                                                   : "float8_e4m3fn";
    refuse(std::string(name) + " must be torch." + wanted + ", got " + std::string(at::toString(t.scalar_type())));
  }
  if (t.device() != device) refuse(std::string(name) + " is on " + t.device().str() + ", the operands on " + device.str());
  bool same = t.dim() == (int64_t)shape.size();
  for (size_t i = 0; same && i < shape.size(); ++i) same = shape[i] < 0 || shape[i] == t.size(i);
  if (!same) refuse(std::string(name) + " must have shape " + shape_of(shape) + ", got " + shape_of(t.sizes()));
}

void last_dense(const char* name, const Tensor& t) {
  if (t.dim() > 0 && t.size(-1) > 1 && t.stride(-1) != 1)
    refuse(std::string(name) + ": the last dimension must be contiguous (stride " + std::to_string(t.stride(-1)) + ")");
}
// an output that a view repeats would be written by several CTAs at once
void not_expanded(const char* name, const Tensor& t) {
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.size(i) > 1 && t.stride(i) == 0) refuse(std::string(name) + ": an output's elements must not overlap");
}
void dense(const char* name, const Tensor& t) {
  if (!t.is_contiguous()) refuse(std::string(name) + " must be contiguous");
}
void on_cuda(const Tensor& t) {
  if (!t.is_cuda()) refuse("all tensors must be CUDA tensors");
}
void head_dim(int64_t D) {
  if (D != 128 && D != 256) refuse("the head dimension must be 128 or 256, got " + std::to_string(D));
}
int to_int(const char* name, int64_t n) {
  if (n < 0 || n > 0x7fffffff) refuse(std::string(name) + " = " + std::to_string(n) + " is out of range");
  return (int)n;
}
// straight from the caching allocator, without the dispatcher's share of a microsecond
Tensor empty_on(at::IntArrayRef shape, at::ScalarType dtype, at::Device device) {
  return Tensor(at::detail::empty_cuda(shape, dtype, device, std::nullopt));
}
void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

struct Cache {
  const Tensor &k, &ke, &v, &ve;
};

int64_t check_cache(const Cache& c, int64_t H, int64_t D, at::Device dev, bool written = false) {
  want("cache.k", c.k, at::kFloat8_e4m3fn, {-1, H, -1, D}, dev);
  want("cache.v", c.v, at::kFloat8_e4m3fn, c.k.sizes(), dev);
  want("cache.ke", c.ke, at::kByte, c.k.sizes().slice(0, 3), dev);
  want("cache.ve", c.ve, at::kByte, c.k.sizes().slice(0, 3), dev);
  if (c.k.strides() != c.v.strides() || c.ke.strides() != c.ve.strides())
    refuse("cache.k and cache.v (and cache.ke and cache.ve) must have the same strides");
  const int64_t page = c.k.size(2);
  if (page <= 0 || page % 16) refuse("the page size must be a multiple of 16, got " + std::to_string(page));
  if (c.k.stride(3) != 1 || c.k.stride(2) != D || c.ke.stride(2) != 1)
    refuse("the rows of a page and head must be contiguous");
  if (written) not_expanded("cache", c.k), not_expanded("cache", c.ke);
  return page;
}

int64_t check_kv(const Tensor& k, const Tensor& v, const Cache& c, const Tensor& slots, bool written = false) {
  if (k.dim() != 3) refuse("k must be [T, H, D], got " + shape_of(k.sizes()));
  const int64_t T = k.size(0), H = k.size(1), D = k.size(2);
  const at::Device dev = k.device();
  want("k", k, at::kBFloat16, {T, H, D}, dev);
  want("v", v, at::kBFloat16, {T, H, D}, dev);
  want("slots", slots, at::kLong, {T}, dev);
  head_dim(D);
  last_dense("k", k);
  last_dense("v", v);
  dense("slots", slots);
  const int64_t page = check_cache(c, H, D, dev, written);
  on_cuda(k);
  return page;
}

int kv_write(const Tensor& k, const Tensor& v, const Tensor& ck, const Tensor& ke, const Tensor& cv, const Tensor& ve,
             const Tensor& slots) {
  const int64_t page = check_kv(k, v, {ck, ke, cv, ve}, slots, /*written=*/true);
  const c10::cuda::CUDAGuard guard(k.device());
  return reax_kv_write(k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), ck.data_ptr(), ke.data_ptr(),
                       cv.data_ptr(), ve.data_ptr(), ck.stride(0), ck.stride(1), ke.stride(0), ke.stride(1),
                       (const long long*)slots.data_ptr(), to_int("T", k.size(0)), to_int("H", k.size(1)), (int)k.size(2),
                       to_int("page", page), ck.size(0), stream_of(k));
}

std::tuple<int, Tensor, Tensor> kv_read(const Tensor& ck, const Tensor& ke, const Tensor& cv, const Tensor& ve,
                                        const Tensor& slots, const OptTensor& k_out, const OptTensor& v_out) {
  if (ck.dim() != 4 || slots.dim() != 1)
    refuse("cache.k must be [pages, H, page, D] and slots [T], got " + shape_of(ck.sizes()) + ", " + shape_of(slots.sizes()));
  if (!k_out || !v_out) on_cuda(slots);
  const auto make = [&](const OptTensor& t) {
    return t ? *t : empty_on({slots.size(0), ck.size(1), ck.size(3)}, at::kBFloat16, slots.device());
  };
  Tensor k = make(k_out), v = make(v_out);
  if (k.dim() == 3 && k.size(0) != slots.size(0)) refuse("k has another number of rows than slots");
  not_expanded("k", k);
  not_expanded("v", v);
  const int64_t page = check_kv(k, v, {ck, ke, cv, ve}, slots);
  const c10::cuda::CUDAGuard guard(k.device());
  const int rc = reax_kv_read(k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), ck.data_ptr(),
                              ke.data_ptr(), cv.data_ptr(), ve.data_ptr(), ck.stride(0), ck.stride(1), ke.stride(0), ke.stride(1),
                              (const long long*)slots.data_ptr(), to_int("T", k.size(0)), to_int("H", k.size(1)), (int)k.size(2),
                              to_int("page", page), ck.size(0), stream_of(k));
  return {rc, k, v};
}

std::tuple<int, Tensor> fmha_paged(const Tensor& q, const Tensor& ck, const Tensor& ke, const Tensor& cv, const Tensor& ve,
                                   const Tensor& table, double scale, const Tensor& qpos, int64_t G, const OptTensor& prefix,
                                   int64_t prefix_len, const OptTensor& out_) {
  if (q.dim() != 4) refuse("q must be [B, H, M, D], got " + shape_of(q.sizes()));
  const int64_t B = q.size(0), H = q.size(1), M = q.size(2), D = q.size(3);
  const at::Device dev = q.device();
  want("q", q, at::kBFloat16, {B, H, M, D}, dev);
  head_dim(D);
  const int64_t page = check_cache({ck, ke, cv, ve}, H, D, dev);
  want("table", table, at::kInt, {B, -1}, dev);
  want("qpos", qpos, at::kInt, {B, -1}, dev);
  if (G <= 0 || M % G || qpos.size(1) < M / G)
    refuse("G = " + std::to_string(G) + " must divide M = " + std::to_string(M) + ", and qpos needs M / G columns, got " +
           std::to_string(qpos.size(1)));
  if (!prefix) {
    if (prefix_len) refuse("prefix_len without a prefix");
  } else {
    want("prefix", *prefix, at::kInt, {-1}, dev);
    if (prefix_len < 0 || prefix_len > prefix->size(0) * page)
      refuse("prefix_len = " + std::to_string(prefix_len) + ", but the prefix has " + std::to_string(prefix->size(0)) +
             " pages of " + std::to_string(page));
    last_dense("prefix", *prefix);
  }
  if (out_) {
    want("out", *out_, at::kBFloat16, {B, H, M, D}, dev);
    last_dense("out", *out_);
    not_expanded("out", *out_);
  }
  last_dense("q", q);
  last_dense("table", table);
  last_dense("qpos", qpos);
  on_cuda(q);
  Tensor out = out_ ? *out_ : empty_on({B, H, M, D}, at::kBFloat16, dev);
  const c10::cuda::CUDAGuard guard(dev);
  const int b = to_int("B", B), h = to_int("H", H), m = to_int("M", M), d = (int)D, P = to_int("P", table.size(1)),
            pg = to_int("page", page), Lp = to_int("prefix_len", prefix_len);
  const int splits = reax_fmha_paged_splits(b, h, m, d, P, pg, Lp);
  if (splits < 0) return {splits, out};
  Tensor ws;
  if (splits > 1 && B && M) ws = empty_on({splits * B * H * M * (D + 1)}, at::kFloat, dev);
  const int rc = reax_fmha_paged(
      q.data_ptr(), q.stride(0), q.stride(1), q.stride(2), ck.data_ptr(), ke.data_ptr(), cv.data_ptr(), ve.data_ptr(), ck.stride(0),
      ck.stride(1), ke.stride(0), ke.stride(1), (const int*)table.data_ptr(), table.stride(0),
      prefix ? (const int*)prefix->data_ptr() : nullptr, Lp, (const int*)qpos.data_ptr(), to_int("G", G), qpos.stride(0), out.data_ptr(),
      out.stride(0), out.stride(1), out.stride(2), ws.defined() ? ws.data_ptr() : nullptr, (float)scale, b, h, m, d, P, pg, ck.size(0),
      stream_of(q));
  return {rc, out};
}

std::tuple<int, Tensor> delta_state(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta,
                                    const Tensor& cu, double scale, const Tensor& state, const OptTensor& slots,
                                    const OptTensor& fresh, const OptTensor& o_) {
  if (q.dim() != 3 || v.dim() != 3 || cu.dim() != 1 || cu.size(0) < 1)
    refuse("q, k, v must be [T, heads, 128] and cu [N + 1]");
  const int64_t T = q.size(0), H = q.size(1), HV = v.size(1), N = cu.size(0) - 1;
  const at::Device dev = q.device();
  if (H <= 0 || HV <= 0 || HV % H)
    refuse("the value heads (" + std::to_string(HV) + ") must be a multiple of the key heads (" + std::to_string(H) + ")");
  want("q", q, at::kBFloat16, {T, H, 128}, dev);
  want("k", k, at::kBFloat16, {T, H, 128}, dev);
  want("v", v, at::kBFloat16, {T, HV, 128}, dev);
  want("beta", beta, at::kBFloat16, {T, HV}, dev);
  want("g", g, at::kFloat, {T, HV}, dev);
  want("cu", cu, at::kLong, {N + 1}, dev);
  want("state", state, at::kFloat, {-1, HV, 128, 128}, dev);
  const int64_t S = state.size(0);
  if (slots) {
    want("slots", *slots, at::kInt, {N}, dev);
    dense("slots", *slots);
  } else if (N > S) {
    refuse(std::to_string(N) + " sequences, but the state has " + std::to_string(S) + " slots");
  }
  if (S > 1 && state.stride(0) < HV * 128 * 128) refuse("the state's slots overlap");
  if (S > 0 && !(state.stride(3) == 1 && state.stride(2) == 128 && (HV == 1 || state.stride(1) == 128 * 128)))
    refuse("state must be contiguous within a slot");
  if (fresh) {
    want("fresh", *fresh, at::kBool, {N}, dev);
    dense("fresh", *fresh);
  }
  if (o_) {
    want("o", *o_, at::kBFloat16, {T, HV, 128}, dev);
    dense("o", *o_);
  }
  dense("q", q);
  dense("k", k);
  dense("v", v);
  dense("beta", beta);
  dense("g", g);
  dense("cu", cu);
  on_cuda(q);
  Tensor o = o_ ? *o_ : empty_on({T, HV, 128}, at::kBFloat16, dev);
  const c10::cuda::CUDAGuard guard(dev);
  const int rc = reax_delta_state(q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(), (const long long*)cu.data_ptr(),
                                  state.data_ptr(), state.stride(0), slots ? (const int*)slots->data_ptr() : nullptr,
                                  fresh ? fresh->data_ptr() : nullptr, o.data_ptr(), (float)scale, T, S, to_int("N", N),
                                  to_int("H", H), to_int("HV", HV), stream_of(q));
  return {rc, o};
}
}  // namespace

PYBIND11_MODULE(_serving, m) {
  m.def("kv_write", &kv_write);
  m.def("kv_read", &kv_read);
  m.def("fmha_paged", &fmha_paged);
  m.def("delta_state", &delta_state);
}
