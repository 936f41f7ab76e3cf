// Host side of the 8-bit operators, in native code: checks, results, workspaces and the launch of a call.
//
// Small calls wait for the host: driven from Python, the norm of 8 rows took 26 us for a kernel of 3, most of it checks,
// views of the results and argument objects.  A function here takes a call whose tensors the kernels read as they lie, on
// whatever device they are; for anything else it returns nothing before it allocates or launches anything, and the caller
// says what is wrong or brings the tensors into shape and asks again.
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <pybind11/stl.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <optional>
#include <stdexcept>
#include <string>
#include <tuple>
#include <vector>

#include "entries.h"

namespace py = pybind11;
using at::Tensor;

namespace {

constexpr long kBlock = 128, kStateBlock = 256, kNormWidth = 16384;
constexpr size_t kStatusWords = 4;
constexpr long kMaxRows = 0x7fffffff, kMaxBlocked = kMaxRows - (kBlock - 1);   // the kernels count in ints, along a row in whole blocks

void check(int rc, const char* what) {
  if (rc != 0) throw std::runtime_error(std::string(what) + " failed with code " + std::to_string(rc));
}
void* stream() { return c10::cuda::getCurrentCUDAStream().stream(); }   // of the current device

int value_type(at::ScalarType t) { return t == at::kFloat ? 0 : t == at::kHalf ? 1 : t == at::kBFloat16 ? 2 : -1; }
int code_type(at::ScalarType t) { return t == at::kFloat8_e4m3fn ? 0 : t == at::kFloat8_e5m2 ? 1 : -1; }
long up(long n, long to) { return (n + to - 1) / to * to; }
long blocks(long n, long size) { return (n + size - 1) / size; }

bool dense(const Tensor& t) { return t.is_cuda() && t.layout() == at::kStrided && !t.is_neg() && !t.is_conj(); }
// a matrix whose rows are contiguous, of any pitch that leaves them apart; one without values may have any strides
bool rows_of(const Tensor& t) {
  return dense(t) && t.dim() == 2 && (t.numel() == 0 || ((t.size(1) <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1))));
}
long pitch(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
bool on_16(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0; }

// The GIL is given up for a call, which may wait for room in the stream's queue; pybind's own guard takes 1.5 us.
struct WithoutGil {
  PyThreadState* state = PyEval_SaveThread();
  ~WithoutGil() { PyEval_RestoreThread(state); }
};

// What is written behind autograd's back: a graph that saved the tensor has to find that it changed.  (Raises for an inference
// tensor outside inference mode, so before anything is launched.)
void changes(const Tensor& t) { t.unsafeGetTensorImpl()->bump_version(); }

// A matrix of its own memory, straight from the allocator (a call through the dispatcher takes 0.8 us, and as much again for a
// view of the result)
Tensor empty_matrix(long rows, long cols, long pitch, at::ScalarType type, const Tensor& like, bool by_cols = false) {
  Tensor t = at::detail::empty_cuda({rows * pitch}, type, like.device(), std::nullopt);
  const int64_t sizes[2] = {by_cols ? cols : rows, by_cols ? rows : cols}, strides[2] = {by_cols ? 1 : pitch, by_cols ? pitch : 1};
  t.unsafeGetTensorImpl()->set_sizes_and_strides(at::IntArrayRef(sizes, 2), at::IntArrayRef(strides, 2));
  return t;
}
Tensor empty_vector(long n, at::ScalarType type, const Tensor& like) { return at::detail::empty_cuda({n}, type, like.device(), std::nullopt); }
// codes whose rows begin on 16 bytes
Tensor empty_codes(long rows, long cols, at::ScalarType type, const Tensor& like) { return empty_matrix(rows, cols, up(cols, 16), type, like); }
// scales of neighbouring blocks along the contraction lie next to one another: those of 128 x 1 blocks by columns
Tensor empty_scales(long rows, long cols, long br, long bc, const Tensor& like) {
  const long nr = blocks(rows, br), nc = blocks(cols, bc);
  return bc == 1 ? empty_matrix(nc, nr, up(nr, 4), at::kFloat8_e8m0fnu, like, true) : empty_matrix(nr, nc, up(nc, 4), at::kFloat8_e8m0fnu, like);
}

using Tensors = std::optional<std::vector<Tensor>>;

// codes and scales, of ways 1 and 2 in this order; ways as dcpk_fp8_quantize has them
Tensors quantize8(const Tensor& x, int ways, bool e5m2) {
  if (!rows_of(x) || value_type(x.scalar_type()) < 0 || x.size(0) > kMaxRows || x.size(1) > kMaxBlocked) return std::nullopt;
  c10::DeviceGuard guard(x.device());
  const long rows = x.size(0), cols = x.size(1);
  const at::ScalarType type = e5m2 ? at::kFloat8_e5m2 : at::kFloat8_e4m3fn;
  std::vector<Tensor> out;
  void* p[4] = {nullptr, nullptr, nullptr, nullptr};
  long scale_pitch[2] = {0, 0};
  for (int w : {0, 1}) {
    if (!(w ? ways & 2 : ways & 5)) continue;
    const long br = w || ways == 4 ? kBlock : 1, bc = w ? 1 : kBlock;
    out.push_back(empty_codes(rows, cols, type, x));
    out.push_back(empty_scales(rows, cols, br, bc, x));
    p[2 * w] = out[out.size() - 2].data_ptr();
    p[2 * w + 1] = out.back().data_ptr();
    scale_pitch[w] = up(w ? blocks(rows, kBlock) : blocks(cols, kBlock), 4);
  }
  check(dcpk_fp8_quantize(value_type(x.scalar_type()), e5m2, ways, x.const_data_ptr(), pitch(x), p[0], up(cols, 16), p[1], scale_pitch[0], p[2],
                          up(cols, 16), p[3], scale_pitch[1], rows, int(cols), stream()),
        "fp8_quantize");
  return out;
}

bool like(const Tensor& t, const Tensor& x) {
  return rows_of(t) && t.sizes() == x.sizes() && t.scalar_type() == x.scalar_type() && t.device() == x.device();
}
bool channels(const Tensor& w, const Tensor& x) {
  return dense(w) && w.dim() == 1 && w.size(0) == x.size(1) && w.is_contiguous() && w.scalar_type() == x.scalar_type() && w.device() == x.device();
}
bool norm_input(const Tensor& x) {
  return rows_of(x) && value_type(x.scalar_type()) >= 0 && x.size(1) >= 1 && x.size(1) <= kNormWidth;
}

// codes, scales, h, rstd
Tensors norm8(const Tensor& x, const Tensor& w, double eps, const std::optional<Tensor>& residual, bool e5m2) {
  if (!norm_input(x) || !channels(w, x) || (residual && !like(*residual, x))) return std::nullopt;
  c10::DeviceGuard guard(x.device());
  const long rows = x.size(0), width = x.size(1);
  Tensor codes = empty_codes(rows, width, e5m2 ? at::kFloat8_e5m2 : at::kFloat8_e4m3fn, x);
  Tensor scales = empty_scales(rows, width, 1, kBlock, x);
  Tensor h = residual ? empty_matrix(rows, width, width, x.scalar_type(), x) : x;
  Tensor rstd = empty_vector(rows, at::kFloat, x);
  check(dcpk_fp8_norm(value_type(x.scalar_type()), e5m2, x.const_data_ptr(), pitch(x), residual ? residual->const_data_ptr() : nullptr,
                      residual ? pitch(*residual) : 0, w.const_data_ptr(), residual ? h.data_ptr() : nullptr, codes.data_ptr(), up(width, 16),
                      scales.data_ptr(), up(blocks(width, kBlock), 4), rstd.data_ptr<float>(), rows, int(width), float(eps), stream()),
        "fp8_norm");
  return std::vector<Tensor>{codes, scales, h, rstd};
}

// dx, dw
Tensors norm8_bwd(const Tensor& h, const Tensor& w, const Tensor& rstd, const Tensor& dy, const std::optional<Tensor>& add, const Tensor& status) {
  if (!norm_input(h) || !channels(w, h) || !like(dy, h) || (add && !like(*add, h)) || !dense(rstd) || rstd.dim() != 1 ||
      rstd.size(0) != h.size(0) || !rstd.is_contiguous() || rstd.scalar_type() != at::kFloat || rstd.device() != h.device())
    return std::nullopt;
  c10::DeviceGuard guard(h.device());
  const long rows = h.size(0), width = h.size(1);
  Tensor dx = empty_matrix(rows, width, width, h.scalar_type(), h), dw = empty_vector(width, at::kFloat, h);
  const Tensor part = empty_vector(dcpk_fp8_norm_bwd_parts(value_type(h.scalar_type()), rows, int(width), add.has_value()) * width, at::kFloat, h);
  check(dcpk_fp8_norm_bwd(value_type(h.scalar_type()), h.const_data_ptr(), pitch(h), w.const_data_ptr(), rstd.const_data_ptr<float>(),
                          dy.const_data_ptr(), pitch(dy), add ? add->const_data_ptr() : nullptr, add ? pitch(*add) : 0, dx.data_ptr(),
                          dw.data_ptr<float>(), part.data_ptr<float>(), rows, int(width), status.data_ptr<int>(), stream()),
        "fp8_norm_bwd");
  return std::vector<Tensor>{dx, dw};
}

// an operand; k_dim: the dimension that is added up.  The product reads it where it is if its rows begin on 16 bytes
bool operand(const Tensor& codes, const Tensor& scales, long br, long bc, int k_dim, DcpkFp8Operand* o) {
  const long b[2] = {br, bc};
  if (!rows_of(codes) || code_type(codes.scalar_type()) < 0 || !dense(scales) || scales.dim() != 2 ||
      scales.scalar_type() != at::kFloat8_e8m0fnu || scales.device() != codes.device())
    return false;
  for (int d : {0, 1})
    if ((b[d] != 1 && b[d] != kBlock) || scales.size(d) != blocks(codes.size(d), b[d])) return false;
  if (b[k_dim] != kBlock || codes.size(k_dim) > kMaxBlocked || codes.size(1 - k_dim) > kMaxRows) return false;
  *o = {codes.const_data_ptr(), codes.size(0) > 1 ? codes.stride(0) : up(codes.size(1), 16), scales.const_data_ptr(), scales.stride(1 - k_dim), scales.stride(k_dim), int(codes.size(1 - k_dim)),
        k_dim == 0, b[1 - k_dim] == kBlock ? 7 : 0, code_type(codes.scalar_type())};
  return true;
}

// Two matrices of one shape and type are one, or share no element: a thread reads what it adds to just before it writes there,
// but not before others write.
bool one_or_apart(const Tensor& a, const Tensor& b) {
  const long m = a.size(0), n = a.size(1), size = long(a.element_size()), pa = pitch(a), pb = pitch(b);
  const long d = long(reinterpret_cast<intptr_t>(b.const_data_ptr()) - reinterpret_cast<intptr_t>(a.const_data_ptr()));
  if ((d == 0 && pa == pb) || d >= ((m - 1) * pa + n) * size || -d >= ((m - 1) * pb + n) * size) return true;
  const long at = (d % (pa * size) + pa * size) % (pa * size);   // of b's rows within a's pitch
  return pa == pb && at >= n * size && at <= (pa - n) * size;    // columns beside one another
}

std::optional<Tensor> matmul8(const Tensor& a, const Tensor& a_scales, std::pair<long, long> a_block, const Tensor& b, const Tensor& b_scales,
                              std::pair<long, long> b_block, bool trans_a, bool trans_b, int out_type, const std::optional<Tensor>& add,
                              const std::optional<Tensor>& out, int form, const Tensor& status) {
  DcpkFp8Operand q, p;
  const int ka = trans_a ? 0 : 1, kb = trans_b ? 1 : 0;
  if (out_type < 0 || out_type > 2 || !operand(a, a_scales, a_block.first, a_block.second, ka, &q) ||
      !operand(b, b_scales, b_block.first, b_block.second, kb, &p) || a.size(ka) != b.size(kb) || a.size(ka) < 1 || q.rows < 1 || p.rows < 1 ||
      a.device() != b.device())
    return std::nullopt;
  const at::ScalarType type = out_type == 0 ? at::kFloat : out_type == 1 ? at::kHalf : at::kBFloat16;
  for (const auto* t : {&add, &out})
    if (*t && (!rows_of(**t) || (*t)->size(0) != q.rows || (*t)->size(1) != p.rows || (*t)->scalar_type() != type || (*t)->device() != a.device() ||
               ((*t)->requires_grad() && at::GradMode::is_enabled())))
      return std::nullopt;
  if (add && out && !one_or_apart(*add, *out)) return std::nullopt;
  c10::DeviceGuard guard(a.device());
  if (out) changes(*out);
  Tensor result = out ? *out : empty_matrix(q.rows, p.rows, p.rows, type, a);
  Tensor laid[2];   // operands whose rows do not begin on 16 bytes
  const Tensor* codes[2] = {&a, &b};
  DcpkFp8Operand* operands[2] = {&q, &p};
  struct { const void* from; long pitch; void* to; int rows, width; } jobs[2] = {};
  int n_jobs = 0;
  for (int i : {0, 1}) {
    DcpkFp8Operand& o = *operands[i];
    if (o.pitch % 16 == 0 && on_16(*codes[i])) continue;
    const int rows = int(codes[i]->size(0)), width = int(codes[i]->size(1));
    laid[i] = empty_codes(rows, width, codes[i]->scalar_type(), a);
    jobs[n_jobs++] = {o.codes, o.pitch, laid[i].data_ptr(), rows, width};
    o.codes = laid[i].const_data_ptr();
    o.pitch = up(width, 16);
  }
  if (n_jobs)
    check(dcpk_fp8_align(jobs[0].from, jobs[0].pitch, jobs[0].to, jobs[0].rows, jobs[0].width, jobs[1].from, jobs[1].pitch, jobs[1].to, jobs[1].rows,
                         jobs[1].width, stream()),
          "fp8_align");
  const long bytes = dcpk_fp8_gemm_work(q.rows, p.rows, q.rows_inner, int(a.size(ka)), form);
  Tensor work;   // of this call alone
  if (bytes > 0) work = empty_vector(bytes, at::kByte, a);
  check(dcpk_fp8_gemm(&q, &p, int(a.size(ka)), result.data_ptr(), pitch(result), add ? add->const_data_ptr() : nullptr, add ? pitch(*add) : 0,
                      out_type, form, bytes > 0 ? work.data_ptr() : nullptr, status.data_ptr<int>(), stream()),
        "fp8_gemm");
  return result;
}

using List = std::vector<Tensor>;

// Whether the call was taken, and the gradients' norm where it is limited.
std::tuple<bool, std::optional<Tensor>> adamw8(const List& params, const List& grads, const std::optional<List>& masters, const List& m,
                                               const List& v, const Tensor& step, double lr, double beta1, double beta2, double eps,
                                               double wd, double grad_scale, double clip, const std::optional<List>& m_scales,
                                               const std::optional<List>& v_scales, unsigned seed, const std::optional<Tensor>& factor,
                                               const List& status) {
  const std::tuple<bool, std::optional<Tensor>> no{false, std::nullopt};
  const size_t n = params.size();
  if (n == 0 || n > 0x7fffffff || grads.size() != n || m.size() != n || v.size() != n || (masters && masters->size() != n) ||
      bool(m_scales) != bool(v_scales) || (m_scales && (m_scales->size() != n || v_scales->size() != n)) || status.size() > kStatusWords || !(clip >= 0) ||
      (clip > 0 && factor) || !(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1))
    return no;
  const auto device = params[0].device();
  const int ptype = value_type(params[0].scalar_type()), gtype = value_type(grads[0].scalar_type());
  const auto state = m_scales ? at::kFloat8_e4m3fn : at::kFloat;
  const auto plain = [&](const Tensor& t, at::ScalarType type, long size) {
    return dense(t) && t.device() == device && t.scalar_type() == type && t.numel() == size && t.is_contiguous();
  };
  if (ptype < 0 || gtype < 0 || (!masters && ptype != 0) || !plain(step, at::kLong, 1) || (factor && !plain(*factor, at::kFloat, 1))) return no;
  for (const Tensor& s : status)
    if (!dense(s) || s.scalar_type() != at::kInt || s.numel() < 1 || s.device() != device) return no;
  std::vector<void*> p(n), w(n), pm(n), pv(n), sm(n), sv(n);
  std::vector<const void*> g(n);
  std::vector<long> sizes(n);
  for (size_t i = 0; i < n; ++i) {
    const long size = params[i].numel(), scales = blocks(size, kStateBlock);
    if (!plain(params[i], params[0].scalar_type(), size) || !plain(grads[i], grads[0].scalar_type(), size) || !plain(m[i], state, size) ||
        !plain(v[i], state, size) || (masters && !plain((*masters)[i], at::kFloat, size)) ||
        (m_scales && (!plain((*m_scales)[i], at::kFloat8_e8m0fnu, scales) || !plain((*v_scales)[i], at::kFloat8_e8m0fnu, scales))))
      return no;
    sizes[i] = size;
    p[i] = params[i].data_ptr(), g[i] = grads[i].const_data_ptr(), pm[i] = m[i].data_ptr(), pv[i] = v[i].data_ptr();
    if (masters) w[i] = (*masters)[i].data_ptr();
    if (m_scales) sm[i] = (*m_scales)[i].data_ptr(), sv[i] = (*v_scales)[i].data_ptr();
  }
  // memory given twice would be written by two blocks at once
  std::vector<std::pair<uintptr_t, uintptr_t>> written;
  written.reserve(6 * n + 1);
  const auto writes = [&](const std::vector<void*>& list, size_t i, long bytes) {
    const uintptr_t start = reinterpret_cast<uintptr_t>(list[i]);
    if (start && bytes > 0) written.emplace_back(start, start + uintptr_t(bytes));
  };
  const long of_param = long(params[0].element_size()), of_state = m_scales ? 1 : 4;
  for (size_t i = 0; i < n; ++i) {
    writes(p, i, sizes[i] * of_param), writes(w, i, sizes[i] * 4);
    writes(pm, i, sizes[i] * of_state), writes(pv, i, sizes[i] * of_state);
    writes(sm, i, blocks(sizes[i], kStateBlock)), writes(sv, i, blocks(sizes[i], kStateBlock));
  }
  written.emplace_back(reinterpret_cast<uintptr_t>(step.const_data_ptr()), reinterpret_cast<uintptr_t>(step.const_data_ptr()) + 8);
  std::sort(written.begin(), written.end());
  for (size_t i = 1; i < written.size(); ++i)
    if (written[i - 1].second > written[i].first) return no;
  // and what is read would change under the readers
  const auto apart = [&](const void* from, long bytes) {
    const uintptr_t start = reinterpret_cast<uintptr_t>(from);
    const auto next = std::lower_bound(written.begin(), written.end(), std::make_pair(start, uintptr_t(0)));
    return bytes <= 0 || ((next == written.end() || next->first >= start + uintptr_t(bytes)) && (next == written.begin() || next[-1].second <= start));
  };
  const long of_grad = long(grads[0].element_size());
  for (size_t i = 0; i < n; ++i)
    if (!apart(g[i], sizes[i] * of_grad)) return no;
  if (factor && !apart(factor->const_data_ptr(), 4)) return no;
  for (const Tensor& s : status)
    if (!apart(s.const_data_ptr(), 4)) return no;
  for (const List* list : {&params, &m, &v})
    for (const Tensor& t : *list) changes(t);
  for (const auto* list : {&masters, &m_scales, &v_scales})
    if (*list)
      for (const Tensor& t : **list) changes(t);
  changes(step);
  c10::DeviceGuard guard(device);
  Tensor work = empty_vector(dcpk_adamw_multi_work(int(n)), at::kDouble, step);
  std::optional<Tensor> norm;
  if (clip > 0) norm = empty_vector(1, at::kFloat, step);
  const int* words[kStatusWords] = {};
  for (size_t i = 0; i < status.size(); ++i) words[i] = status[i].const_data_ptr<int>();
  check(dcpk_adamw_multi(int(n), p.data(), g.data(), masters ? w.data() : nullptr, pm.data(), pv.data(), m_scales ? sm.data() : nullptr,
                         m_scales ? sv.data() : nullptr, sizes.data(), ptype, gtype, step.data_ptr<int64_t>(), float(lr), beta1, beta2,
                         float(eps), float(wd), float(grad_scale), float(clip), factor ? factor->const_data_ptr<float>() : nullptr, seed,
                         norm ? norm->data_ptr<float>() : nullptr, words, int(status.size()), work.data_ptr<double>(), stream()),
        "adamw_multi");
  return {true, norm};
}

}  // namespace

void bind_ops8(py::module_& m) {
  const py::call_guard<WithoutGil> free_gil;
  m.def("quantize8", &quantize8, free_gil);
  m.def("norm8", &norm8, free_gil);
  m.def("norm8_bwd", &norm8_bwd, free_gil);
  m.def("matmul8", &matmul8, free_gil);
  m.def("adamw8", &adamw8, free_gil);
}
