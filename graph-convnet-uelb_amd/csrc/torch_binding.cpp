// Native side of the Python entry points whose calls are shorter than what it costs to prepare them in Python: the AdamW step
// and the gradient norm on lists of tensors (a table of addresses per list) and the rules on logits with their gradient.  It
// checks the arguments, allocates results and calls the C ABI, whose functions the Python side hands over once (bind), so
// that this file needs no GPU toolchain and works with whichever build of the library is loaded.
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <cmath>
#include <cstddef>
#include <cstring>
#include <memory>
#include <optional>
#include <sstream>
#include <string>
#include <utility>
#include <vector>

#include "../../include/gcn_uelb_hip.h"

namespace py = pybind11;

namespace {

struct Api {
    decltype(&gcn_last_error) last_error = nullptr;
    decltype(&gcn_adamw_step) adamw_step = nullptr;
    decltype(&gcn_adamw_hyper_bytes) adamw_hyper_bytes = nullptr;
    decltype(&gcn_grad_norm_ws_bytes) grad_norm_ws_bytes = nullptr;
    decltype(&gcn_grad_norm) grad_norm = nullptr;
    decltype(&gcn_logits_process) logits_process = nullptr;
    decltype(&gcn_logits_bwd_ws_bytes) logits_bwd_ws_bytes = nullptr;
    decltype(&gcn_logits_process_bwd) logits_process_bwd = nullptr;
};
Api api;
PyObject* hip_error = nullptr;       // GcnHipError

template <typename... A>
std::string text(const A&... a) {
    std::ostringstream s;
    (s << ... << a);
    return s.str();
}
template <typename... A>
[[noreturn]] void value_error(const A&... a) { throw py::value_error(text(a...)); }
template <typename... A>
[[noreturn]] void type_error(const A&... a) { throw py::type_error(text(a...)); }
template <typename... A>
[[noreturn]] void gcn_error(const A&... a) {
    PyErr_SetString(hip_error, text(a...).c_str());
    throw py::error_already_set();
}
void check(int rc, const char* what) {
    if (rc != 0) gcn_error(what, " failed (", rc, "): ", api.last_error());
}
void need_gpu(const at::Tensor& t, const char* name) {
    if (!t.is_cuda())
        gcn_error(name, " is on ", t.device(), ": the gfx950 HIP path needs tensors on a ROCm GPU (there is no CPU fallback; use the oracle "
                  "under oracle/ for CPU checks)");
}
void* stream_of(c10::Device d) { return c10::hip::getCurrentHIPStream(d.index()).stream(); }
bool capturing() { return c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None; }

int type_id(at::ScalarType t) { return t == at::kFloat ? GCN_F32 : t == at::kBFloat16 ? GCN_BF16 : t == at::kHalf ? GCN_F16 : -1; }

const at::Tensor* as_tensor(py::handle h) { return THPVariable_Check(h.ptr()) ? &THPVariable_Unpack(h.ptr()) : nullptr; }

// ---------------------------------------------------------------------------------------------- lists of tensors
struct List {
    const char* name;
    py::object held;
    std::vector<const at::Tensor*> t;
    std::vector<void*> ptr;
    bool given = false;

    // own: the tensors outlive the caller's list
    List(const char* name, py::handle h, bool own = false) : name(name) {
        if (h.is_none()) return;
        given = true;
        held = py::reinterpret_steal<py::object>(own ? PySequence_Tuple(h.ptr()) : PySequence_Fast(h.ptr(), text(name, " is a list of tensors").c_str()));
        if (!held) throw py::error_already_set();
        const Py_ssize_t n = PySequence_Fast_GET_SIZE(held.ptr());
        PyObject** items = PySequence_Fast_ITEMS(held.ptr());
        t.resize(n);
        for (Py_ssize_t k = 0; k < n; ++k) {
            t[k] = as_tensor(items[k]);
            if (!t[k]) type_error(name, " is a list of tensors");
        }
    }
    // as many tensors as `sizes`, of these sizes (or as many blocks of them) and this type, contiguous
    void check(const std::vector<int64_t>& sizes, at::ScalarType type, int64_t block = 1) {
        if (t.size() != sizes.size()) value_error(t.size(), " tensors in ", name, " for ", sizes.size(), " parameters");
        for (size_t k = 0; k < t.size(); ++k) {
            const at::TensorImpl* x = t[k]->unsafeGetTensorImpl();
            if (x->numel() != (block == 1 ? sizes[k] : (sizes[k] + block - 1) / block)) value_error("the tensors in ", name, " do not have the parameters' sizes");
            if (x->dtype() != at::scalarTypeToTypeMeta(type)) type_error(name, " holds ", t[k]->scalar_type(), " (expected ", type, ")");
            if (!x->is_contiguous()) value_error(name, " needs contiguous tensors");
        }
    }
    // all on that GPU; their addresses for the library
    void place(c10::Device d, bool written) {
        ptr.resize(t.size());
        for (size_t k = 0; k < t.size(); ++k) {
            if (t[k]->device() != d) {
                need_gpu(*t[k], "tensor");
                value_error("the tensors of one call are on one GPU");
            }
            ptr[k] = written ? t[k]->mutable_data_ptr() : const_cast<void*>(t[k]->const_data_ptr());
        }
    }
    // autograd hears of what was written
    void written() const {
        for (const at::Tensor* x : t)
            if (!x->is_inference()) x->unsafeGetTensorImpl()->bump_version();
    }
    void* const* table() const { return given ? ptr.data() : nullptr; }
};

const float* device_scalar(py::handle h, const char* name, c10::Device d) {
    if (h.is_none()) return nullptr;
    const at::Tensor* t = as_tensor(h);
    if (!t || t->scalar_type() != at::kFloat || t->numel() != 1) type_error(name, " is a float32 tensor of one element");
    if (t->device() != d) value_error(name, " is on ", t->device(), ", the tensors are on ", d);
    return static_cast<const float*>(t->const_data_ptr());
}

at::ScalarType one_type(const List& l, const char* what) {
    for (const at::Tensor* x : l.t)
        if (type_id(x->scalar_type()) < 0 || x->scalar_type() != l.t[0]->scalar_type())
            type_error(what, " of one type per call (float32, bfloat16 or float16), got ", l.t[0]->scalar_type(), " and ", x->scalar_type());
    return l.t.empty() ? at::kFloat : l.t[0]->scalar_type();
}
std::vector<int64_t> sizes_of(const List& l) {
    std::vector<int64_t> n;
    n.reserve(l.t.size());
    for (const at::Tensor* x : l.t) n.push_back(x->numel());
    return n;
}

// An AdamW step on lists of tensors in two parts: all that can be refused, and the launch.
struct AdamwCall {
    List params, grads, m, v, masters, em, ev;
    at::ScalarType type;
    bool eight;
    std::vector<int64_t> sizes;
    c10::Device d = at::kCPU;

    AdamwCall(py::handle params_, py::handle grads_, py::handle exp_avgs_, py::handle exp_avg_sqs_, py::handle masters_, py::handle exps_,
              py::handle sq_exps_, bool own)
        : params("params", params_, own), grads("grads", grads_, own), m("exp_avgs", exp_avgs_, own), v("exp_avg_sqs", exp_avg_sqs_, own),
          masters("masters", masters_, own), em("exp_avg_exps", exps_, own), ev("exp_avg_sq_exps", sq_exps_, own) {
        if (em.given != ev.given) value_error("exp_avg_exps and exp_avg_sq_exps go together");
        type = one_type(params, "parameters");
        const bool half = !params.t.empty() && type != at::kFloat;
        eight = em.given;
        sizes = sizes_of(params);
        params.check(sizes, type);
        grads.check(sizes, type);
        if (!params.t.empty() && half != masters.given) value_error("master copies go with 16-bit parameters, and only with them");
        m.check(sizes, eight ? at::kByte : at::kFloat);
        v.check(sizes, eight ? at::kByte : at::kFloat);
        if (half) masters.check(sizes, at::kFloat);
        if (eight) {
            em.check(sizes, at::kByte, GCN_STATE8_BLOCK);
            ev.check(sizes, at::kByte, GCN_STATE8_BLOCK);
        }
        if (params.t.empty()) return;
        d = params.t[0]->device();
        need_gpu(*params.t[0], "tensor");
        for (List* l : {&params, &grads, &m, &v, &masters, &em, &ev}) l->place(d, l != &grads);
        // a tensor twice, or a part of another, would be updated by two workgroups at once
        const size_t width = half ? 2 : 4;
        std::vector<std::pair<const char*, const char*>> once;
        for (size_t k = 0; k < sizes.size(); ++k)
            if (sizes[k] > 0) once.emplace_back(static_cast<char*>(params.ptr[k]), static_cast<char*>(params.ptr[k]) + sizes[k] * width);
        std::sort(once.begin(), once.end());
        for (size_t k = 1; k < once.size(); ++k) {
            if (once[k].first == once[k - 1].first) value_error("a parameter is in the list twice");
            if (once[k].first < once[k - 1].second) value_error("parameters overlap in memory");
        }
    }
    gcn_adamw_desc describe(double lr, double beta1, double beta2, double eps, double weight_decay) const {
        gcn_adamw_desc desc = {};
        desc.param_type = type_id(type);
        desc.state_bits = eight ? 8 : 32;
        desc.lr = lr; desc.beta1 = beta1; desc.beta2 = beta2; desc.eps = eps; desc.weight_decay = weight_decay;
        return desc;
    }
    // what run() would refuse of these
    void check_numbers(double lr, double beta1, double beta2, double eps, double weight_decay, py::handle grad_scale) const {
        if (params.t.empty()) return;
        device_scalar(grad_scale, "grad_scale", d);
        gcn_adamw_desc desc = describe(lr, beta1, beta2, eps, weight_decay);
        desc.step = 1;                              // and no tensors: nothing is launched
        check(api.adamw_step(&desc, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr), "gcn_adamw_step");
    }
    void run(long long step, double lr, double beta1, double beta2, double eps, double weight_decay, unsigned long long seed,
             unsigned int first_tensor, py::handle grad_scale, py::handle clip_coef, py::handle hyper_) const {
        if (params.t.empty()) return;
        const void* hyper = nullptr;
        if (!hyper_.is_none()) {
            const at::Tensor* t = as_tensor(hyper_);
            if (!t || t->scalar_type() != at::kByte || t->device() != d || static_cast<size_t>(t->numel()) < api.adamw_hyper_bytes())
                value_error("hyper is what adamw_hyper returned, on the tensors' device");
            hyper = t->const_data_ptr();
        }
        const float *scale = device_scalar(grad_scale, "grad_scale", d), *clip = device_scalar(clip_coef, "clip_coef", d);
        c10::DeviceGuard guard(d);
        if (!hyper && capturing()) gcn_error("a captured step would repeat its step count: pass hyper (adamw_advance_)");
        gcn_adamw_desc desc = describe(lr, beta1, beta2, eps, weight_decay);
        desc.n = static_cast<int>(sizes.size());
        desc.first_tensor = first_tensor;
        desc.step = step;
        desc.seed = seed;
        static_assert(sizeof(long long) == sizeof(int64_t), "sizes are handed over as they are");
        check(api.adamw_step(&desc, params.table(), grads.table(), reinterpret_cast<float* const*>(masters.table()), m.table(), v.table(),
                             reinterpret_cast<unsigned char* const*>(em.table()), reinterpret_cast<unsigned char* const*>(ev.table()),
                             reinterpret_cast<const long long*>(sizes.data()), scale, clip, hyper, stream_of(d)),
              "gcn_adamw_step");
        for (const List* l : {&params, &m, &v, &masters, &em, &ev}) l->written();
    }
};

void adamw_step(py::handle params, py::handle grads, py::handle exp_avgs, py::handle exp_avg_sqs, py::handle masters, py::handle exps, py::handle sq_exps,
                long long step, double lr, double beta1, double beta2, double eps, double weight_decay, unsigned long long seed,
                unsigned int first_tensor, py::handle grad_scale, py::handle clip_coef, py::handle hyper) {
    AdamwCall(params, grads, exp_avgs, exp_avg_sqs, masters, exps, sq_exps, false)
        .run(step, lr, beta1, beta2, eps, weight_decay, seed, first_tensor, grad_scale, clip_coef, hyper);
}

py::tuple grad_norm(py::handle grads_, py::handle max_norm_, py::handle grad_scale) {
    List grads("grads", grads_);
    if (grads.t.empty()) type_error("gradients of one type per call, got none");
    const at::ScalarType type = one_type(grads, "gradients");
    const bool clip = !max_norm_.is_none();
    const double max_norm = clip ? py::cast<double>(max_norm_) : 1.0;
    if (!(max_norm >= 0.0)) value_error("max_norm is not negative, got ", max_norm);
    const std::vector<int64_t> sizes = sizes_of(grads);
    grads.check(sizes, type);
    const c10::Device d = grads.t[0]->device();
    need_gpu(*grads.t[0], "tensor");
    grads.place(d, false);
    const float* scale = device_scalar(grad_scale, "grad_scale", d);
    c10::DeviceGuard guard(d);
    const int n = static_cast<int>(sizes.size());
    const long long* numel = reinterpret_cast<const long long*>(sizes.data());
    const size_t bytes = api.grad_norm_ws_bytes(n, numel);
    at::Tensor ws = at::empty({static_cast<int64_t>(bytes)}, at::TensorOptions().dtype(at::kByte).device(d));
    at::Tensor out = at::empty({2}, at::TensorOptions().dtype(at::kFloat).device(d));
    check(api.grad_norm(n, type_id(type), reinterpret_cast<const void* const*>(grads.table()), numel, scale, max_norm,
                        static_cast<float*>(out.mutable_data_ptr()), ws.mutable_data_ptr(), bytes, stream_of(d)),
          "gcn_grad_norm");
    return py::make_tuple(out.select(0, 0), clip ? py::cast(out.select(0, 1)) : py::none());
}

// ---------------------------------------------------------------------------------------------- logits
// The distance between consecutive rows of t[lead..., dim, ...] in elements; -1 if rows are not dense or not evenly spaced.
int64_t row_stride(const at::Tensor& t, int64_t dim) {
    int64_t want = 1;
    for (int64_t k = t.dim() - 1; k >= dim; --k) {
        if (t.size(k) != 1 && t.stride(k) != want) return -1;
        want *= t.size(k);
    }
    int64_t stride = -1, reach = 0;
    for (int64_t k = dim - 1; k >= 0; --k) {
        if (t.size(k) == 1) continue;
        if (stride < 0) stride = t.stride(k);
        else if (t.stride(k) != reach) return -1;
        reach = t.stride(k) * t.size(k);
    }
    return stride < 0 ? want : stride;
}

// What a tensor that is saved for the backward pass has to be when it comes back: hooks on saved tensors may return another one,
// with strides and an address of its own.
struct Saved {
    const char* name;
    std::vector<int64_t> sizes;
    at::ScalarType type;
    c10::Device device;

    Saved(const char* name, const at::Tensor& t) : name(name), sizes(t.sizes().vec()), type(t.scalar_type()), device(t.device()) {}
    void check(const at::Tensor& t) const {
        TORCH_CHECK(t.defined() && t.layout() == at::kStrided && t.sizes() == at::IntArrayRef(sizes) && t.scalar_type() == type && t.device() == device,
                    "process_logits: ", name, " was saved as ", type, " ", at::IntArrayRef(sizes), " on ", device, " and came back as something else");
    }
};

struct Rules : torch::CustomClassHolder {
    gcn_logits_desc d = {};
    int64_t dim = 0;
    std::vector<at::Tensor> kept;                  // what the descriptor points into (the bias apart), until it is saved
    std::vector<size_t> fields;                    // which of its fields, as offsets
    std::vector<const char*> names;
    std::vector<Saved> saved;                      // the logits, then what was kept
    at::Tensor bias;

    // rows of an argument whose leading dimensions are the first `lead` of t: all of the logits' leading dimensions, the last few
    // of them, or ones.  The outermost that it has may divide the logits' own: their row o takes row o mod rows
    long long rows_of(const char* name, const at::Tensor& t, int64_t lead, const at::Tensor& logits) const {
        int64_t n = 1, skip = 0;
        for (int64_t k = 0; k < lead; ++k) n *= t.size(k);
        if (n == 1) return 1;
        while (lead - skip > dim && t.size(skip) == 1) ++skip;
        bool fits = lead - skip <= dim;
        for (int64_t k = skip; fits && k < lead; ++k) {
            const int64_t have = t.size(k), of = logits.size(dim - lead + k);
            fits = have == of || (k == skip && have > 0 && of % have == 0);
        }
        if (!fits) value_error(name, ": leading dimensions ", t.sizes().slice(0, lead), " do not match the logits' ", logits.sizes().slice(0, dim), " from the last one on");
        return n;
    }
    // t's address goes into the descriptor's field at that offset (a pointer to const); t is made contiguous
    static void point(gcn_logits_desc* d, size_t field, const at::Tensor& t) {
        const void* address = t.const_data_ptr();
        std::memcpy(reinterpret_cast<char*>(d) + field, &address, sizeof(address));
    }
    void place(const char* name, const at::Tensor& t, const at::Tensor& logits, size_t field) {
        if (t.device() != logits.device()) value_error(name, " is on ", t.device(), ", the logits are on ", logits.device());
        kept.push_back(t.is_contiguous() ? t : t.contiguous());
        fields.push_back(field);
        names.push_back(name);
        point(&d, field, kept.back());
    }
    // What the gradient reads (not the bias): the logits, then what was kept.  From here on only autograd holds it, and its own
    // check of changes in between covers it.
    std::vector<at::Tensor> save(const at::Tensor& x) {
        std::vector<at::Tensor> out{x};
        saved.emplace_back("logits", x);
        for (size_t k = 0; k < kept.size(); ++k) {
            saved.emplace_back(names[k], kept[k]);
            out.push_back(std::move(kept[k]));
        }
        kept.clear();
        return out;
    }
    // The descriptor for what came back; `back` keeps what it points into, the logits first.
    gcn_logits_desc restore(std::vector<at::Tensor>* back) const {
        TORCH_CHECK(back->size() == saved.size(), "process_logits: saved tensors are missing");
        for (size_t k = 0; k < back->size(); ++k) saved[k].check((*back)[k]);
        gcn_logits_desc now = d;
        at::Tensor& x = (*back)[0];
        now.in_stride = row_stride(x, dim);
        if (now.in_stride < 0) {
            x = x.contiguous();
            now.in_stride = now.vocab * now.inner;
        }
        for (size_t k = 0; k < fields.size(); ++k) {
            const void* was;
            std::memcpy(&was, reinterpret_cast<const char*>(&d) + fields[k], sizeof(was));
            if (!was) continue;                     // not used: lengths of an empty history
            at::Tensor& t = (*back)[k + 1];
            if (!t.is_contiguous()) t = t.contiguous();
            point(&now, fields[k], t);
        }
        return now;
    }
};

bool is_int(const at::Tensor& t) { return t.scalar_type() == at::kInt || t.scalar_type() == at::kLong; }

const at::Tensor* tensor_or_none(py::handle h, const char* name) {
    if (h.is_none()) return nullptr;
    const at::Tensor* t = as_tensor(h);
    if (!t) type_error(name, " is a tensor");
    return t;
}

void penalty(Rules& r, py::handle h, const char* name, const at::Tensor& logits, bool positive, float* value, size_t table, long long* rows) {
    *rows = 1;
    if (const at::Tensor* t = as_tensor(h)) {
        if (t->scalar_type() != at::kFloat) type_error(name, " is a number or float32, got ", t->scalar_type());
        *rows = r.rows_of(name, *t, t->dim(), logits);
        r.place(name, *t, logits, table);
        return;
    }
    const double x = PyFloat_AsDouble(h.ptr());
    if (x == -1.0 && PyErr_Occurred()) throw py::error_already_set();
    *value = static_cast<float>(x);
    if (!std::isfinite(*value) || (positive && !(*value > 0.f && std::isfinite(1.f / *value)))) value_error(name, " ", x);
}

// Memory of `rows` rows of `len` bytes, `step` apart.
struct Region {
    uintptr_t at;
    int64_t step, len, rows;

    uintptr_t end() const { return at + (rows - 1) * step + len; }
    bool meets(uintptr_t lo, uintptr_t hi) const {
        if (hi <= at || lo >= end()) return false;
        const int64_t before = static_cast<int64_t>(lo - at) - len;             // the first row that ends behind lo
        const int64_t k = lo < at || before < 0 ? 0 : before / step + 1;
        return k < rows && at + k * step < hi;
    }
    bool meets(const Region& o) const {
        if (o.end() <= at || o.at >= end()) return false;
        for (int64_t k = 0; k < (o.step ? o.rows : 1); ++k)
            if (meets(o.at + k * o.step, o.at + k * o.step + o.len)) return true;
        return false;
    }
};
Region region_of(const at::Tensor& t, int64_t stride, int64_t rows) {
    const int64_t size = t.element_size(), len = t.numel() / rows * size;
    return {reinterpret_cast<uintptr_t>(t.const_data_ptr()), rows > 1 ? stride * size : len, len, rows};
}
// out is written while other workgroups read: its rows are the logits' own, or lie apart from them and from every argument.
void check_apart(const Rules& r, const at::Tensor& x, const at::Tensor& out) {
    if (out.numel() == 0) return;
    const Region to = region_of(out, row_stride(out, r.dim), r.d.rows), from = region_of(x, r.d.in_stride, r.d.rows);
    if (!(to.at == from.at && to.step == from.step) && to.meets(from)) value_error("out overlaps the logits, and is not the logits themselves");
    for (size_t k = 0; k <= r.kept.size(); ++k) {
        const at::Tensor& t = k < r.kept.size() ? r.kept[k] : r.bias;
        if (!t.defined() || t.numel() == 0) continue;
        const uintptr_t at = reinterpret_cast<uintptr_t>(t.const_data_ptr());
        if (to.meets(at, at + t.numel() * t.element_size())) value_error("out overlaps ", k < r.kept.size() ? r.names[k] : "bias");
    }
}

at::Tensor run_forward(Rules& r, const at::Tensor& x, const at::Tensor& out) {
    r.d.out_stride = row_stride(out, r.dim);
    c10::DeviceGuard guard(x.device());
    check(api.logits_process(&r.d, x.const_data_ptr(), out.mutable_data_ptr(), stream_of(x.device())), "gcn_logits_process");
    return out;
}

// A leaf's gradients are accumulated by a node that lives as long as any graph over the leaf does, on the stream of the first of
// them.  A captured backward that meets one of another stream would wait for work outside its capture, which ends the process.
void check_leaf(const at::Tensor& t, const char* name) {
    if (!t.requires_grad() || !t.is_leaf()) return;
    const std::shared_ptr<torch::autograd::Node> node = torch::autograd::impl::try_get_grad_accumulator(t);
    if (!node) return;
    const std::optional<c10::Stream> stream = node->stream();
    if (stream && *stream != c10::hip::getCurrentHIPStream(t.device().index()).unwrap())
        gcn_error("process_logits: ", name, " is a leaf of a graph that lives on another stream; free what that graph computed (its outputs) "
                  "before capturing one, or capture over a detached copy");
}

// There is no forward-mode derivative: a tangent would be lost without a word.
void check_tangent(const at::Tensor& t, const char* name) {
    if (t._fw_grad(0).defined()) gcn_error("process_logits: ", name, " carries a tangent, and there is no forward-mode derivative");
}

struct ProcessLogits : torch::autograd::Function<ProcessLogits> {
    static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& logits, const std::optional<at::Tensor>& bias, const at::Tensor& x,
                              c10::intrusive_ptr<Rules> r) {
        at::Tensor out = at::empty(logits.sizes(), logits.options());
        if (logits.numel()) run_forward(*r, x, out);
        ctx->save_for_backward(r->save(x));
        ctx->saved_data["rules"] = c10::IValue::make_capsule(r);
        if (bias) ctx->saved_data["bias_shape"] = bias->sizes().vec();
        return out;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        std::vector<at::Tensor> back = ctx->get_saved_variables();
        const bool want_x = ctx->needs_input_grad(0), want_bias = ctx->saved_data.count("bias_shape") && ctx->needs_input_grad(1);
        at::Tensor dx, dbias;
        {
            at::NoGradGuard no_grad;
            c10::intrusive_ptr<torch::CustomClassHolder> holder = ctx->saved_data["rules"].toCapsule();
            gcn_logits_desc d = static_cast<Rules*>(holder.get())->restore(&back);
            const at::Tensor& x = back[0];
            const at::Tensor dy = grads[0].contiguous();
            d.out_stride = d.vocab * d.inner;
            c10::DeviceGuard guard(x.device());
            if (want_x) dx = at::empty(dy.sizes(), dy.options());
            const at::TensorOptions options = at::TensorOptions().device(x.device()).dtype(at::kFloat);
            if (want_bias) {
                const std::vector<int64_t> shape = ctx->saved_data["bias_shape"].toIntVector();
                dbias = dy.numel() ? at::empty(shape, options) : at::zeros(shape, options);
            }
            if (dy.numel() && (want_x || want_bias)) {
                const size_t bytes = want_bias ? api.logits_bwd_ws_bytes(&d) : 0;
                at::Tensor ws = bytes ? at::empty({static_cast<int64_t>(bytes)}, options.dtype(at::kByte)) : at::Tensor();
                const int rc = api.logits_process_bwd(&d, x.const_data_ptr(), dy.const_data_ptr(), want_x ? dx.mutable_data_ptr() : nullptr,
                                                      want_bias ? static_cast<float*>(dbias.mutable_data_ptr()) : nullptr,
                                                      bytes ? ws.mutable_data_ptr() : nullptr, bytes, stream_of(x.device()));
                TORCH_CHECK(rc == 0, "gcn_logits_process_bwd failed (", rc, "): ", api.last_error());
            }
        }
        torch::autograd::variable_list out{dx, dbias, at::Tensor(), at::Tensor()};
        if (at::GradMode::is_enabled() && grads[0].requires_grad()) {
            auto error = std::make_shared<torch::autograd::DelayedError>("process_logits is once_differentiable: its gradient has no gradient", 2);
            for (at::Tensor* t : {&dx, &dbias})
                if (t->defined()) *t = t->detach().set_requires_grad(true);
            torch::autograd::variable_list marked = (*error)({dx, dbias});
            out[0] = marked[0];
            out[1] = marked[1];
        }
        return out;
    }
};

py::object process_logits(py::handle logits_, int64_t dim, py::handle history_, py::handle history_lens_, py::handle prompt_lens_, py::handle repetition,
                          py::handle presence, py::handle frequency, py::handle bias_, py::handle mask_, py::handle temperature, double masked_value,
                          py::handle out_) {
    const at::Tensor* lp = as_tensor(logits_);
    if (!lp || type_id(lp->scalar_type()) < 0) type_error("logits are float32, bfloat16 or float16 tensors");
    const at::Tensor& logits = *lp;
    check_tangent(logits, "logits");
    if (dim < -logits.dim() || dim >= logits.dim()) value_error("logits of shape ", logits.sizes(), " have no dimension ", dim);
    auto rules = c10::make_intrusive<Rules>();
    Rules& r = *rules;
    gcn_logits_desc& d = r.d;
    r.dim = dim < 0 ? dim + logits.dim() : dim;
    d.rows = d.inner = 1;
    for (int64_t k = 0; k < logits.dim(); ++k) (k < r.dim ? d.rows : k == r.dim ? d.vocab : d.inner) *= k == r.dim ? 1 : logits.size(k);
    d.vocab = logits.size(r.dim);
    d.type = type_id(logits.scalar_type());
    d.masked_value = static_cast<float>(masked_value);
    d.history_rows = d.bias_rows = d.mask_rows = 1;
    const at::Tensor *history = tensor_or_none(history_, "history"), *lens = tensor_or_none(history_lens_, "history_lens"),
                     *prompts = tensor_or_none(prompt_lens_, "prompt_lens");
    if (history) {
        if (!is_int(*history) || history->dim() == 0) type_error("history holds int32 or int64 entries [..., length]");
        d.history_rows = r.rows_of("history", *history, history->dim() - 1, logits);
        d.history_len = history->size(-1);
        d.history_wide = history->scalar_type() == at::kLong;
        r.place("history", *history, logits, offsetof(gcn_logits_desc, history));
        for (const at::Tensor* t : {lens, prompts}) {
            if (!t) continue;
            if (!is_int(*t) || (lens && t->scalar_type() != lens->scalar_type())) type_error("history_lens and prompt_lens are int32 or int64, both alike");
            if (t->sizes() != history->sizes().slice(0, history->dim() - 1))
                value_error("lengths of shape ", t->sizes(), " for a history with rows ", history->sizes().slice(0, history->dim() - 1));
            d.lens_wide = t->scalar_type() == at::kLong;
            r.place("history_lens and prompt_lens", *t, logits, t == lens ? offsetof(gcn_logits_desc, history_lens) : offsetof(gcn_logits_desc, prompt_lens));
        }
        // without entries nothing is read; an empty tensor has no address
        if (!d.history) d.history_lens = d.prompt_lens = nullptr;
    } else if (lens || prompts) {
        value_error("history_lens and prompt_lens go with a history");
    }
    penalty(r, repetition, "repetition penalty", logits, true, &d.repetition, offsetof(gcn_logits_desc, repetition_t), &d.repetition_rows);
    penalty(r, presence, "presence penalty", logits, false, &d.presence, offsetof(gcn_logits_desc, presence_t), &d.presence_rows);
    penalty(r, frequency, "frequency penalty", logits, false, &d.frequency, offsetof(gcn_logits_desc, frequency_t), &d.frequency_rows);
    penalty(r, temperature, "temperature", logits, true, &d.temperature, offsetof(gcn_logits_desc, temperature_t), &d.temperature_rows);
    if (const at::Tensor* mask = tensor_or_none(mask_, "mask")) {
        if ((mask->scalar_type() != at::kBool && mask->scalar_type() != at::kInt) || mask->dim() == 0) type_error("mask holds truth values, or bits in int32 words");
        d.mask_type = mask->scalar_type() == at::kBool ? 1 : 2;
        if (mask->size(-1) != (d.mask_type == 1 ? d.vocab : (d.vocab + 31) / 32)) value_error("mask of shape ", mask->sizes(), " for ", d.vocab, " entries");
        d.mask_rows = r.rows_of("mask", *mask, mask->dim() - 1, logits);
        r.place("mask", *mask, logits, offsetof(gcn_logits_desc, mask));
    }
    const at::Tensor* bias = tensor_or_none(bias_, "bias");
    if (bias) {
        check_tangent(*bias, "bias");
        if (bias->scalar_type() != at::kFloat || bias->dim() == 0) type_error("bias is float32 [..., vocabulary]");
        if (bias->size(-1) != d.vocab) value_error("bias of shape ", bias->sizes(), " for ", d.vocab, " entries");
        d.bias_rows = r.rows_of("bias", *bias, bias->dim() - 1, logits);
        if (bias->device() != logits.device()) value_error("bias is on ", bias->device(), ", the logits are on ", logits.device());
        r.bias = bias->is_contiguous() ? *bias : bias->detach().contiguous();
        d.bias = static_cast<const float*>(r.bias.const_data_ptr());
    }
    const bool grad = at::GradMode::is_enabled() && (logits.requires_grad() || (bias && bias->requires_grad()));
    const at::Tensor* out = tensor_or_none(out_, "out");
    if (out) {
        check_tangent(*out, "out");
        if (grad || (at::GradMode::is_enabled() && out->requires_grad())) value_error("out does not go with gradients");
        if (out->sizes() != logits.sizes() || out->scalar_type() != logits.scalar_type() || out->device() != logits.device())
            value_error("out is a tensor like the logits");
        const int64_t stride = row_stride(*out, r.dim);
        if (stride < 0 || (d.rows > 1 && stride < d.vocab * d.inner)) value_error("out needs dense rows that do not overlap");
    }
    need_gpu(logits, "logits");
    if (logits.numel() == 0 && !grad) return out ? py::reinterpret_borrow<py::object>(out_) : py::cast(at::empty(logits.sizes(), logits.options()));
    if (d.mask_type && !d.mask) d.mask_type = 0;      // an empty one, for no rows
    d.in_stride = row_stride(logits, r.dim);
    at::Tensor x = logits;
    if (d.in_stride < 0) {
        x = logits.detach().contiguous();
        d.in_stride = d.vocab * d.inner;
    }
    if (out) check_apart(r, x, *out);
    if (grad) {
        c10::DeviceGuard guard(logits.device());
        if (capturing()) {
            check_leaf(logits, "logits");
            if (bias) check_leaf(*bias, "bias");
        }
    }
    if (grad) return py::cast(ProcessLogits::apply(logits, bias ? std::optional<at::Tensor>(*bias) : std::nullopt, x.detach(), rules));
    if (out) {
        run_forward(r, x, *out);
        if (!out->is_inference()) out->unsafeGetTensorImpl()->bump_version();
        return py::reinterpret_borrow<py::object>(out_);
    }
    return py::cast(run_forward(r, x, at::empty(logits.sizes(), logits.options())));
}

void bind(const py::dict& addresses, py::object error) {
    const auto get = [&](const char* name, auto& fn) { fn = reinterpret_cast<std::decay_t<decltype(fn)>>(py::cast<uintptr_t>(addresses[name])); };
    get("gcn_last_error", api.last_error);
    get("gcn_adamw_step", api.adamw_step);
    get("gcn_adamw_hyper_bytes", api.adamw_hyper_bytes);
    get("gcn_grad_norm_ws_bytes", api.grad_norm_ws_bytes);
    get("gcn_grad_norm", api.grad_norm);
    get("gcn_logits_process", api.logits_process);
    get("gcn_logits_bwd_ws_bytes", api.logits_bwd_ws_bytes);
    get("gcn_logits_process_bwd", api.logits_process_bwd);
    hip_error = error.release().ptr();
}

}  // namespace

PYBIND11_MODULE(gcn_uelb_torch, m) {
    m.def("bind", &bind);
    m.def("adamw_step", &adamw_step);
    py::class_<AdamwCall>(m, "AdamwCall")
        .def(py::init([](py::handle params, py::handle grads, py::handle exp_avgs, py::handle exp_avg_sqs, py::handle masters, py::handle exps,
                         py::handle sq_exps) { return std::make_unique<AdamwCall>(params, grads, exp_avgs, exp_avg_sqs, masters, exps, sq_exps, true); }))
        .def("check_numbers", &AdamwCall::check_numbers)
        .def("run", &AdamwCall::run);
    m.def("grad_norm", &grad_norm);
    m.def("process_logits", &process_logits);
    m.def("row_stride", [](const at::Tensor& t, int64_t dim) { return row_stride(t, dim); });
    m.def("rows_meet", [](const at::Tensor& a, const at::Tensor& b) {
        return region_of(a, row_stride(a, 1), a.size(0)).meets(region_of(b, row_stride(b, 1), b.size(0)));
    });
    m.def("check_saved", [](const at::Tensor& was, const at::Tensor& now) { Saved("tensor", was).check(now); });
}
