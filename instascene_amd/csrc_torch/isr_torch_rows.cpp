// The row and gradient operators of instascene_amd/rows.py and optim.py for torch: argument checks, allocation, the autograd node of
// rms_norm, and the calls into the C ABI (include/instascene_ops.h).  Host glue only, like isr_torch_ext.cpp: these calls take a few
// microseconds of kernel time at decode sizes, so what surrounds them is compiled (an rms_norm of one row forward: 11 us through ctypes).
// Errors: TypeError / ValueError for arguments, instascene_amd._lib.IsrError for what the library refuses.
#include <torch/extension.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <limits>
#include <optional>
#include <stdexcept>
#include <string>
#include <vector>

#include "instascene_rasterizer.h"
#include "instascene_ops.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

struct LibraryError : std::runtime_error { using std::runtime_error::runtime_error; };

void check(int rc, const char* what) {
    if (rc != ISR_OK) throw LibraryError(std::string(what) + " failed (code " + std::to_string(rc) + "): " + isr_last_error());
}
void* stream_on(const c10::Device& d) { return (void*)c10::hip::getCurrentHIPStream(d.index()).stream(); }

int row_type(at::ScalarType t) { return t == at::kFloat ? 0 : t == at::kBFloat16 ? 1 : t == at::kHalf ? 2 : -1; }
int code_type(at::ScalarType t) { return t == at::kChar ? 1 : t == at::kFloat8_e4m3fn ? 2 : 0; }

constexpr int64_t MAX_WIDTH = 1 << 24;

// The kernels write through raw pointers, which a trace does not record (what it would keep is the uninitialised output) and which carry no
// tangent: both are refused, by every entry, before anything else is looked at.
void refuse_trace(const char* what) {
    using c10::impl::TorchDispatchModeKey;
    TORCH_CHECK(!torch::jit::tracer::isTracing() && !c10::impl::TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::PROXY).has_value(), what,
                " cannot be traced: its kernels would not be recorded");
}
void refuse_tangent(const char* what, const Tensor& t) {
    TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(/*level=*/0).defined(), what, " has no forward-mode derivative, and an input carries a tangent");
}
void refuse_modes(const char* what, std::initializer_list<OptTensor> inputs) {
    refuse_trace(what);
    for (const OptTensor& t : inputs)
        if (t) refuse_tangent(what, *t);
}

void check_rows(const char* what, const Tensor& x) {
    TORCH_CHECK(x.is_cuda(), what, ": needs CUDA tensors (the HIP library is the only backend)");
    TORCH_CHECK_TYPE(row_type(x.scalar_type()) >= 0, what, ": float32, bfloat16 or float16, not ", x.scalar_type());
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= MAX_WIDTH, what, ": rows of 1 to 2^24 columns, not a tensor of shape ", x.sizes());
}
void check_norm(const char* what, const Tensor& x, const OptTensor& weight, double eps, const OptTensor& residual) {
    check_rows(what, x);
    // (as the kernels see it: float32)
    TORCH_CHECK_VALUE((float)eps > 0.0f && std::isfinite((float)eps), what, ": eps must be positive and finite in float32");
    if (weight) {
        TORCH_CHECK_VALUE(weight->device() == x.device() && weight->dim() == 1 && weight->size(0) == x.size(-1), what, ": weight must be [", x.size(-1),
                          "] on ", x.device(), ", not ", weight->sizes(), " on ", weight->device());
        TORCH_CHECK_TYPE(weight->scalar_type() == at::kFloat || weight->scalar_type() == x.scalar_type(), what, ": weight must be float32 or ",
                         x.scalar_type(), ", not ", weight->scalar_type());
    }
    if (residual)
        TORCH_CHECK_VALUE(residual->sizes() == x.sizes() && residual->scalar_type() == x.scalar_type() && residual->device() == x.device(), what,
                          ": residual must be a ", x.scalar_type(), " ", x.sizes(), " on ", x.device(), " like x");
}
int64_t check_group(const char* what, int64_t width, std::optional<int64_t> group) {
    if (!group || *group == width) return width;
    TORCH_CHECK_VALUE((*group == 32 || *group == 64 || *group == 128) && width % *group == 0, what,
                      ": groups of 32, 64 or 128 columns that divide the row, or None for one per row: not ", *group, " of ", width);
    return *group;
}
int check_code(const char* what, at::ScalarType t) {
    TORCH_CHECK_TYPE(code_type(t) != 0, what, ": dtype must be torch.int8 or torch.float8_e4m3fn, not ", t);
    return code_type(t);
}
// [rows, F] with the columns of a row next to each other (a copy only where they are not, or where the memory holds the negative of the values)
Tensor as_stored(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }
Tensor rows2d(const Tensor& t) {
    Tensor r = t.dim() == 2 ? t : t.reshape({t.numel() / t.size(-1), t.size(-1)});
    return as_stored(r.size(1) == 1 || r.stride(1) == 1 ? r : r.contiguous());
}
Tensor gain_of(const Tensor& w) { return w.defined() ? as_stored(w.contiguous()) : Tensor(); }
// a tensor that may be absent, as rows
struct Rows {
    Tensor t;
    Rows() = default;
    explicit Rows(const Tensor& x) { if (x.defined()) t = rows2d(x); }
    const void* data() const { return t.defined() ? t.data_ptr() : nullptr; }
    long long stride() const { return t.defined() ? t.stride(0) : 0; }
};
const void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

struct Forward { Tensor y, s, rstd; };
Forward norm_forward(const Tensor& x, const Tensor& weight, double eps, const Tensor& residual, bool want_rstd) {
    const c10::DeviceGuard guard(x.device());
    const Rows x2(x), r2(residual);
    const Tensor w = gain_of(weight);
    Forward f;
    f.y = at::empty(x.sizes(), x.options());
    if (residual.defined()) f.s = at::empty(x.sizes(), x.options());
    if (want_rstd) f.rstd = at::empty({x2.t.size(0)}, x.options().dtype(at::kFloat));
    check(iso_rms_norm_forward(row_type(x.scalar_type()), x2.t.size(0), (int)x2.t.size(1), x2.data(), x2.stride(), r2.data(), r2.stride(), ptr(w),
                               w.defined() && w.scalar_type() == at::kFloat, (float)eps, f.y.data_ptr(), (void*)ptr(f.s), (float*)ptr(f.rstd),
                               stream_on(x.device())), "iso_rms_norm_forward");
    return f;
}

class RmsNorm : public torch::autograd::Function<RmsNorm> {
public:
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const OptTensor& weight_, double eps,
                                                  const OptTensor& residual_) {
        const Tensor weight = weight_.value_or(Tensor()), residual = residual_.value_or(Tensor());
        const Forward f = norm_forward(x, weight, eps, residual, true);
        // float32: s is x + residual exactly as the norm took it.  16 bits: s was rounded once more on its way out, and the gradient of the weight
        // would carry that (2^-9 of every term): x and the residual are read again instead
        const bool from_s = residual.defined() && x.scalar_type() == at::kFloat;
        ctx->save_for_backward({from_s ? f.s : x, from_s ? Tensor() : residual, weight, f.rstd});
        ctx->set_materialize_grads(false);
        ctx->saved_data["x"] = x.requires_grad();
        ctx->saved_data["w"] = weight.defined() && weight.requires_grad();
        ctx->saved_data["r"] = residual.defined() && residual.requires_grad();
        if (residual.defined()) return {f.y, f.s};
        return {f.y};
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        const bool again = at::GradMode::is_enabled();          // create_graph: the gradients cannot be differentiated once more
        torch::autograd::variable_list out;
        {
            at::AutoGradMode off(false);
            out = gradients(ctx, grads[0], grads.size() > 1 ? grads[1] : Tensor());
        }
        if (again) {                    // an error for whoever does differentiate them
            torch::autograd::variable_list some;
            for (const Tensor& t : out)
                if (t.defined()) some.push_back(t.detach().set_requires_grad(true));
            auto error = std::make_shared<torch::autograd::DelayedError>("rms_norm: the gradients of its backward pass are not available", (int)some.size());
            some = (*error)(std::move(some));
            size_t k = 0;
            for (Tensor& t : out)
                if (t.defined()) t = some[k++];
        }
        return out;
    }

private:
    static torch::autograd::variable_list gradients(torch::autograd::AutogradContext* ctx, const Tensor& gy, const Tensor& gs) {
        const bool need_x = ctx->saved_data["x"].toBool(), need_w = ctx->saved_data["w"].toBool(), need_r = ctx->saved_data["r"].toBool();
        if (!gy.defined())                                      // only the sum was used: its gradient passes through
            return {need_x ? gs : Tensor(), Tensor(), Tensor(), need_r ? gs : Tensor()};
        refuse_modes("the backward pass of rms_norm", {gy, gs});
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &residual = saved[1], &weight = saved[2], &rstd = saved[3];
        const c10::DeviceGuard guard(x.device());
        const Rows x2(x), r2(residual), g2(gy), q2(gs);
        const int type = row_type(x.scalar_type());
        const int64_t n = x2.t.size(0), F = x2.t.size(1);
        const Tensor w = gain_of(weight);
        Tensor ds, dw, scratch;
        if (need_x || need_r) ds = at::empty(x.sizes(), x.options());
        size_t bytes = 0;
        if (need_w) {
            dw = n > 0 ? at::empty({F}, weight.options()) : at::zeros({F}, weight.options());
            bytes = iso_rms_norm_scratch_bytes(type, n, (int)F);
            scratch = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
        }
        if (ds.defined() || dw.defined())
            check(iso_rms_norm_backward(type, n, (int)F, x2.data(), x2.stride(), r2.data(), r2.stride(), ptr(w), w.defined() && w.scalar_type() == at::kFloat,
                                        (const float*)ptr(rstd), g2.data(), g2.stride(), q2.data(), q2.stride(), (void*)ptr(ds), (void*)ptr(dw),
                                        (void*)ptr(scratch), bytes, stream_on(x.device())), "iso_rms_norm_backward");
        return {need_x ? ds : Tensor(), dw, Tensor(), need_r ? ds : Tensor()};
    }
};

bool wants_grad(const Tensor& x, const OptTensor& weight, const OptTensor& residual) {
    return at::GradMode::is_enabled() && (x.requires_grad() || (weight && weight->requires_grad()) || (residual && residual->requires_grad()));
}

// (y, s), s None without a residual
std::pair<Tensor, OptTensor> rms_norm(const Tensor& x, const OptTensor& weight, double eps, const OptTensor& residual) {
    refuse_modes("rms_norm", {x, weight, residual});
    check_norm("rms_norm", x, weight, eps, residual);
    if (wants_grad(x, weight, residual)) {
        auto out = RmsNorm::apply(x, weight, eps, residual);
        return {out[0], residual ? OptTensor(out[1]) : std::nullopt};
    }
    const Forward f = norm_forward(x, weight.value_or(Tensor()), eps, residual.value_or(Tensor()), false);
    return {f.y, residual ? OptTensor(f.s) : std::nullopt};
}

// (codes, scales, s)
std::tuple<Tensor, Tensor, OptTensor> rms_norm_quantized(const Tensor& x, const OptTensor& weight_, double eps, const OptTensor& residual_,
                                                         at::ScalarType dtype, std::optional<int64_t> group) {
    const char* what = "rms_norm_quantized";
    refuse_modes(what, {x, weight_, residual_});
    check_norm(what, x, weight_, eps, residual_);
    TORCH_CHECK_VALUE(x.dim() == 2, what, ": x must be [rows, F]");
    const int code = check_code(what, dtype);
    TORCH_CHECK(!wants_grad(x, weight_, residual_), what, " has no gradient: call it under torch.no_grad() or on detached tensors");
    const c10::DeviceGuard guard(x.device());
    const int64_t n = x.size(0), F = x.size(1), G = check_group(what, F, group);
    const Rows x2(x), r2(residual_.value_or(Tensor()));
    const Tensor w = gain_of(weight_.value_or(Tensor()));
    Tensor codes = at::empty({n, F}, x.options().dtype(dtype)), scales = at::empty({n, F / G}, x.options().dtype(at::kFloat)), s;
    if (residual_) s = at::empty({n, F}, x.options());
    check(iso_rms_norm_quant(row_type(x.scalar_type()), code, n, (int)F, (int)G, x2.data(), x2.stride(), r2.data(), r2.stride(), ptr(w),
                             w.defined() && w.scalar_type() == at::kFloat, (float)eps, codes.data_ptr(), (float*)scales.data_ptr(), (void*)ptr(s),
                             stream_on(x.device())), "iso_rms_norm_quant");
    return {codes, scales, residual_ ? OptTensor(s) : std::nullopt};
}

Tensor check_index(const char* what, const Tensor& index, const Tensor& codes, int64_t n) {
    TORCH_CHECK_VALUE(index.dim() == 1 && (index.scalar_type() == at::kLong || index.scalar_type() == at::kInt) && index.device() == codes.device(), what,
                      ": index must be a 1-D int64 or int32 tensor on ", codes.device());
    TORCH_CHECK_VALUE(n < 0 || index.size(0) == n, what, ": ", index.size(0), " indices for ", n, " rows");
    return index.contiguous();
}

// rows into the table: `index` (with `owner` beyond ISO_ROWS8_SCAN of them), or the rows from `first` on
void rows8_write(const Tensor& codes, const Tensor& scales, const OptTensor& owner, const Tensor& rows, const OptTensor& index, int64_t first) {
    const char* what = "QuantizedRows.write";
    refuse_modes(what, {rows});
    const int64_t P = codes.size(0), F = codes.size(1);
    check_rows(what, rows);
    TORCH_CHECK_VALUE(rows.dim() == 2 && rows.size(1) == F && rows.device() == codes.device(), what, ": rows must be [n, ", F, "] on ", codes.device(), ", not ",
                      rows.sizes(), " on ", rows.device());
    const int64_t n = rows.size(0);
    const c10::DeviceGuard guard(codes.device());
    const Rows r(rows);
    Tensor ix;
    if (index) ix = check_index(what, *index, codes, n);
    else TORCH_CHECK_VALUE(first >= 0 && first <= P && n <= P - first, what, ": rows [", first, ", ", first + n, ") of a table of ", P);
    check(iso_rows8_write(row_type(rows.scalar_type()), code_type(codes.scalar_type()), n, (int)F, (int)(F / scales.size(1)), P, r.data(), r.stride(), first,
                          ptr(ix), ix.defined() && ix.scalar_type() == at::kLong, owner ? (int*)owner->data_ptr() : nullptr, codes.data_ptr(),
                          (float*)scales.data_ptr(), stream_on(codes.device())), "iso_rows8_write");
    codes.unsafeGetTensorImpl()->bump_version();            // the kernel wrote through raw pointers
    scales.unsafeGetTensorImpl()->bump_version();
}

Tensor rows8_read(const Tensor& codes, const Tensor& scales, const OptTensor& index, int64_t first, int64_t count, at::ScalarType out_dtype,
                  std::optional<double> norm_eps) {
    const char* what = "QuantizedRows.read";
    refuse_trace(what);
    const int type = row_type(out_dtype);
    TORCH_CHECK_TYPE(type >= 0, what, ": out_dtype must be float32, bfloat16 or float16, not ", out_dtype);
    TORCH_CHECK_VALUE(!norm_eps || (*norm_eps >= 0.0 && std::isfinite((float)*norm_eps)), what, ": norm_eps must be finite and not negative");
    const int64_t P = codes.size(0), F = codes.size(1);
    const c10::DeviceGuard guard(codes.device());
    Tensor ix;
    if (index) ix = check_index(what, *index, codes, -1);
    const int64_t n = index ? ix.size(0) : count;
    Tensor out = at::empty({n, F}, scales.options().dtype(out_dtype));
    check(iso_rows8_read(type, code_type(codes.scalar_type()), n, (int)F, (int)(F / scales.size(1)), P, codes.data_ptr(), (const float*)scales.data_ptr(), first,
                         ptr(ix), ix.defined() && ix.scalar_type() == at::kLong, norm_eps.has_value(), (float)norm_eps.value_or(0.0), out.data_ptr(),
                         stream_on(codes.device())), "iso_rows8_read");
    return out;
}

// one stretch of memory, each element once (in any order of the dimensions)
bool is_dense(const Tensor& t) { return t.is_contiguous() || t.is_non_overlapping_and_dense(); }

// Memory that strided tensors share, decided on the host: a byte of `a` is a byte of `b` where  sum stride_k x_k = address(a) - address(b)  has a
// solution in whole numbers, with the indices of b counted up, those of a counted down and a byte within an element as one more dimension.
struct Dim { int64_t stride, lo, hi; };
int64_t floor_div(int64_t a, int64_t b) { return a >= 0 ? a / b : -((-a + b - 1) / b); }
// dims by falling stride.  Nested strides, as views have them, leave two or three candidates per dimension; a search that does not end within
// `left` steps (strides that no view of a bucket has) counts as shared.
bool reaches(const std::vector<Dim>& dims, size_t k, int64_t target, int& left) {
    if (k == dims.size()) return target == 0;
    if (--left < 0) return true;
    int64_t least = 0, most = 0;                // what the smaller strides reach
    for (size_t j = k + 1; j < dims.size(); j++) { least += dims[j].stride * dims[j].lo; most += dims[j].stride * dims[j].hi; }
    const int64_t s = dims[k].stride, from = std::max(dims[k].lo, -floor_div(most - target, s)), to = std::min(dims[k].hi, floor_div(target - least, s));
    for (int64_t x = from; x <= to; x++)
        if (reaches(dims, k + 1, target - s * x, left)) return true;
    return false;
}
void add_dims(std::vector<Dim>& dims, const Tensor& t, bool up, bool down) {
    auto add = [&](int64_t stride, int64_t n) {
        for (Dim& d : dims)
            if (d.stride == stride) { d.lo -= down ? n : 0; d.hi += up ? n : 0; return; }
        dims.push_back({stride, down ? -n : 0, up ? n : 0});
    };
    const int64_t size = t.element_size();
    add(1, size - 1);
    for (int64_t i = 0; i < t.dim(); i++)
        if (t.size(i) > 1) add(t.stride(i) * size, t.size(i) - 1);
}
constexpr int SEARCH = 100000;
void by_stride(std::vector<Dim>& dims) { std::sort(dims.begin(), dims.end(), [](const Dim& a, const Dim& b) { return a.stride > b.stride; }); }
bool share_memory(const Tensor& a, const Tensor& b) {
    std::vector<Dim> dims;
    add_dims(dims, a, false, true);
    add_dims(dims, b, true, false);
    by_stride(dims);
    int left = SEARCH;
    return reaches(dims, 0, (int64_t)((intptr_t)a.data_ptr() - (intptr_t)b.data_ptr()), left);
}
// two elements of one tensor in one place (strides that are not 0)
bool overlaps_itself(const Tensor& t) {
    const int64_t size = t.element_size();
    int left = SEARCH;
    for (int64_t i = 0; i < t.dim(); i++) {
        if (t.size(i) <= 1) continue;
        std::vector<Dim> dims;
        add_dims(dims, t.select(i, 0), true, true);
        dims.push_back({t.stride(i) * size, 1, t.size(i) - 1});
        by_stride(dims);
        if (reaches(dims, 0, 0, left)) return true;
    }
    return false;
}
void refuse_shared_memory(const std::vector<Tensor>& tensors) {
    struct Span { uintptr_t from, to; const Tensor* t; bool dense; };
    std::vector<Span> spans;
    for (const Tensor& t : tensors) {
        if (t.numel() == 0) continue;
        int64_t reach = 1;
        for (int64_t d = 0; d < t.dim(); d++) reach += (t.size(d) - 1) * t.stride(d);
        const uintptr_t from = (uintptr_t)t.data_ptr();
        spans.push_back({from, from + (uintptr_t)(reach * (int64_t)t.element_size()), &t, is_dense(t)});
        if (!spans.back().dense && overlaps_itself(t)) throw LibraryError("clip_grads_: a tensor to be clipped has elements that share memory");
    }
    std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.from < b.from; });
    for (size_t i = 0; i < spans.size(); i++)
        for (size_t j = i + 1; j < spans.size() && spans[j].from < spans[i].to; j++)
            if ((!spans[i].dense || !spans[j].dense) && share_memory(*spans[i].t, *spans[j].t))
                throw LibraryError("clip_grads_: two of the tensors to be clipped share memory");
}

// (norm, factor) of all elements together [, and the tensors scaled in place]
Tensor norm_and_factor(const std::vector<Tensor>& tensors, double norm_type, double max_norm, bool clip) {
    const char* what = clip ? "clip_grads_" : "grad_norm";
    refuse_trace(what);
    for (const Tensor& t : tensors) refuse_tangent(what, t);
    const int kind = norm_type == 2.0 ? 2 : norm_type == 1.0 ? 1 : norm_type == std::numeric_limits<double>::infinity() ? 0 : -1;
    TORCH_CHECK_VALUE(kind >= 0, what, ": norm_type must be 1, 2 or inf, not ", norm_type);
    const at::AutoGradMode off(false);
    const int n = (int)tensors.size();
    const c10::Device dev = tensors[0].device();
    std::vector<void*> at_(n);
    std::vector<long long> sizes(n);
    std::vector<int> types(n);
    std::vector<std::pair<int, Tensor>> copies;             // tensors that are no stretch of memory go through a copy
    for (int i = 0; i < n; i++) {
        const Tensor& t = tensors[i];
        TORCH_CHECK(t.layout() == at::kStrided && t.is_cuda(), what, ": needs dense CUDA tensors (the HIP library is the only backend)");
        TORCH_CHECK_TYPE(row_type(t.scalar_type()) >= 0, what, ": float32, bfloat16 or float16 gradients, not ", t.scalar_type());
        TORCH_CHECK_VALUE(t.device() == dev, what, ": all gradients must be on one device, not ", dev, " and ", t.device());
        void* p = nullptr;
        if (is_dense(t)) p = t.data_ptr();
        else {
            if (clip)
                for (int64_t d = 0; d < t.dim(); d++) TORCH_CHECK_VALUE(t.stride(d) != 0 || t.size(d) <= 1, what, ": an expanded tensor cannot be clipped in place");
            copies.emplace_back(i, t.contiguous());
            p = copies.back().second.data_ptr();
        }
        at_[i] = p;
        sizes[i] = t.numel();
        types[i] = row_type(t.scalar_type());
    }
    if (clip && !copies.empty()) refuse_shared_memory(tensors);        // (the library sees the copies' addresses)
    const c10::DeviceGuard guard(dev);
    const size_t bytes = iso_grad_norm_scratch_bytes(n, sizes.data());
    const auto opts = tensors[0].options().memory_format(std::nullopt);
    const Tensor scratch = at::empty({(int64_t)bytes}, opts.dtype(at::kByte)), out = at::empty({2}, opts.dtype(at::kFloat));
    check(iso_grad_norm(n, at_.data(), sizes.data(), types.data(), kind, (float)max_norm, clip, (float*)out.data_ptr(), scratch.data_ptr(), bytes, stream_on(dev)),
          "iso_grad_norm");
    if (clip) {
        for (const Tensor& t : tensors) t.unsafeGetTensorImpl()->bump_version();
        for (const auto& [i, c] : copies) tensors[i].copy_(c);
    }
    return out;
}
Tensor grad_norm(const std::vector<Tensor>& tensors, double norm_type, double max_norm, bool clip) { return norm_and_factor(tensors, norm_type, max_norm, clip)[0]; }
Tensor grad_norm_coef(const std::vector<Tensor>& tensors, double norm_type, double max_norm) { return norm_and_factor(tensors, norm_type, max_norm, false); }

}  // namespace

void bind_rows(pybind11::module_& m) {
    namespace py = pybind11;
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const LibraryError& e) {
            PyErr_SetString(py::module_::import("instascene_amd._lib").attr("IsrError").ptr(), e.what());
        }
    });
    m.def("rms_norm", &rms_norm);
    m.def("rms_norm_quantized", &rms_norm_quantized);
    m.def("rows8_write", &rows8_write);
    m.def("rows8_read", &rows8_read);
    m.def("grad_norm", &grad_norm);
    m.def("grad_norm_coef", &grad_norm_coef);
}
