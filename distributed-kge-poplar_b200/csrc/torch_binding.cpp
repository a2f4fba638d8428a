// The operators on device arrays for torch tensors: checks of types, shapes and strides, torch's allocator and current stream.
//
// A call's work on the GPU takes a few microseconds when it is small, so that what the host does for it counts: the same checks
// and allocations in Python took 20 to 25 us a call, here they take 3 to 5.
#include <torch/extension.h>

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <limits>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "kge_b200.h"

namespace py = pybind11;
using at::Tensor;
using OptionalTensor = std::optional<Tensor>;

namespace {

std::string text(const std::string& s) { return s; }
std::string text(c10::Device d) { return d.str(); }
std::string text(int64_t v) { return std::to_string(v); }
std::string text(size_t v) { return std::to_string(v); }
std::string text(at::IntArrayRef shape) {
    std::string s = "[";
    for (size_t i = 0; i < shape.size(); ++i) s += (i ? ", " : "") + std::to_string(shape[i]);
    return s + "]";
}
template <class... Parts>
[[noreturn]] void refuse(const Parts&... parts) {
    throw py::value_error((text(parts) + ...));
}
void check(int status) {
    if (status == KGE_OK) return;
    const char* const text = kge_last_error(nullptr);
    if (status == KGE_INVALID_ARGUMENT) throw py::value_error(text);
    throw std::runtime_error(text);
}

constexpr int kNoType = -1;
int float_type(at::ScalarType t) {
    return t == at::kFloat ? KGE_F32 : t == at::kHalf ? KGE_F16 : t == at::kBFloat16 ? KGE_BF16 : kNoType;
}
std::string type_name(at::ScalarType t) { return py::str(py::cast(t)); }
void must_be_float(const char* what, at::ScalarType t) {
    if (float_type(t) == kNoType) refuse(what, " must be torch.float32 or torch.float16 or torch.bfloat16, not ", type_name(t));
}
void must_be_on_gpu(const char* what, const Tensor& t) {
    if (!t.is_cuda()) refuse(what, " must be on a GPU, not on ", t.device());
}
void must_be_with(const char* what, const Tensor& t, c10::Device device) {
    must_be_on_gpu(what, t);
    if (t.device() != device) refuse(what, " is on ", t.device(), ", the other tensors on ", device);
}
void must_have_shape(const char* what, const Tensor& t, at::IntArrayRef shape) {
    if (t.sizes() != shape) refuse(what, " has shape ", t.sizes(), ", expected ", shape);
}
void must_be_matrix(const char* what, const Tensor& t) {
    if (t.dim() != 2) refuse(what, " must have two dimensions, not ", t.dim());
    if (t.size(1) > 1 && t.stride(1) != 1) refuse(what, " must be contiguous along its rows, not ", t.stride(1), " apart");
}
// The row stride; that of a single row or of none says nothing.
long long rows_apart(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

std::pair<uintptr_t, uintptr_t> span(const Tensor& t) {
    const uintptr_t first = reinterpret_cast<uintptr_t>(t.data_ptr());
    int64_t last = 0;
    for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
    return {first, first + (uintptr_t)(last + 1) * t.element_size()};
}
// What is written must not be what is read beside it.  `b` undefined or either empty: nothing to say.
void must_not_overlap(const char* what_a, const Tensor& a, const char* what_b, const Tensor& b) {
    if (!b.defined() || a.numel() == 0 || b.numel() == 0) return;
    const auto [a_first, a_end] = span(a);
    const auto [b_first, b_end] = span(b);
    if (a_first < b_end && b_first < a_end) refuse(what_a, " and ", what_b, " overlap in memory");
}
void must_not_overlap(const char* what_a, const Tensor& a, const char* what_b, const OptionalTensor& b) {
    if (b) must_not_overlap(what_a, a, what_b, *b);
}
void* stream_of(c10::Device device) { return c10::cuda::getCurrentCUDAStream(device.index()).stream(); }

// ---------------------------------------------------------------------------

// All results of a row in one allocation: [rows, 4] state, log_prob, entropy, log_sum, lists.
struct LogProbs {
    Tensor memory;
    OptionalTensor target, mask, count;
    double scale;
    int64_t rows, cols, n_best;
    int64_t at_log_prob() const { return 4 * rows; }
    int64_t at_entropy() const { return 5 * rows; }
    int64_t at_log_sum() const { return 6 * rows; }
    int64_t at_best() const { return 7 * rows; }
    int64_t at_index() const { return (7 + n_best) * rows; }
    float* at(int64_t offset) const { return memory.data_ptr<float>() + offset; }
    Tensor vector(int64_t offset) const { return memory.as_strided({rows}, {1}, offset); }
    Tensor matrix(int64_t offset) const { return memory.as_strided({rows, n_best}, {n_best, 1}, offset); }
};

kge_scores scores_of(const Tensor& x, const OptionalTensor& target, const OptionalTensor& mask, const OptionalTensor& count, double scale) {
    must_be_float("scores", x.scalar_type());
    must_be_on_gpu("scores", x);
    must_be_matrix("scores", x);
    const int64_t rows = x.size(0), cols = x.size(1);
    kge_scores s{};
    s.x = x.data_ptr();
    s.float_type = float_type(x.scalar_type());
    s.rows = (size_t)rows;
    s.cols = (size_t)cols;
    s.row_stride = rows_apart(x);
    s.scale = (float)scale;
    const auto indices = [&](const char* what, const OptionalTensor& t) -> const int32_t* {
        if (!t) return nullptr;
        if (t->scalar_type() != at::kInt) refuse(what, " must be torch.int32, not ", type_name(t->scalar_type()));
        must_be_with(what, *t, x.device());
        must_have_shape(what, *t, {rows});
        if (rows > 1 && t->stride(0) != 1) refuse(what, " must be contiguous");
        return t->data_ptr<int32_t>();
    };
    s.target = indices("target", target);
    s.count = indices("count", count);
    if (mask) {
        if (mask->scalar_type() != at::kBool && mask->scalar_type() != at::kByte) refuse("mask must be torch.bool or torch.uint8, not ", type_name(mask->scalar_type()));
        must_be_with("mask", *mask, x.device());
        must_have_shape("mask", *mask, {rows, cols});
        must_be_matrix("mask", *mask);
        s.mask = static_cast<const uint8_t*>(mask->data_ptr());
        s.mask_stride = rows > 1 ? mask->stride(0) : cols;
    }
    return s;
}

LogProbs log_probs(const Tensor& scores, const OptionalTensor& target, const OptionalTensor& mask, const OptionalTensor& count, double scale, int64_t n_best) {
    if (n_best < 0 || n_best > 128) refuse("n_best must be between 0 and 128, not ", n_best);
    const kge_scores s = scores_of(scores, target, mask, count, scale);
    const c10::cuda::CUDAGuard guard(scores.device());
    const int64_t rows = scores.size(0);
    const size_t wanted = kge_op_log_probs_workspace(s.rows, s.cols, (size_t)n_best);
    LogProbs r{at::empty({rows * (7 + 2 * n_best)}, scores.options().dtype(at::kFloat)), target, mask, count, scale, rows, scores.size(1), n_best};
    kge_log_probs_out out{};
    out.row_state = r.at(0);
    out.log_prob = r.at(r.at_log_prob());
    out.entropy = r.at(r.at_entropy());
    out.log_sum = r.at(r.at_log_sum());
    out.n_best = (size_t)n_best;
    out.best_log_prob = r.at(r.at_best());
    out.best_index = reinterpret_cast<int32_t*>(r.at(r.at_index()));
    Tensor workspace;
    if (wanted) workspace = at::empty({(int64_t)wanted}, scores.options().dtype(at::kByte));
    check(kge_op_log_probs(&s, &out, wanted ? workspace.data_ptr() : nullptr, wanted, stream_of(scores.device())));
    return r;
}

Tensor log_probs_grad(const Tensor& scores, const LogProbs& r, const OptionalTensor& grad_log_prob, const OptionalTensor& grad_entropy,
                      const OptionalTensor& grad_best, const OptionalTensor& out_given) {
    const kge_scores s = scores_of(scores, r.target, r.mask, r.count, r.scale);
    if (scores.size(0) != r.rows || scores.size(1) != r.cols) refuse("scores have shape ", scores.sizes(), ", the result is of [", r.rows, ", ", r.cols, "]");
    must_be_with("result", r.memory, scores.device());
    const c10::cuda::CUDAGuard guard(scores.device());
    const auto grads = [&](const char* what, const OptionalTensor& g, at::IntArrayRef shape) -> Tensor {
        if (!g) return Tensor();
        if (g->scalar_type() != at::kFloat) refuse(what, " must be torch.float32, not ", type_name(g->scalar_type()));
        must_be_with(what, *g, scores.device());
        must_have_shape(what, *g, shape);
        return g->contiguous();
    };
    const Tensor a = grads("grad_log_prob", grad_log_prob, {r.rows}), b = grads("grad_entropy", grad_entropy, {r.rows}),
                 c = grads("grad_best", grad_best, {r.rows, r.n_best});
    Tensor out;
    if (out_given) {
        out = *out_given;
        if (out.scalar_type() != scores.scalar_type()) refuse("out must be ", type_name(scores.scalar_type()), ", not ", type_name(out.scalar_type()));
        must_be_with("out", out, scores.device());
        must_have_shape("out", out, scores.sizes());
        must_be_matrix("out", out);
        if (out.data_ptr() != scores.data_ptr() || rows_apart(out) != rows_apart(scores)) must_not_overlap("out", out, "scores", scores);
        must_not_overlap("out", out, "the result", r.memory);
        must_not_overlap("out", out, "target", r.target);
        must_not_overlap("out", out, "mask", r.mask);
        must_not_overlap("out", out, "count", r.count);
        must_not_overlap("out", out, "grad_log_prob", a);
        must_not_overlap("out", out, "grad_entropy", b);
        must_not_overlap("out", out, "grad_best", c);
        out.unsafeGetTensorImpl()->bump_version();
    } else {
        out = at::empty(scores.sizes(), scores.options());
    }
    const auto pointer = [](const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; };
    check(kge_op_log_probs_grad(&s, r.at(0), pointer(a), pointer(b), (size_t)r.n_best, reinterpret_cast<const int32_t*>(r.at(r.at_index())), pointer(c),
                                out.data_ptr(), rows_apart(out), stream_of(scores.device())));
    return out;
}

// ---------------------------------------------------------------------------

struct Rows8 {
    Tensor values, exponents;
    int64_t rows, cols;
};

Rows8 quantise_rows(const Tensor& x, bool transposed) {
    must_be_float("x", x.scalar_type());
    must_be_on_gpu("x", x);
    must_be_matrix("x", x);
    const c10::cuda::CUDAGuard guard(x.device());
    const int64_t rows = x.size(transposed ? 1 : 0), cols = x.size(transposed ? 0 : 1);
    size_t values = 0, exponents = 0;
    check(kge_op_rows8_bytes((size_t)rows, (size_t)cols, &values, &exponents));
    const auto bytes = x.options().dtype(at::kByte);
    Rows8 r{at::empty({rows, rows ? (int64_t)values / rows : 0}, bytes), at::empty({(int64_t)exponents}, bytes), rows, cols};
    check(kge_op_quantise_rows(x.data_ptr(), float_type(x.scalar_type()), (size_t)x.size(0), (size_t)x.size(1), rows_apart(x), transposed,
                               r.values.data_ptr<uint8_t>(), r.exponents.data_ptr<uint8_t>(), stream_of(x.device())));
    return r;
}

Tensor product8(const Rows8& a, const Rows8& b, at::ScalarType dtype, const OptionalTensor& out_given) {
    if (a.cols != b.cols) refuse("rows of ", a.cols, " and of ", b.cols, " values");
    const c10::Device device = a.values.device();
    if (b.values.device() != device) refuse("a is on ", device, ", b on ", b.values.device());
    const c10::cuda::CUDAGuard guard(device);
    Tensor out;
    if (out_given) {
        out = *out_given;
        must_be_float("out", out.scalar_type());
        must_be_with("out", out, device);
        must_have_shape("out", out, {a.rows, b.rows});
        must_be_matrix("out", out);
        must_not_overlap("out", out, "a", a.values);
        must_not_overlap("out", out, "a", a.exponents);
        must_not_overlap("out", out, "b", b.values);
        must_not_overlap("out", out, "b", b.exponents);
        out.unsafeGetTensorImpl()->bump_version();
    } else {
        must_be_float("dtype", dtype);
        out = at::empty({a.rows, b.rows}, a.values.options().dtype(dtype));
    }
    const size_t wanted = kge_op_product8_workspace((size_t)a.rows, (size_t)b.rows, (size_t)a.cols);
    Tensor workspace;
    if (wanted) workspace = at::empty({(int64_t)wanted}, a.values.options());
    check(kge_op_product8(a.values.data_ptr<uint8_t>(), a.exponents.data_ptr<uint8_t>(), (size_t)a.rows, b.values.data_ptr<uint8_t>(),
                          b.exponents.data_ptr<uint8_t>(), (size_t)b.rows, (size_t)a.cols, out.data_ptr(), float_type(out.scalar_type()), rows_apart(out),
                          wanted ? workspace.data_ptr() : nullptr, wanted, stream_of(device)));
    return out;
}

// ---------------------------------------------------------------------------

// The tensors of an optimiser and their moments' places.
struct AdamWTensors {
    std::vector<Tensor> params;
    std::vector<kge_adamw_tensor> table;
    std::vector<int64_t> first, sizes;
    std::vector<size_t> order;  // of those that are not empty, by where they lay
    at::ScalarType type;
    int64_t total = 0;

    explicit AdamWTensors(std::vector<Tensor> given) : params(std::move(given)) {
        if (params.empty()) refuse("AdamW needs at least one tensor");
        type = params[0].scalar_type();
        std::vector<std::tuple<uintptr_t, uintptr_t, size_t>> spans;
        for (size_t i = 0; i < params.size(); ++i) {
            const Tensor& p = params[i];
            const std::string what = "parameter " + std::to_string(i);
            if (p.scalar_type() != at::kFloat && p.scalar_type() != at::kBFloat16)
                refuse(what, " must be torch.float32 or torch.bfloat16, not ", type_name(p.scalar_type()));
            must_be_on_gpu(what.c_str(), p);
            if (i) must_be_with(what.c_str(), p, params[0].device());
            if (p.scalar_type() != type) refuse(what, " is ", type_name(p.scalar_type()), ", parameter 0 ", type_name(type), ": an optimiser for each type");
            if (!p.is_contiguous()) refuse(what, " must be contiguous");
            if (p.numel()) {
                const auto [begin, end] = span(p);
                spans.emplace_back(begin, end, i);
            }
            table.push_back(kge_adamw_tensor{nullptr, nullptr, 0, (size_t)total});
            first.push_back(total);
            sizes.push_back(p.numel());
            total += (p.numel() + 127) / 128 * 128;
        }
        std::sort(spans.begin(), spans.end());
        refuse_neighbours(spans);
        for (const auto& s : spans) order.push_back(std::get<2>(s));
    }

    // The parameters of a step may not overlap one another (their memory may have been replaced) nor its gradients.  They are gone through
    // in the order that they lay in at first; one that has moved costs a sort.
    void must_not_meet(size_t grad_bytes) const {
        std::vector<std::tuple<uintptr_t, uintptr_t, size_t>> spans;
        for (const size_t i : order)
            if (table[i].size) {
                const auto first = reinterpret_cast<uintptr_t>(table[i].param);
                spans.emplace_back(first, first + table[i].size * params[i].element_size(), i);
            }
        if (!std::is_sorted(spans.begin(), spans.end())) std::sort(spans.begin(), spans.end());
        refuse_neighbours(spans);
        for (size_t i = 0; i < table.size(); ++i) {
            if (!table[i].size) continue;
            const auto first = reinterpret_cast<uintptr_t>(table[i].grad), end = first + table[i].size * grad_bytes;
            const auto next = std::lower_bound(spans.begin(), spans.end(), end, [](const auto& s, uintptr_t at) { return std::get<0>(s) < at; });
            if (next != spans.begin() && std::get<1>(*std::prev(next)) > first) refuse("gradient ", i, " and parameter ", std::get<2>(*std::prev(next)), " overlap in memory");
        }
    }
    static void refuse_neighbours(const std::vector<std::tuple<uintptr_t, uintptr_t, size_t>>& spans) {
        for (size_t i = 1; i < spans.size(); ++i)
            if (std::get<0>(spans[i]) < std::get<1>(spans[i - 1])) refuse("parameters ", std::get<2>(spans[i - 1]), " and ", std::get<2>(spans[i]), " overlap in memory");
    }

    void step(const std::vector<OptionalTensor>& grads, int state_bits, const Tensor& adam_m, const Tensor& adam_v, const OptionalTensor& m_exponent,
              const OptionalTensor& v_exponent, double beta_m, double beta_v, double epsilon, double grad_scale, double decay, double step_size,
              double inv_sqrt_correction, uint32_t key, const OptionalTensor& schedule) {
        if (grads.size() != params.size()) refuse(grads.size(), " gradients for ", params.size(), " parameters");
        const c10::Device device = adam_m.device();
        const auto must_be_moments = [&](const char* what, const Tensor& t, at::ScalarType kind, int64_t size) {
            must_be_with(what, t, device);
            if (t.scalar_type() != kind) refuse(what, " must be ", type_name(kind), ", not ", type_name(t.scalar_type()));
            must_have_shape(what, t, {size});
            if (!t.is_contiguous()) refuse(what, " must be contiguous");
        };
        must_be_moments("adam_m", adam_m, state_bits == 8 ? at::kByte : at::kFloat, total);
        must_be_moments("adam_v", adam_v, state_bits == 8 ? at::kByte : at::kFloat, total);
        if (state_bits == 8 && !(m_exponent && v_exponent)) refuse("moments in 8 bits have exponents");
        if (m_exponent) must_be_moments("m_exponent", *m_exponent, at::kByte, total / 128);
        if (v_exponent) must_be_moments("v_exponent", *v_exponent, at::kByte, total / 128);
        std::optional<at::ScalarType> grad_type;
        for (size_t i = 0; i < grads.size(); ++i) {
            table[i].size = 0;
            if (!grads[i]) continue;
            const Tensor &g = *grads[i], &p = params[i];
            // what a tensor holds may have been replaced since the optimiser was made
            if (p.device() != device || p.scalar_type() != type || p.numel() != sizes[i] || !p.is_contiguous())
                refuse("parameter ", i, " is no longer ", sizes[i], " contiguous values of ", type_name(type), " on ", device);
            if (!grad_type) {
                must_be_float("gradients", g.scalar_type());
                grad_type = g.scalar_type();
            }
            if (g.scalar_type() != *grad_type) refuse("gradient ", i, " is ", type_name(g.scalar_type()), ", others ", type_name(*grad_type));
            if (g.device() != device) refuse("gradient ", i, " is on ", g.device(), ", the parameters on ", device);
            if (g.sizes() != p.sizes()) refuse("gradient ", i, " has shape ", g.sizes(), ", its parameter ", p.sizes());
            if (!g.is_contiguous()) refuse("gradient ", i, " must be contiguous");
            table[i].param = p.data_ptr();
            table[i].grad = g.data_ptr();
            table[i].size = (size_t)p.numel();
        }
        if (!grad_type) return;
        kge_adamw_args a{};
        a.param_type = float_type(type);
        a.grad_type = float_type(*grad_type);
        a.state_bits = state_bits;
        a.adam_m = adam_m.data_ptr();
        a.adam_v = adam_v.data_ptr();
        if (m_exponent) a.m_exponent = m_exponent->data_ptr<uint8_t>();
        if (v_exponent) a.v_exponent = v_exponent->data_ptr<uint8_t>();
        a.beta_m = beta_m, a.beta_v = beta_v, a.epsilon = epsilon, a.grad_scale = grad_scale;
        a.decay = decay, a.step_size = step_size, a.inv_sqrt_correction = inv_sqrt_correction, a.key = key;
        if (schedule) {
            if (schedule->scalar_type() != at::kFloat) refuse("schedule must be torch.float32, not ", type_name(schedule->scalar_type()));
            must_be_with("schedule", *schedule, device);
            must_have_shape("schedule", *schedule, {4});
            if (!schedule->is_contiguous()) refuse("schedule must be contiguous");
            a.schedule = schedule->data_ptr<float>();
        }
        must_not_meet(c10::elementSize(*grad_type));
        // as any operator that writes in place tells autograd; it may refuse (tensors of inference mode), so it comes first
        for (size_t i = 0; i < params.size(); ++i)
            if (table[i].size) params[i].unsafeGetTensorImpl()->bump_version();
        const c10::cuda::CUDAGuard guard(device);
        check(kge_op_adamw(&a, table.data(), table.size(), stream_of(device)));
    }
};

std::pair<Tensor, Tensor> adamw_moments(const Tensor& adam_m, const Tensor& m_exponent, const Tensor& adam_v, const Tensor& v_exponent) {
    // what an optimiser holds may have been replaced since it was made
    const int64_t size = adam_m.numel();
    const auto must_be = [&](const char* what, const Tensor& t, int64_t n) {
        if (t.scalar_type() != at::kByte) refuse(what, " must be torch.uint8, not ", type_name(t.scalar_type()));
        must_have_shape(what, t, {n});
        if (!t.is_contiguous()) refuse(what, " must be contiguous");
    };
    must_be("m_exponent", m_exponent, size / 128);
    must_be("v_exponent", v_exponent, size / 128);
    must_be("adam_v", adam_v, size);
    must_be("adam_m", adam_m, size);
    must_be_with("m_exponent", m_exponent, adam_m.device());
    must_be_with("v_exponent", v_exponent, adam_m.device());
    must_be_with("adam_v", adam_v, adam_m.device());
    const c10::cuda::CUDAGuard guard(adam_m.device());
    const auto type = adam_m.options().dtype(at::kBFloat16);
    Tensor m = at::empty(adam_m.sizes(), type), v = at::empty(adam_m.sizes(), type);
    check(kge_op_adamw_moments(adam_m.data_ptr<uint8_t>(), m_exponent.data_ptr<uint8_t>(), adam_v.data_ptr<uint8_t>(), v_exponent.data_ptr<uint8_t>(),
                               (size_t)adam_m.numel(), m.data_ptr(), v.data_ptr(), stream_of(adam_m.device())));
    return {m, v};
}

}  // namespace

PYBIND11_MODULE(libkge_torch, m) {
    py::class_<LogProbs>(m, "LogProbs",
                         "What log_probs found, and what log_probs_grad needs of it.\n\n"
                         "log_prob       [rows]          of the target: 0 where there is none, -inf where it is not live\n"
                         "entropy        [rows]          of the distribution over the live columns, 0 where there are none\n"
                         "log_sum        [rows]          log of the sum of exp(scale * score), -inf where no column is live\n"
                         "best_log_prob  [rows, n_best]  highest score first, equal scores by the lower column, -inf past the live columns\n"
                         "best_index     [rows, n_best]  int32, -1 past the live columns\n\n"
                         "All are views of one allocation.")
        .def_property_readonly("log_prob", [](const LogProbs& r) { return r.vector(r.at_log_prob()); })
        .def_property_readonly("entropy", [](const LogProbs& r) { return r.vector(r.at_entropy()); })
        .def_property_readonly("log_sum", [](const LogProbs& r) { return r.vector(r.at_log_sum()); })
        .def_property_readonly("best_log_prob", [](const LogProbs& r) { return r.matrix(r.at_best()); })
        .def_property_readonly("best_index", [](const LogProbs& r) { return r.matrix(r.at_index()).view(at::kInt); })
        .def_readonly("target", &LogProbs::target)
        .def_readonly("mask", &LogProbs::mask)
        .def_readonly("count", &LogProbs::count)
        .def_readonly("scale", &LogProbs::scale);
    m.def("log_probs", &log_probs);
    m.def("log_probs_grad", &log_probs_grad);
    py::class_<Rows8>(m, "Rows8",
                      "rows x cols values in 8-bit floating point with a power of two for each 128 values along a row (values, exponents), laid\n"
                      "out as kge_op_quantise_rows states.  One byte and 1/128 a value.")
        .def_readonly("values", &Rows8::values)
        .def_readonly("exponents", &Rows8::exponents)
        .def_readonly("rows", &Rows8::rows)
        .def_readonly("cols", &Rows8::cols);
    m.def("quantise_rows", &quantise_rows);
    m.def("product8", &product8);
    py::class_<AdamWTensors>(m, "AdamWTensors")
        .def(py::init<std::vector<Tensor>>())
        .def_readonly("first", &AdamWTensors::first)
        .def_readonly("total", &AdamWTensors::total)
        .def("step", &AdamWTensors::step);
    m.def("adamw_moments", &adamw_moments);
    m.def("adamw_key", &kge_op_adamw_key);
}
