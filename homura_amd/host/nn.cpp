// Front end of the operators of libhomura_nn: shapes, types and devices are checked here, outputs allocated, and what
// the entry points take as three dimensions is made of what users have.
#include "homura.hpp"

namespace homura {

namespace {

std::vector<int64_t> as_spec(const Shape &shape) { return std::vector<int64_t>(shape.begin(), shape.end()); }

void expect_rocm(const char *op, const Tensor &first, const std::vector<std::pair<const char *, const Tensor *>> &others) {
    if (first.device().kind != Device::K::Rocm) throw Error(std::string(op) + " runs on ROCm tensors only");
    for (const auto &[name, t] : others) {
        if (t && t->device() != first.device()) {
            throw Error(std::string(op) + " expects all tensors on " + first.device().str() + ", but " + name + " is on " + t->device().str());
        }
    }
}

void expect_float(const char *op, DType dtype) {
    if (!is_floating_point(dtype)) throw Error(std::string(op) + " is not implemented for " + name_of(dtype) + " tensors");
}

void expect_dtype(const char *op, const char *name, const Tensor &t, DType dtype, DType or_this) {
    if (t.dtype() == dtype || t.dtype() == or_this) return;
    std::string wants = name_of(dtype);
    if (or_this != dtype) wants += std::string(" or ") + name_of(or_this);
    throw Error(std::string(op) + " expects " + name + " to be " + wants + ", but got " + name_of(t.dtype()));
}

void expect_shape(const char *op, const char *name, const Tensor &t, const Shape &shape) {
    if (t.shape() == shape) return;
    throw Error(std::string(op) + " expects " + name + " of shape " + shape_str(shape) + ", but got " + shape_str(t.shape()));
}

const Tensor *ptr(const std::optional<Tensor> &t) { return t ? &*t : nullptr; }
const TensorData *data(const std::optional<Tensor> &t) { return t ? &t->data() : nullptr; }

DType wide(DType dtype) { return dtype == DType::F64 ? DType::F64 : DType::F32; }

int64_t product(const Shape &shape, size_t from, size_t to) {
    int64_t n = 1;
    for (size_t d = from; d < to; ++d) n *= shape[d];
    return n;
}

// The [B, T, C] view of sequences and the [B, C] view of states.
struct Batch {
    Shape shape, states;
    int64_t B, T, C;
    Tensor sequences(const Tensor &t) const { return t.reshape({B, T, C}); }
    Tensor state(const Tensor &t) const { return t.reshape({B, C}); }
    std::optional<Tensor> state(const std::optional<Tensor> &t) const {
        if (!t) return std::nullopt;
        return state(*t);
    }
};

Batch check_recurrence(const char *op, const Tensor &gate, const Tensor &input, const std::optional<Tensor> &initial,
                       const std::optional<Tensor> &lengths) {
    expect_rocm(op, input, {{"the gate", &gate}, {"the initial state", ptr(initial)}, {"lengths", ptr(lengths)}});
    expect_float(op, input.dtype());
    expect_dtype(op, "the gate", gate, input.dtype(), input.dtype());
    if (input.num_dims() < 2) throw Error(std::string(op) + " expects an input of at least two dimensions, but got " + shape_str(input.shape()));
    if (!is_expandable_to(gate.shape(), input.shape())) {
        throw Error(std::string(op) + " expects a gate that broadcasts to " + shape_str(input.shape()) + ", but got " + shape_str(gate.shape()));
    }
    Batch b;
    b.shape = input.shape();
    b.states = input.shape();
    b.states.erase(b.states.begin() + 1);
    b.B = b.shape[0], b.T = b.shape[1], b.C = product(b.shape, 2, b.shape.size());
    if (initial) {
        expect_shape(op, "an initial state", *initial, b.states);
        expect_dtype(op, "the initial state", *initial, input.dtype(), wide(input.dtype()));
    }
    if (lengths) {
        expect_shape(op, "lengths", *lengths, Shape{b.B});
        expect_dtype(op, "lengths", *lengths, DType::I32, DType::I64);
    }
    return b;
}

// The [N, S, C] view of maps.
struct MapsShape {
    int64_t N, S, C;
    Tensor maps(const Tensor &t) const { return t.reshape({N, S, C}); }
};

MapsShape check_norm(const char *op, const Tensor &x, int64_t groups, const std::optional<Tensor> &weight,
                     const std::optional<Tensor> &bias, std::optional<UnaryOp> activation) {
    expect_rocm(op, x, {{"the weight", ptr(weight)}, {"the bias", ptr(bias)}});
    expect_float(op, x.dtype());
    if (x.num_dims() < 2) throw Error(std::string(op) + " expects at least two dimensions, but got " + shape_str(x.shape()));
    const size_t last = x.num_dims() - 1;
    const MapsShape m{x.shape()[0], product(x.shape(), 1, last), x.shape()[last]};
    if (groups < 1 || m.C % groups != 0) {
        throw Error(std::string(op) + " expects the number of channels (" + std::to_string(m.C) + ") to be a multiple of the number of groups (" +
                    std::to_string(groups) + ")");
    }
    if (activation && *activation != UnaryOp::Relu && *activation != UnaryOp::Silu && *activation != UnaryOp::Gelu &&
        *activation != UnaryOp::GeluTanh) {
        throw Error(std::string(op) + " applies relu, silu, gelu or gelu_tanh");
    }
    const std::pair<const char *, const Tensor *> per_channel[2] = {{"the weight", ptr(weight)}, {"the bias", ptr(bias)}};
    for (const auto &[name, t] : per_channel) {
        if (!t) continue;
        expect_shape(op, name, *t, Shape{m.C});
        expect_dtype(op, name, *t, x.dtype(), wide(x.dtype()));
    }
    return m;
}

}  // namespace

RecurrenceStates linear_recurrence(const Tensor &gate, const Tensor &input, const std::optional<Tensor> &initial,
                                   const std::optional<Tensor> &lengths, bool sigmoid) {
    const Batch b = check_recurrence("linear_recurrence", gate, input, initial, lengths);
    Tensor out = Tensor::uninit_on({b.B, b.T, b.C}, input.dtype(), input.device());
    Tensor last = Tensor::uninit_on({b.B, b.C}, initial ? initial->dtype() : wide(input.dtype()), input.device());
    const std::optional<Tensor> from = b.state(initial);
    backend::recurrence(sigmoid, out.data(), last.data(), b.sequences(gate.expand(as_spec(b.shape))).data(), b.sequences(input).data(),
                        data(from), data(lengths));
    return {out.reshape(as_spec(b.shape)), last.reshape(as_spec(b.states))};
}

namespace grad {

Recurrence linear_recurrence(const std::optional<Tensor> &g, const std::optional<Tensor> &g_last, const Tensor &gate, const Tensor &input,
                             const Tensor &out, const std::optional<Tensor> &initial, const std::optional<Tensor> &lengths, bool sigmoid) {
    constexpr const char *op = "grad::linear_recurrence";
    const Batch b = check_recurrence(op, gate, input, initial, lengths);
    expect_rocm(op, input, {{"the output", &out}, {"its gradient", ptr(g)}, {"the last state's gradient", ptr(g_last)}});
    expect_shape(op, "the output", out, b.shape);
    expect_dtype(op, "the output", out, input.dtype(), input.dtype());
    if (g) {
        expect_shape(op, "the output's gradient", *g, b.shape);
        expect_dtype(op, "the output's gradient", *g, input.dtype(), input.dtype());
    }
    if (g_last) {
        expect_shape(op, "the last state's gradient", *g_last, b.states);
        expect_dtype(op, "the last state's gradient", *g_last, input.dtype(), wide(input.dtype()));
    }
    const Tensor dy = g ? *g : Tensor::full({1}, Scalar::of_float(0.0), input.dtype(), input.device()).expand(as_spec(b.shape));
    // A gate that was broadcast gets the sum of many gradients, which are rounded to its type once, after that.
    const bool shared = gate.shape() != b.shape;
    Tensor d_gate = Tensor::uninit_on({b.B, b.T, b.C}, shared ? wide(input.dtype()) : input.dtype(), input.device());
    Tensor d_input = Tensor::uninit_on({b.B, b.T, b.C}, input.dtype(), input.device());
    Tensor d_initial = Tensor::uninit_on({b.B, b.C}, initial ? initial->dtype() : wide(input.dtype()), input.device());
    const std::optional<Tensor> from = b.state(initial), from_last = b.state(g_last);
    backend::recurrence_backward(sigmoid, d_gate.data(), d_input.data(), d_initial.data(), b.sequences(dy).data(), data(from_last),
                                 b.sequences(gate.expand(as_spec(b.shape))).data(), b.sequences(input).data(), b.sequences(out).data(),
                                 data(from), data(lengths));
    d_gate = d_gate.reshape(as_spec(b.shape));
    if (shared) d_gate = d_gate.sum_to_size(gate.shape()).to(input.dtype());
    return {d_gate, d_input.reshape(as_spec(b.shape)), d_initial.reshape(as_spec(b.states))};
}

}  // namespace grad

NormOutput group_norm(const Tensor &x, int64_t groups, const std::optional<Tensor> &weight, const std::optional<Tensor> &bias, double eps,
                      std::optional<UnaryOp> activation) {
    const MapsShape m = check_norm("group_norm", x, groups, weight, bias, activation);
    Tensor out = Tensor::uninit_on({m.N, m.S, m.C}, x.dtype(), x.device());
    Tensor mean = Tensor::uninit_on({m.N, groups}, wide(x.dtype()), x.device());
    Tensor rstd = Tensor::uninit_on({m.N, groups}, wide(x.dtype()), x.device());
    backend::group_norm(out.data(), mean.data(), rstd.data(), m.maps(x).data(), data(weight), data(bias), groups, eps, activation);
    return {out.reshape(as_spec(x.shape())), mean, rstd};
}

namespace grad {

Norm group_norm(const Tensor &g, const Tensor &x, const Tensor &mean, const Tensor &rstd, int64_t groups, const std::optional<Tensor> &weight,
                const std::optional<Tensor> &bias, std::optional<UnaryOp> activation) {
    constexpr const char *op = "grad::group_norm";
    const MapsShape m = check_norm(op, x, groups, weight, bias, activation);
    expect_rocm(op, x, {{"the output's gradient", &g}, {"the mean", &mean}, {"rstd", &rstd}});
    expect_shape(op, "the output's gradient", g, x.shape());
    expect_dtype(op, "the output's gradient", g, x.dtype(), x.dtype());
    const std::pair<const char *, const Tensor *> statistics[2] = {{"the mean", &mean}, {"rstd", &rstd}};
    for (const auto &[name, t] : statistics) {
        expect_shape(op, name, *t, Shape{m.N, groups});
        expect_dtype(op, name, *t, wide(x.dtype()), wide(x.dtype()));
    }
    Tensor d_x = Tensor::uninit_on({m.N, m.S, m.C}, x.dtype(), x.device());
    Norm r;
    if (weight) r.d_weight = Tensor::uninit_on({m.C}, weight->dtype(), x.device());
    if (bias) r.d_bias = Tensor::uninit_on({m.C}, bias->dtype(), x.device());
    backend::group_norm_backward(d_x.data(), data(r.d_weight), data(r.d_bias), m.maps(g).data(), m.maps(x).data(), mean.data(), rstd.data(),
                                 data(weight), data(bias), groups, activation);
    r.d_x = d_x.reshape(as_spec(x.shape()));
    return r;
}

}  // namespace grad

namespace {

// Everything that can refuse a dropout; returns the residual broadcast to x.
std::optional<Tensor> check_dropout(const Tensor &x, double p, const std::optional<Tensor> &residual) {
    constexpr const char *op = "dropout";
    expect_rocm(op, x, {{"the residual", ptr(residual)}});
    expect_float(op, x.dtype());
    if (!(p >= 0.0 && p <= 1.0)) throw Error("dropout expects a probability between 0 and 1, but got " + Scalar::of_float(p).str());
    if (!residual) return std::nullopt;
    expect_dtype(op, "the residual", *residual, x.dtype(), x.dtype());
    if (!is_expandable_to(residual->shape(), x.shape())) {
        throw Error("dropout expects a residual that broadcasts to " + shape_str(x.shape()) + ", but got " + shape_str(residual->shape()));
    }
    return residual->expand(as_spec(x.shape()));
}

}  // namespace

Tensor dropout_with(const Tensor &x, const DropoutMask &mask, const std::optional<Tensor> &residual) {
    const std::optional<Tensor> onto = check_dropout(x, mask.p, residual);
    Tensor out = Tensor::uninit_on(x.shape(), x.dtype(), x.device());
    backend::dropout(out.data(), x.data(), data(onto), mask);
    return out;
}

DropoutOutput dropout(const Tensor &x, double p, const std::optional<Tensor> &residual) {
    check_dropout(x, p, residual);  // first, so that a refused call leaves the generator where it was
    DropoutMask mask{p, 0, 0};
    const uint64_t n = static_cast<uint64_t>(x.num_elements());
    reserve_random_blocks(n / 4 + (n % 4 != 0), mask.seed, mask.offset);
    return {dropout_with(x, mask, residual), mask};
}

namespace grad {

Tensor dropout(const Tensor &g, const DropoutMask &mask) { return dropout_with(g, mask, std::nullopt); }

}  // namespace grad

}  // namespace homura
