// hmn_recurrence and hmn_recurrence_backward: h_t = a_t h_{t-1} + b_t along the sequences of a [B, T, C] batch.
#include "nn_recurrence.hpp"

namespace hmr {
namespace nn {
namespace {

// ---- one thread per channel ----------------------------------------------------------------------------------
//
// Decoding and other sequences of a few steps: nothing to fold, one launch, the states in registers ([64, 1, 4096] bf16 takes
// 3.5 us, of which the memory would take one). Also steps so far apart that a tile of the scan spans more than its 32-bit
// offsets (a million elements of 16 bits: time-major batches with as many channels in all, which keep the memory busy a
// thread each). `last` may be `initial`: a channel's state is read and written by its own thread.

template <class T, int FORM>
__global__ void __launch_bounds__(kBlock) forward_kernel(RecurrenceArgs a) {
    using C = typename Comp<T>::C;
    const int64_t chains = a.B * a.C;
    for (int64_t k = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; k < chains; k += static_cast<int64_t>(gridDim.x) * kBlock) {
        const int64_t b = k / a.C, c = k - b * a.C;
        const int64_t steps = a.steps(b);
        C h = a.entry.p != nullptr ? load_state<T>(a.entry.p, a.entry.at(b, c), a.entry.wide) : C(0);
        for (int64_t t = 0; t < a.T; ++t) {
            C f, u, y = 0;
            if (t < steps) {
                factor_and_input<T, FORM>(Comp<T>::up(a.gate.template get<T>(b, t, c)), Comp<T>::up(a.input.template get<T>(b, t, c)), f, u);
                y = h = fma_(f, h, u);
            }
            a.out.template put<T>(b, t, c, Comp<T>::down(y));
        }
        if (a.exit.p != nullptr) store_state<T>(a.exit.p, a.exit.at(b, c), a.exit.wide, h);
    }
}

template <class T, int FORM>
__global__ void __launch_bounds__(kBlock) backward_kernel(RecurrenceArgs a) {
    using C = typename Comp<T>::C;
    const int64_t chains = a.B * a.C;
    for (int64_t k = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; k < chains; k += static_cast<int64_t>(gridDim.x) * kBlock) {
        const int64_t b = k / a.C, c = k - b * a.C;
        const int64_t steps = a.steps(b);
        C e = a.entry.p != nullptr ? load_state<T>(a.entry.p, a.entry.at(b, c), a.entry.wide) : C(0);
        for (int64_t t = a.T - 1; t >= 0; --t) {
            C dg = 0, dx = 0;
            if (t < steps) {
                const C z = Comp<T>::up(a.gate.template get<T>(b, t, c)), x = FORM == HMN_GATE_SIGMOID ? Comp<T>::up(a.input.template get<T>(b, t, c)) : C(0);
                const C g = Comp<T>::up(a.grad.template get<T>(b, t, c)) + e;
                C before = 0;
                if (t > 0) before = Comp<T>::up(a.state.template get<T>(b, t - 1, c));
                else if (a.initial.p != nullptr) before = load_state<T>(a.initial.p, a.initial.at(b, c), a.initial.wide);
                e = step_back<T, FORM>(z, x, g, before, dg, dx);
            }
            store_state<T>(a.d_gate.p, a.d_gate.at(b, t, c), a.d_gate_wide, dg);
            a.d_input.template put<T>(b, t, c, Comp<T>::down(dx));
        }
        if (a.exit.p != nullptr) store_state<T>(a.exit.p, a.exit.at(b, c), a.exit.wide, e);
    }
}

// ---- checks ----------------------------------------------------------------------------------------------------

struct Named {
    const char *name;
    const hmr_tensor_desc *d;
    bool output;
};

hmr_status check_batch(const char *who, int32_t form, const hmr_tensor_desc *gate, std::initializer_list<Named> sequences,
                       std::initializer_list<Named> states, const hmr_tensor_desc *lengths) {
    if (form != HMN_GATE_FACTOR && form != HMN_GATE_SIGMOID) return refuse(who, "unknown form " + std::to_string(form));
    if (gate == nullptr) return refuse(who, "gate is NULL");
    if (hmr_status s = check_operand(who, "gate", gate, 3, gate->sizes, false)) return s;
    if (!is_float(gate->dtype)) return refuse(who, "a recurrence takes floating point tensors");
    for (const Named &x : sequences) {
        if (hmr_status s = check_operand(who, x.name, x.d, 3, gate->sizes, x.output)) return s;
        if (x.d->dtype != gate->dtype) return refuse(who, std::string(x.name) + " has another dtype than gate");
    }
    const int64_t state_sizes[2] = {gate->sizes[0], gate->sizes[2]};
    for (const Named &x : states) {
        if (x.d == nullptr) continue;
        if (hmr_status s = check_operand(who, x.name, x.d, 2, state_sizes, x.output)) return s;
        if (hmr_status s = check_type(who, x.name, x.d->dtype, gate->dtype, wide_type(gate->dtype))) return s;
    }
    if (lengths != nullptr) {
        if (hmr_status s = check_operand(who, "lengths", lengths, 1, gate->sizes, false)) return s;
        if (lengths->dtype != HMR_I32 && lengths->dtype != HMR_I64) return refuse(who, "lengths are I32 or I64");
    }
    return HMR_OK;
}

Sequences sequences_of(const hmr_tensor_desc *d) {
    if (d == nullptr) return Sequences{};
    return Sequences{first(*d), d->strides[0], d->strides[1], d->strides[2]};
}
States states_of(const hmr_tensor_desc *d) {
    if (d == nullptr) return States{};
    return States{first(*d), d->strides[0], d->strides[1], d->dtype == HMR_F32};
}

RecurrenceArgs batch_args(const hmr_tensor_desc *gate, const hmr_tensor_desc *lengths) {
    RecurrenceArgs a{};
    a.B = gate->sizes[0], a.T = gate->sizes[1], a.C = gate->sizes[2];
    a.gate = sequences_of(gate);
    if (lengths != nullptr) a.lengths = first(*lengths), a.lengths_stride = lengths->strides[0], a.lengths64 = lengths->dtype == HMR_I64;
    return a;
}

ScanLayout layout_of(std::initializer_list<const hmr_tensor_desc *> operands) {
    ScanLayout layout{true, true};
    for (const hmr_tensor_desc *d : operands) {
        const int64_t size = dtype_size(d->dtype);
        layout.adjacent = layout.adjacent && d->strides[2] == 1;
        layout.whole_lines = layout.whole_lines && reinterpret_cast<uintptr_t>(first(*d)) % 128 == 0 && d->strides[0] * size % 128 == 0 &&
                             d->strides[1] * size % 128 == 0;
    }
    return layout;
}

// Whether a tile of the scan's largest shape spans less than 2^31 bytes in every operand.
bool near_by(std::initializer_list<const hmr_tensor_desc *> operands) {
    for (const hmr_tensor_desc *d : operands) {
        const int64_t most = (int64_t{1} << 30) / dtype_size(d->dtype);
        if (d->strides[1] > most / (kMostSteps + 1) || d->strides[2] > most / kMostChannels) return false;
    }
    return true;
}

// Without a step there is only the state to hand over; without anyone who wants it nothing, however many sequences there are.
bool nothing_to_write(const RecurrenceArgs &a) { return a.B == 0 || a.C == 0 || (a.T == 0 && a.exit.p == nullptr); }

uint32_t grid_of(hmr_context_t ctx, const RecurrenceArgs &a) {
    const int64_t groups = (a.B * a.C + kBlock - 1) / kBlock, most = int64_t{64} * ctx->compute_units;
    return static_cast<uint32_t>(groups < most ? groups : most);
}

hmr_status forward(hmr_context_t ctx, int32_t form, const hmr_tensor_desc *out, const hmr_tensor_desc *last,
                   const hmr_tensor_desc *gate, const hmr_tensor_desc *input, const hmr_tensor_desc *initial,
                   const hmr_tensor_desc *lengths, void *workspace, int64_t workspace_bytes) {
    constexpr const char *who = "hmn_recurrence";
    if (hmr_status s = check_batch(who, form, gate, {{"out", out, true}, {"input", input, false}},
                                   {{"last", last, true}, {"initial", initial, false}}, lengths)) {
        return s;
    }
    RecurrenceArgs a = batch_args(gate, lengths);
    a.input = sequences_of(input), a.out = sequences_of(out), a.entry = states_of(initial), a.exit = states_of(last);
    if (hmr_status s = check_room(who, workspace, workspace_bytes, room_for(gate))) return s;
    if (ctx == nullptr) return refuse(who, "null context");
    if (nothing_to_write(a)) return HMR_OK;
    return queue_on(ctx, who, [&](hipStream_t stream) {
        return with_float_type(gate->dtype, [&](auto tag) {
            using T = typename decltype(tag)::type;
            const ScanLayout layout = layout_of({gate, input, out});
            if ((scan_used(gate) || short_scan_used(gate, layout, false)) && near_by({gate, input, out})) {
                queue_scan_forward(stream, gate->dtype, form, a, layout, workspace);
                return;
            }
            with_code(form, std::integer_sequence<int, HMN_GATE_FACTOR, HMN_GATE_SIGMOID>{}, [&](auto f) {
                forward_kernel<T, decltype(f)::value><<<grid_of(ctx, a), kBlock, 0, stream>>>(a);
            });
        });
    });
}

hmr_status backward(hmr_context_t ctx, int32_t form, const hmr_tensor_desc *d_gate, const hmr_tensor_desc *d_input,
                    const hmr_tensor_desc *d_initial, const hmr_tensor_desc *grad, const hmr_tensor_desc *grad_last,
                    const hmr_tensor_desc *gate, const hmr_tensor_desc *input, const hmr_tensor_desc *out,
                    const hmr_tensor_desc *initial, const hmr_tensor_desc *lengths, void *workspace, int64_t workspace_bytes) {
    constexpr const char *who = "hmn_recurrence_backward";
    // The factor form's gradients do not need its input.
    if (form == HMN_GATE_FACTOR && input == nullptr) input = gate;
    if (hmr_status s = check_batch(who, form, gate,
                                   {{"d_input", d_input, true}, {"grad", grad, false}, {"input", input, false}, {"out", out, false}},
                                   {{"d_initial", d_initial, true}, {"grad_last", grad_last, false}, {"initial", initial, false}},
                                   lengths)) {
        return s;
    }
    if (hmr_status s = check_operand(who, "d_gate", d_gate, 3, gate->sizes, true)) return s;
    if (hmr_status s = check_type(who, "d_gate", d_gate->dtype, gate->dtype, wide_type(gate->dtype))) return s;
    RecurrenceArgs a = batch_args(gate, lengths);
    a.input = sequences_of(input), a.grad = sequences_of(grad), a.state = sequences_of(out);
    a.d_gate = sequences_of(d_gate), a.d_gate_wide = d_gate->dtype == HMR_F32, a.d_input = sequences_of(d_input);
    a.entry = states_of(grad_last), a.exit = states_of(d_initial), a.initial = states_of(initial);
    if (hmr_status s = check_room(who, workspace, workspace_bytes, room_for(gate))) return s;
    if (ctx == nullptr) return refuse(who, "null context");
    if (nothing_to_write(a)) return HMR_OK;
    return queue_on(ctx, who, [&](hipStream_t stream) {
        return with_float_type(gate->dtype, [&](auto tag) {
            using T = typename decltype(tag)::type;
            const ScanLayout layout = layout_of({gate, input, out, grad, d_gate, d_input});
            if ((scan_used(gate) || short_scan_used(gate, layout, true)) && near_by({gate, input, out, grad, d_gate, d_input})) {
                queue_scan_backward(stream, gate->dtype, form, a, layout, workspace);
                return;
            }
            with_code(form, std::integer_sequence<int, HMN_GATE_FACTOR, HMN_GATE_SIGMOID>{}, [&](auto f) {
                backward_kernel<T, decltype(f)::value><<<grid_of(ctx, a), kBlock, 0, stream>>>(a);
            });
        });
    });
}

}  // namespace

}  // namespace nn
}  // namespace hmr

extern "C" {

hmr_status hmn_recurrence_workspace(const hmr_tensor_desc *gate, int64_t *bytes) {
    return hmr::fenced([&] {
        constexpr const char *who = "hmn_recurrence_workspace";
        if (gate == nullptr || bytes == nullptr) return hmr::nn::refuse(who, "an argument is NULL");
        int64_t n = 0;
        if (hmr_status s = hmr::check_desc(*gate, n)) return s;
        if (gate->ndim != 3) return hmr::nn::refuse(who, "gate has " + std::to_string(gate->ndim) + " dimensions, not 3");
        if (!hmr::nn::is_float(gate->dtype)) return hmr::nn::refuse(who, "a recurrence takes floating point tensors");
        *bytes = hmr::nn::room_for(gate);
        return HMR_OK;
    });
}

hmr_status hmn_recurrence(hmr_context_t ctx, int32_t form, const hmr_tensor_desc *out, const hmr_tensor_desc *last,
                          const hmr_tensor_desc *gate, const hmr_tensor_desc *input, const hmr_tensor_desc *initial,
                          const hmr_tensor_desc *lengths, void *workspace, int64_t workspace_bytes) {
    return hmr::fenced([&] {
        return hmr::nn::forward(ctx, form, out, last, gate, input, initial, lengths, workspace, workspace_bytes);
    });
}

hmr_status hmn_recurrence_backward(hmr_context_t ctx, int32_t form, const hmr_tensor_desc *d_gate,
                                   const hmr_tensor_desc *d_input, const hmr_tensor_desc *d_initial,
                                   const hmr_tensor_desc *grad, const hmr_tensor_desc *grad_last, const hmr_tensor_desc *gate,
                                   const hmr_tensor_desc *input, const hmr_tensor_desc *out, const hmr_tensor_desc *initial,
                                   const hmr_tensor_desc *lengths, void *workspace, int64_t workspace_bytes) {
    return hmr::fenced([&] {
        return hmr::nn::backward(ctx, form, d_gate, d_input, d_initial, grad, grad_last, gate, input, out, initial, lengths,
                                 workspace, workspace_bytes);
    });
}

}  // extern "C"
