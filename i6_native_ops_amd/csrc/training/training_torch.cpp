// PyTorch-ROCm binding of libi6train.so: module `training_core`.  torch is used for device memory, the current
// stream and the autograd graph; all arithmetic is behind the C ABI declared in include/i6train.h.  The graph's nodes
// are C++: the smallest training steps take as long as their host work, of which nodes in Python would be the larger part.
#include <algorithm>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include "../../../include/i6fbw.h"
#include "../../../include/i6delta.h"
#include "../../../include/i6logp.h"
#include "../../../include/i6orth.h"
#include "../../../include/i6train.h"

namespace {

using Optional = std::optional<torch::Tensor>;

// The messages of the other bindings' checks.
#define CHECK_CUDA(x) TORCH_CHECK(x.device().is_cuda(), #x " must be a CUDA tensor")
#define CHECK_CONTIGUOUS(x) TORCH_CHECK(x.is_contiguous(), #x " must be contiguous")
#define CHECK_TYPE(x, type) \
    TORCH_CHECK(x.dtype() == type, "Expected " #x " to contain elements of type ", type, ", but got type ", x.dtype())
#define CHECK_DEVICE(x, y) TORCH_CHECK(x.device() == y.device(), #x " must be on the device of " #y)

int dtype_of(const torch::Tensor& x, const char* name) {
    TORCH_CHECK(x.scalar_type() == torch::kFloat32 || x.scalar_type() == torch::kBFloat16, "Expected ", name,
                " to contain elements of type Float or BFloat16, but got type ", x.dtype());
    return x.scalar_type() == torch::kBFloat16 ? I6TRAIN_BF16 : I6TRAIN_F32;
}

void check(const char* op, int rc) { TORCH_CHECK(rc == I6TRAIN_OK, "NativeOp: ", op, ": ", i6train_strerror(rc)); }

hipStream_t current_stream() { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream(); }

void raise_reported(const char* prefix) {
    int code = 0, seq = -1;
    check("status", i6train_poll_status(&code, &seq));
    TORCH_CHECK(code == I6TRAIN_OK, prefix, "sequence ", seq, ": ", i6train_strerror(code));
}

// As the status mode of the other modules says: not at all, by waiting, or by a later call.
void report(hipStream_t stream, const char* op = "linear_cross_entropy") {
    const int mode = i6fbw_get_status_mode();
    if (mode == 0) return;
    hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(stream, &capture) != hipSuccess || capture != hipStreamCaptureStatusNone) return;
    if (mode == 1) TORCH_CHECK(hipStreamSynchronize(stream) == hipSuccess, "NativeOp: HIP call failed");
    raise_reported(mode == 1 ? (std::string("NativeOp: ") + op + ": ").c_str() : "NativeOp: an earlier call reported: ");
}

void check_status() {
    TORCH_CHECK(hipDeviceSynchronize() == hipSuccess, "NativeOp: HIP call failed");
    raise_reported("NativeOp: an earlier call reported: ");
}

bool unit_stride(const torch::Tensor& x) { return x.dim() == 0 || x.stride(-1) == 1 || x.size(-1) == 1; }

torch::Tensor bytes(size_t n, const torch::Tensor& like) {
    return torch::empty({(int64_t)n}, torch::TensorOptions().device(like.device()).dtype(torch::kUInt8));
}

// ------------------------------------------------------------------------------------------------------ cross entropy

i6train_ce_problem ce_problem(const torch::Tensor& hidden, const torch::Tensor& weight, const torch::Tensor& targets, const torch::Tensor& seq_lens,
                              const Optional& bias) {
    i6train_ce_problem p{};
    p.B = (int)hidden.size(0); p.T = (int)hidden.size(1); p.D = (int)hidden.size(2); p.F = (int)weight.size(0);
    p.hidden = hidden.data_ptr(); p.hidden_stride_b = hidden.stride(0); p.hidden_stride_t = hidden.stride(1);
    p.dtype = dtype_of(weight, "weight");
    p.weight = weight.data_ptr(); p.weight_stride_f = weight.stride(0);
    p.bias = bias ? bias->data_ptr() : nullptr;
    p.targets = targets.data_ptr<int32_t>(); p.targets_stride_b = targets.stride(0); p.targets_stride_t = targets.stride(1);
    p.seq_lens = seq_lens.data_ptr<int32_t>();
    return p;
}

std::tuple<torch::Tensor, torch::Tensor> linear_cross_entropy_forward(const torch::Tensor& hidden, const torch::Tensor& weight, const torch::Tensor& targets, const torch::Tensor& seq_lens,
                                                        const Optional& bias) {
    CHECK_CUDA(hidden);
    dtype_of(hidden, "hidden");
    CHECK_CUDA(weight);
    CHECK_TYPE(weight, hidden.dtype());
    CHECK_CUDA(targets);
    CHECK_TYPE(targets, torch::kInt32);
    CHECK_CUDA(seq_lens);
    CHECK_CONTIGUOUS(seq_lens);
    CHECK_TYPE(seq_lens, torch::kInt32);
    TORCH_CHECK(hidden.dim() == 3 && unit_stride(hidden), "hidden must have shape (B, T, D) with unit innermost stride");
    TORCH_CHECK(weight.dim() == 2 && weight.size(1) == hidden.size(2) && unit_stride(weight), "weight must have shape (F, D) with unit innermost stride");
    TORCH_CHECK(targets.dim() == 2 && targets.size(0) == hidden.size(0) && targets.size(1) == hidden.size(1), "targets must have shape (B, T)");
    TORCH_CHECK(seq_lens.dim() == 1 && seq_lens.size(0) == hidden.size(0), "seq_lens must have shape (B,)");
    CHECK_DEVICE(weight, hidden);
    CHECK_DEVICE(targets, hidden);
    CHECK_DEVICE(seq_lens, hidden);
    if (bias) {
        const torch::Tensor& b = *bias;
        TORCH_CHECK(b.device() == hidden.device() && b.dtype() == hidden.dtype() && b.dim() == 1 && b.size(0) == weight.size(0) && b.is_contiguous(),
                    "bias must be a contiguous tensor of shape (F,), of the type and on the device of hidden");
    }
    TORCH_CHECK(hidden.numel() > 0 && weight.numel() > 0, "NativeOp assertion failed: B > 0, T > 0, F > 0, D > 0");
    TORCH_CHECK(hidden.size(0) < (1 << 30) && hidden.size(1) < (1 << 30) && hidden.size(2) < (1 << 30) && weight.size(0) < (1 << 30), "NativeOp: linear_cross_entropy: ",
                i6train_strerror(I6TRAIN_ERR_TOO_LARGE));
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(hidden.device());
    const i6train_ce_problem p = ce_problem(hidden, weight, targets, seq_lens, bias);
    size_t forward_bytes = 0, backward_bytes = 0;
    check("linear_cross_entropy", i6train_ce_workspace_size(&p, &forward_bytes, &backward_bytes));
    torch::Tensor workspace = bytes(forward_bytes, hidden);
    torch::Tensor loss = torch::empty({p.B, p.T}, hidden.options().dtype(torch::kFloat32));
    hipStream_t stream = current_stream();
    check("linear_cross_entropy", i6train_ce_forward(&p, loss.data_ptr<float>(), workspace.data_ptr(), forward_bytes, (void*)stream));
    report(stream);
    return {loss, workspace};
}

std::vector<Optional> linear_cross_entropy_backward(const torch::Tensor& grad_loss, const torch::Tensor& hidden, const torch::Tensor& weight, const torch::Tensor& targets,
                                                    const torch::Tensor& seq_lens, const Optional& bias, const torch::Tensor& forward_workspace, bool need_hidden,
                                                    bool need_weight, bool need_bias) {
    CHECK_CUDA(grad_loss);
    CHECK_TYPE(grad_loss, torch::kFloat32);
    CHECK_DEVICE(grad_loss, weight);
    TORCH_CHECK(grad_loss.sizes() == targets.sizes(), "grad_loss must have shape (B, T)");
    CHECK_CUDA(forward_workspace);
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(weight.device());
    const i6train_ce_problem p = ce_problem(hidden, weight, targets, seq_lens, bias);
    size_t forward_bytes = 0, backward_bytes = 0;
    check("linear_cross_entropy", i6train_ce_workspace_size(&p, &forward_bytes, &backward_bytes));
    torch::Tensor workspace = bytes(backward_bytes, weight);
    const auto opts = weight.options();
    Optional grad_hidden, grad_weight, grad_bias;
    if (need_hidden) grad_hidden = torch::empty({p.B, p.T, p.D}, opts);
    if (need_weight) grad_weight = torch::empty({p.F, p.D}, opts);
    if (need_bias && bias) grad_bias = torch::empty({p.F}, opts);
    const auto ptr = [](Optional& t) { return t ? t->data_ptr() : nullptr; };
    check("linear_cross_entropy", i6train_ce_backward(&p, grad_loss.data_ptr<float>(), grad_loss.stride(0), grad_loss.stride(1), ptr(grad_hidden), ptr(grad_weight), ptr(grad_bias),
                                                      forward_workspace.data_ptr(), forward_workspace.numel(), workspace.data_ptr(), backward_bytes, (void*)current_stream()));
    return {grad_hidden, grad_weight, grad_bias};
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// The last dimension with unit stride.  Where it has one value its stride says nothing and may be anything, contiguous() or not.
torch::Tensor rows(const torch::Tensor& x) { return unit_stride(x) ? x : x.contiguous(); }
Optional given(const torch::Tensor& x) { return x.defined() ? Optional(x) : Optional(); }
torch::Tensor or_none(const Optional& x) { return x ? *x : torch::Tensor(); }
// Tangents would be lost in silence: the kernels know nothing of them.
void refuse_tangents(const char* op, std::initializer_list<torch::Tensor> inputs) {
    for (const torch::Tensor& x : inputs) TORCH_CHECK(!x.defined() || !x._fw_grad(/*level=*/0).defined(), op, " has no forward-mode derivative");
}
bool wants_gradient(std::initializer_list<torch::Tensor> inputs) {
    if (!at::GradMode::is_enabled()) return false;
    for (const torch::Tensor& x : inputs)
        if (x.defined() && x.requires_grad()) return true;
    return false;
}

// Gradients of gradients are refused as they are asked for, not as create_graph is.  A gradient depends on the inputs as it does on the incoming one.
variable_list once(const char* op, const variable_list& incoming, std::initializer_list<torch::Tensor> inputs, variable_list outgoing) {
    if (!at::GradMode::is_enabled()) return outgoing;
    bool tracked = wants_gradient(inputs);
    for (const torch::Tensor& g : incoming) tracked = tracked || (g.defined() && g.requires_grad());
    if (!tracked) return outgoing;
    for (torch::Tensor& g : outgoing)
        if (g.defined()) g = g.detach().requires_grad_();
    return (*std::make_shared<torch::autograd::DelayedError>(std::string(op) + " can be differentiated once", (int64_t)outgoing.size()))(std::move(outgoing));
}

struct LinearCrossEntropy : torch::autograd::Function<LinearCrossEntropy> {
    static torch::Tensor forward(AutogradContext* ctx, const torch::Tensor& hidden, const torch::Tensor& weight, const Optional& bias, const torch::Tensor& targets,
                                 const torch::Tensor& seq_lens) {
        auto [loss, workspace] = linear_cross_entropy_forward(hidden, weight, targets, seq_lens, bias);
        ctx->save_for_backward({hidden, weight, or_none(bias), targets, seq_lens, workspace});
        return loss;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        const variable_list saved = ctx->get_saved_variables();
        const std::vector<Optional> got = linear_cross_entropy_backward(grads[0], saved[0], saved[1], saved[3], saved[4], given(saved[2]), saved[5],
                                                                        ctx->needs_input_grad(0), ctx->needs_input_grad(1), saved[2].defined() && ctx->needs_input_grad(2));      // (a missing bias has no number)
        variable_list out(5);
        for (int i = 0; i < 3; i++)
            if (got[i]) out[i] = *got[i];
        return once("linear_cross_entropy", grads, {saved[0], saved[1], saved[2]}, std::move(out));
    }
};

torch::Tensor linear_cross_entropy(const torch::Tensor& hidden, const torch::Tensor& weight, const torch::Tensor& targets, const torch::Tensor& seq_lens, const Optional& bias) {
    refuse_tangents("linear_cross_entropy", {hidden, weight, or_none(bias)});
    if (wants_gradient({hidden, weight, or_none(bias)}))
        return LinearCrossEntropy::apply(rows(hidden), rows(weight), bias, targets, seq_lens);
    return std::get<0>(linear_cross_entropy_forward(rows(hidden), rows(weight), targets, seq_lens, bias));
}

// --------------------------------------------------------------------------------------------------------- recurrence

i6train_rec_problem rec_problem(const torch::Tensor& x, const torch::Tensor& gate, const Optional& seq_lens, const Optional& initial) {
    CHECK_CUDA(x);
    i6train_rec_problem p{};
    p.dtype = dtype_of(x, "x");
    CHECK_CUDA(gate);
    CHECK_TYPE(gate, x.dtype());
    CHECK_DEVICE(gate, x);
    TORCH_CHECK(x.dim() == 3 && unit_stride(x), "x must have shape (B, T, D) with unit innermost stride");
    TORCH_CHECK(gate.sizes() == x.sizes() && unit_stride(gate), "gate must have the shape of x, with unit innermost stride");
    TORCH_CHECK(x.numel() > 0, "NativeOp assertion failed: B > 0, T > 0, D > 0");
    TORCH_CHECK(x.size(0) <= 65535 && x.size(1) <= (1 << 30) && x.size(2) <= (1 << 30), "NativeOp: gated_recurrence: at most 65535 sequences");
    if (seq_lens) {
        CHECK_CUDA((*seq_lens));
        TORCH_CHECK(seq_lens->dtype() == torch::kInt32 && seq_lens->is_contiguous() && seq_lens->dim() == 1 && seq_lens->size(0) == x.size(0) && seq_lens->device() == x.device(),
                    "seq_lens must be a contiguous int32 tensor of shape (B,) on the device of x");
    }
    if (initial) {
        CHECK_CUDA((*initial));
        TORCH_CHECK(initial->dtype() == torch::kFloat32 && initial->is_contiguous() && initial->dim() == 2 && initial->size(0) == x.size(0) && initial->size(1) == x.size(2) &&
                        initial->device() == x.device(),
                    "initial_state must be a contiguous float32 tensor of shape (B, D) on the device of x");
    }
    p.B = (int)x.size(0); p.T = (int)x.size(1); p.D = (int)x.size(2);
    p.x = x.data_ptr(); p.x_stride_b = x.stride(0); p.x_stride_t = x.stride(1);
    p.gate = gate.data_ptr(); p.gate_stride_b = gate.stride(0); p.gate_stride_t = gate.stride(1);
    p.seq_lens = seq_lens ? seq_lens->data_ptr<int32_t>() : nullptr;
    p.initial = initial ? initial->data_ptr<float>() : nullptr;
    return p;
}

Optional rec_workspace(const i6train_rec_problem& p, const torch::Tensor& x, size_t& n) {
    check("gated_recurrence", i6train_rec_workspace_size(&p, &n));
    return n ? Optional(bytes(n, x)) : Optional();
}

std::vector<Optional> gated_recurrence_forward(const torch::Tensor& x, const torch::Tensor& gate, const Optional& seq_lens, const Optional& initial, bool keep_states) {
    const i6train_rec_problem p = rec_problem(x, gate, seq_lens, initial);
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    torch::Tensor h = torch::empty({p.B, p.T, p.D}, x.options());
    torch::Tensor last = torch::empty({p.B, p.D}, x.options().dtype(torch::kFloat32));
    Optional states;
    if (keep_states) {
        size_t n = 0;
        check("gated_recurrence", i6train_rec_states_size(&p, &n));
        states = torch::empty({(int64_t)(n / sizeof(float))}, x.options().dtype(torch::kFloat32));
    }
    size_t n = 0;
    Optional workspace = rec_workspace(p, x, n);
    check("gated_recurrence", i6train_rec_forward(&p, h.data_ptr(), last.data_ptr<float>(), states ? states->data_ptr<float>() : nullptr, workspace ? workspace->data_ptr() : nullptr, n,
                                                  (void*)current_stream()));
    return {h, last, states};
}

std::vector<torch::Tensor> gated_recurrence_backward(const Optional& grad_h, const Optional& grad_last, const torch::Tensor& x, const torch::Tensor& gate, const Optional& seq_lens,
                                                     const torch::Tensor& states) {
    const i6train_rec_problem p = rec_problem(x, gate, seq_lens, Optional());
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    if (grad_h) TORCH_CHECK(grad_h->sizes() == x.sizes() && grad_h->dtype() == x.dtype() && unit_stride(*grad_h) && grad_h->device() == x.device(), "grad_h must match x");
    if (grad_last)
        TORCH_CHECK(grad_last->dtype() == torch::kFloat32 && grad_last->is_contiguous() && grad_last->numel() == (int64_t)p.B * p.D && grad_last->device() == x.device(),
                    "grad_last must be a contiguous float32 tensor of shape (B, D)");
    torch::Tensor grad_x = torch::empty({p.B, p.T, p.D}, x.options()), grad_gate = torch::empty_like(grad_x);
    torch::Tensor grad_initial = torch::empty({p.B, p.D}, x.options().dtype(torch::kFloat32));
    size_t n = 0;
    Optional workspace = rec_workspace(p, x, n);
    check("gated_recurrence", i6train_rec_backward(&p, grad_h ? grad_h->data_ptr() : nullptr, grad_h ? grad_h->stride(0) : 0, grad_h ? grad_h->stride(1) : 0,
                                                   grad_last ? grad_last->data_ptr<float>() : nullptr, states.data_ptr<float>(), grad_x.data_ptr(), grad_gate.data_ptr(),
                                                   grad_initial.data_ptr<float>(), workspace ? workspace->data_ptr() : nullptr, n, (void*)current_stream()));
    return {grad_x, grad_gate, grad_initial};
}

struct GatedRecurrence : torch::autograd::Function<GatedRecurrence> {
    static variable_list forward(AutogradContext* ctx, const torch::Tensor& x, const torch::Tensor& gate, const Optional& initial, const Optional& seq_lens) {
        std::vector<Optional> got = gated_recurrence_forward(x, gate, seq_lens, initial, true);
        ctx->save_for_backward({x, gate, or_none(seq_lens), *got[2], or_none(initial)});
        ctx->set_materialize_grads(false);
        return {*got[0], *got[1]};
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        const variable_list saved = ctx->get_saved_variables();
        const Optional grad_h = grads[0].defined() ? Optional(rows(grads[0])) : Optional(), grad_last = grads[1].defined() ? Optional(grads[1].contiguous()) : Optional();
        const std::vector<torch::Tensor> got = gated_recurrence_backward(grad_h, grad_last, saved[0], saved[1], given(saved[2]), saved[3]);
        return once("gated_recurrence", grads, {saved[0], saved[1], saved[4]}, {got[0], got[1], saved[4].defined() && ctx->needs_input_grad(2) ? got[2] : torch::Tensor(), torch::Tensor()});
    }
};

std::tuple<torch::Tensor, torch::Tensor> gated_recurrence(const torch::Tensor& x, const torch::Tensor& gate, const Optional& seq_lens, const Optional& initial) {
    refuse_tangents("gated_recurrence", {x, gate, or_none(initial)});
    if (wants_gradient({x, gate, or_none(initial)})) {
        const variable_list out = GatedRecurrence::apply(rows(x), rows(gate), initial, seq_lens);
        return {out[0], out[1]};
    }
    std::vector<Optional> got = gated_recurrence_forward(rows(x), rows(gate), seq_lens, initial, false);
    return {*got[0], *got[1]};
}

// -------------------------------------------------------------------------------------------------------------- AdamW

void adamw_step(const std::vector<torch::Tensor>& params, const std::vector<torch::Tensor>& grads, const std::vector<torch::Tensor>& exp_avgs,
                const std::vector<torch::Tensor>& exp_avg_sqs, const std::vector<std::pair<torch::Tensor, torch::Tensor>>& scales, int64_t step, double lr, double beta1, double beta2,
                double eps, double weight_decay) {
    const size_t n = params.size();
    TORCH_CHECK(grads.size() == n && exp_avgs.size() == n && exp_avg_sqs.size() == n, "params, grads, exp_avgs and exp_avg_sqs must have the same length");
    if (n == 0) return;
    const auto device = params[0].device();
    const auto type = params[0].scalar_type();
    const int dtype = dtype_of(params[0], "params");
    const int bits = exp_avgs[0].scalar_type() == torch::kFloat8_e4m3fn ? 8 : 32;
    const auto state_type = bits == 8 ? torch::kFloat8_e4m3fn : torch::kFloat32;
    TORCH_CHECK(bits == 8 ? scales.size() == n : scales.empty(), "scales belong to states in 8 bits, a pair for each tensor");
    std::vector<i6train_adamw_tensor> table(n);
    for (size_t i = 0; i < n; i++) {
        const torch::Tensor &p = params[i], &g = grads[i], &m = exp_avgs[i], &v = exp_avg_sqs[i];
        const int64_t count = p.numel();
        TORCH_CHECK(p.device().is_cuda() && p.device() == device && p.scalar_type() == type && p.is_contiguous(), "params[", i,
                    "] must be a contiguous CUDA tensor, of the type and on the device of the first");
        TORCH_CHECK(g.device() == device && g.scalar_type() == type && g.is_contiguous() && g.numel() == count, "grads[", i, "] must be contiguous and match params[", i, "]");
        TORCH_CHECK(m.device() == device && m.scalar_type() == state_type && m.is_contiguous() && m.numel() == count, "exp_avgs[", i,
                    "] must be contiguous, of params' size and float32 or float8_e4m3fn like the first");
        TORCH_CHECK(v.device() == device && v.scalar_type() == state_type && v.is_contiguous() && v.numel() == count, "exp_avg_sqs[", i, "] must match exp_avgs[", i, "]");
        table[i] = {p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr(), nullptr, nullptr, count};
        if (bits == 8) {
            const int64_t blocks = (count + I6TRAIN_BLOCK - 1) / I6TRAIN_BLOCK;
            for (const torch::Tensor* s : {&scales[i].first, &scales[i].second})
                TORCH_CHECK(s->device() == device && s->scalar_type() == torch::kFloat32 && s->is_contiguous() && s->numel() == blocks, "scales[", i,
                            "] must be two contiguous float32 tensors of a value for each 256 values");
            table[i].exp_avg_scale = scales[i].first.data_ptr<float>();
            table[i].exp_avg_sq_scale = scales[i].second.data_ptr<float>();
        }
    }
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(device);
    const int rc = i6train_adamw(table.data(), (int)n, dtype, bits, step, lr, beta1, beta2, eps, weight_decay, (void*)current_stream());
    // what a graph has saved of these tensors is not what it was; tensors made in inference mode are in no graph and have no version
    const auto changed = [](const torch::Tensor& t) {
        if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    };
    for (const auto* list : {&params, &exp_avgs, &exp_avg_sqs})
        for (const torch::Tensor& t : *list) changed(t);
    for (const auto& pair : scales) {
        changed(pair.first);
        changed(pair.second);
    }
    check("adamw_step", rc);
}

#include "more_torch.inc"

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("linear_cross_entropy", &linear_cross_entropy, "loss (B, T)");
    m.def("gated_recurrence", &gated_recurrence, "h (B, T, D), last (B, D)");
    m.def("adamw_step", &adamw_step, "One AdamW step over lists of tensors, in place");
    m.def("target_log_probs", &target_log_probs, "log_prob (B, T), entropy (B, T), top_log_probs (B, T, k), top_classes (B, T, k)");
    m.def("gated_delta_rule", &gated_delta_rule, "o (B, T, H, V), last (B, H, K, V)");
    m.def("orthogonalize", &orthogonalize, "The orthogonal factors of matrices");
    m.def("muon_step", &muon_step, "One step on the orthogonal factors of the averaged gradients, in place");
    m.def("check_status", &check_status, "Waits for the device and raises the first problem that kernels of earlier calls reported");
}
