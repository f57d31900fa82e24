// The host's half of cpp_extension/block_ops.py: checks, buffers and launches of the entry points of schemanet_blocks.h on torch tensors,
// and their autograd nodes.  Built into lib/_schemanet_blocks.so, a Python module without a link to the kernel library: bind() hands
// it the entry points of the one that is loaded.
// Why not Python: a small call is bound by its host part, most of all in training, where the autograd engine runs the backward half on a
// thread of its own that has to fetch the interpreter first.
#include <Python.h>

#include <cstdarg>
#include <cstring>
#include <stdexcept>

#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>

#include "schemanet_blocks.h"

namespace {

using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

// ---------------------------------------------------------------------------------------------------------- the bound library
struct Library {
    decltype(&sn_last_error) last_error;
    decltype(&sn_checkpoint8) checkpoint8;
    decltype(&sn_checkpoint8_restore) restore;
    decltype(&sn_checkpoint8_weight_grad_workspace) weight_grad_workspace;
    decltype(&sn_checkpoint8_weight_grad) weight_grad;
    decltype(&sn_block_norms_forward) norms_forward;
    decltype(&sn_block_norms_workspace) norms_workspace;
    decltype(&sn_block_norms_backward) norms_backward;
    decltype(&sn_label_log_probs_workspace) scores_workspace;
    decltype(&sn_label_log_probs) scores;
    decltype(&sn_label_log_probs_backward) scores_backward;
} lib;
constexpr Py_ssize_t kEntries = sizeof(Library) / sizeof(void *);
PyObject *require_gpu = nullptr;             // called before the first launch, then dropped

[[noreturn]] void refuse(const char *format, ...)
{
    char text[512];
    va_list args;
    va_start(args, format);
    vsnprintf(text, sizeof text, format, args);
    va_end(args);
    throw std::runtime_error(text);
}

// tuple(shape) as Python prints it
std::string shown(at::IntArrayRef shape)
{
    std::string s = "(";
    for (size_t i = 0; i < shape.size(); ++i) s += (i ? ", " : "") + std::to_string(shape[i]);
    return s + (shape.size() == 1 ? ",)" : ")");
}

int type_of(at::ScalarType t) { return t == at::kFloat ? SN_F32 : t == at::kBFloat16 ? SN_BF16 : t == at::kHalf ? SN_F16 : -1; }
int type_of(const Tensor &t) { return type_of(t.scalar_type()); }

void one_device(std::initializer_list<const Tensor *> tensors)
{
    const Tensor *first = nullptr;
    for (const Tensor *t : tensors) {
        if (!t->defined()) continue;
        if (!t->is_cuda()) refuse("expected CUDA tensors (the HIP path has no CPU fallback)");
        if (!first) first = t;
        else if (t->device() != first->device())
            refuse("tensors on different devices: %s vs %s", first->device().str().c_str(), t->device().str().c_str());
    }
}

// Forward-mode derivatives are not carried: the result of a tensor with a tangent would read as one whose tangent is zero.  (Inside a
// Function's forward the mode is off, and the Function's own jvp answers for its inputs.)
void no_tangents(std::initializer_list<const Tensor *> tensors, const char *who)
{
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    for (const Tensor *t : tensors)
        TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), who, ": no forward-mode derivatives");
}

void before_launch()
{
    if (!require_gpu) return;
    PyObject *r = PyObject_CallNoArgs(require_gpu);
    if (!r) throw python_error();
    Py_DECREF(r);
    Py_CLEAR(require_gpu);
}

void check(int rc, const char *what)
{
    if (rc != 0) refuse("libschemanet_hip %s failed (%d): %s", what, rc, lib.last_error());
}

void *stream_of(const Tensor &t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
// (a NULL pointer tells the library that there is no such tensor: one whose storage was freed must not pass for that)
void *pointer(const Tensor &t)
{
    if (!t.defined()) return nullptr;
    void *const p = t.data_ptr();
    if (!p && t.numel()) refuse("a tensor of shape %s has no memory: its storage was freed", shown(t.sizes()).c_str());
    return p;
}
Tensor empty(at::IntArrayRef sizes, const Tensor &like, at::ScalarType type) { return at::empty(sizes, like.options().dtype(type).requires_grad(false)); }

// [..., width]: a tensor that holds the rows (itself where they lie evenly apart, else a copy) and the elements from one row to the next
struct Rows { Tensor t; int64_t stride; };
Rows rows_of(const Tensor &t, int64_t width)
{
    if (!t.defined()) return {t, 0};
    if (t.is_neg()) return {t.resolve_neg().contiguous(), width};           // (a view that stands for its negative, as imag of a conjugate)
    if (t.is_contiguous()) return {t, width};
    if (t.stride(-1) != 1 && width > 1) return {t.contiguous(), width};
    int64_t stride = -1, next = 0;
    for (int64_t d = t.dim() - 2; d >= 0; --d) {
        if (t.size(d) == 1) continue;
        if (stride < 0) stride = t.stride(d);
        else if (t.stride(d) != next) return {t.contiguous(), width};
        next = t.stride(d) * t.size(d);
    }
    return {t, stride < 0 ? width : stride};
}

int64_t rows_in(at::IntArrayRef shape)
{
    int64_t rows = 1;
    for (size_t i = 0; i + 1 < shape.size(); ++i) rows *= shape[i];
    return rows;
}

// The kernels read codes and exponents by the activation's shape.  Checked at each use: either may have been resized or freed in place
// since the checkpoint was made, or come back from a hook for saved tensors.
void check_kept(const Tensor &codes, const Tensor &exps, at::IntArrayRef shape)
{
    const int64_t rows = rows_in(shape), npad = (shape.back() + 31) / 32 * 32;
    auto fits = [&](const Tensor &t, at::ScalarType type, int64_t columns) {
        return t.defined() && t.scalar_type() == type && t.dim() == 2 && t.size(0) == rows && t.size(1) == columns && t.is_contiguous() &&
               (int64_t)t.storage().nbytes() >= t.storage_offset() + rows * columns;
    };
    if (!fits(codes, at::kChar, npad) || !fits(exps, at::kByte, npad / 32))
        refuse("checkpoint8: codes and exponents do not hold an activation %s (any more)", shown(shape).c_str());
}

// What a node saved (undefined if there was nothing), as it comes back: hooks for saved tensors may hand over anything, and the kernels
// read it by the forward call's types and sizes.
Tensor unpack(const SavedVariable &v, at::ScalarType type, at::IntArrayRef sizes, c10::Device device, const char *who)
{
    Tensor t = v.unpack();
    if (t.defined() && (t.scalar_type() != type || t.sizes() != sizes || t.device() != device))
        refuse("%s: a saved tensor of type %s and shape %s on %s came back as %s, %s on %s", who, c10::toString(type), shown(sizes).c_str(), device.str().c_str(),
               c10::toString(t.scalar_type()), shown(t.sizes()).c_str(), t.device().str().c_str());
    return t;
}
Tensor unpack_whole(const SavedVariable &v, at::ScalarType type, at::IntArrayRef sizes, c10::Device device, const char *who)
{
    const Tensor t = unpack(v, type, sizes, device, who);
    return t.defined() ? t.contiguous() : t;
}

// A backward pass captured into a graph must not reach autograd nodes of the default stream, which cannot take part in a capture: those
// that an eager graph of the same leaves keeps alive.  The engine would find out on its own thread and end the process.
void before_capture(const torch::autograd::edge_list &edges, const char *who)
{
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    for (const torch::autograd::Edge &e : edges) {
        if (!e.is_valid()) continue;
        const auto stream = e.function->stream();
        if (stream && stream->id() == 0)
            refuse("%s: captured into a graph while an autograd graph of the default stream uses the same tensors (drop its results first)", who);
    }
}

// Results of a backward pass that was asked for its own graph: whoever differentiates them, with respect to the node's inputs or to the
// upstream gradients, gets an error.
variable_list without_second(const torch::autograd::Node &node, const variable_list &upstream, variable_list out)
{
    if (!at::GradMode::is_enabled()) return out;
    torch::autograd::edge_list edges = node.next_edges();
    for (const Tensor &g : upstream)
        if (g.defined() && g.requires_grad()) edges.push_back(torch::autograd::impl::gradient_edge(g));
    const std::shared_ptr<torch::autograd::Node> error(new torch::autograd::Error(node.name() + ": no second derivatives", std::move(edges)),
                                                       torch::autograd::deleteNode);
    for (Tensor &t : out) {
        if (!t.defined()) continue;
        t = t.detach();
        torch::autograd::set_history(t, error);
    }
    return out;
}

// -------------------------------------------------------------------------------------------------------------------- norms
struct NormsCall {
    bool rms;
    float eps;
    Tensor n_valid;
    Tensor params[5];                        // scale, post weight, post bias, pre weight, pre bias
};

sn_block_norms_args norms_args(const NormsCall &c, int type, at::IntArrayRef shape, int64_t rows)
{
    sn_block_norms_args a = {};
    a.struct_size = sizeof a;
    a.dtype = type;
    for (const Tensor &p : c.params)
        if (p.defined()) { a.param_dtype = type_of(p); break; }
    a.rms = c.rms;
    a.rows = rows;
    a.width = (int32_t)shape.back();
    a.n_valid = (const int32_t *)pointer(c.n_valid);
    a.rows_per_graph = c.n_valid.defined() ? (int32_t)shape[1] : 0;
    a.eps = c.eps;
    a.has_post = c.params[1].defined();
    a.has_pre = c.params[3].defined();
    a.scale = pointer(c.params[0]);
    a.post_weight = pointer(c.params[1]);
    a.post_bias = pointer(c.params[2]);
    a.pre_weight = pointer(c.params[3]);
    a.pre_bias = pointer(c.params[4]);
    return a;
}

struct GatedResidualNormsBackward : torch::autograd::Node {
    SavedVariable params[5], n_valid, stats, held[6];        // held: x, branch, gate or their checkpoints (codes, exps)
    at::DimVector shape;
    at::TensorOptions options;
    at::ScalarType param_type = at::kFloat;
    bool rms = false, kept = false, gated = false, empty_rows = false;
    float eps = 0;

    std::string name() const override { return "GatedResidualNormsBackward"; }
    void release_variables() override
    {
        std::lock_guard<std::mutex> lock(mutex_);
        for (auto &v : params) v.reset_data();
        for (auto &v : held) v.reset_data();
        n_valid.reset_data();
        stats.reset_data();
    }
    variable_list apply(variable_list &&grads) override
    {
        std::lock_guard<std::mutex> lock(mutex_);
        no_tangents({&grads.front(), &grads.back()}, "gated_residual_norms (backward)");
        variable_list out(8);
        {
            at::AutoDispatchBelowADInplaceOrView raw;
            run(grads[0], grads.size() > 1 ? grads[1] : Tensor(), out);
        }
        return without_second(*this, grads, std::move(out));
    }

    void run(const Tensor &dy, const Tensor &dh, variable_list &out)
    {
        if (!dy.defined() && !dh.defined()) return;
        const char *const who = "gated_residual_norms (backward)";
        const c10::Device place = options.device();
        const int64_t rows = rows_in(shape), width = shape.back();
        NormsCall c = {rms, eps, unpack_whole(n_valid, at::kInt, at::IntArrayRef(shape).slice(0, 1), place, who), {}};
        for (int i = 0; i < 5; ++i) c.params[i] = unpack_whole(params[i], param_type, width, place, who);
        bool want[8], columns = false;
        for (int i = 0; i < 8; ++i) want[i] = task_should_compute_output(i);
        want[2] = want[2] && gated;
        if (empty_rows) {
            for (int i = 0; i < 3; ++i)
                if (want[i]) out[i] = at::zeros(shape, options);
            for (int i = 0; i < 5; ++i)
                if (want[3 + i] && c.params[i].defined()) out[3 + i] = at::zeros_like(c.params[i]);
            return;
        }
        const Tensor st = unpack_whole(stats, at::kFloat, {rows, 4}, place, who), &any = dy.defined() ? dy : dh;
        Tensor h[6];
        if (kept) {
            for (int i = 0; i < 6; ++i) h[i] = held[i].unpack();
            for (int i = 0; i < (gated ? 6 : 4); i += 2) {
                check_kept(h[i], h[i + 1], {rows, width});
                one_device({&any, &h[i], &h[i + 1]});
            }
        } else {
            for (int i = 0; i < 3; ++i) h[i] = unpack(held[i], at::typeMetaToScalarType(options.dtype()), shape, place, who);
        }
        const c10::DeviceGuard device(any.device());
        sn_block_norms_args a = norms_args(c, type_of(any), shape, rows);
        a.stats = (float *)pointer(st);
        Rows x, b, g;
        if (kept) {
            a.x_codes = pointer(h[0]), a.x_exps = pointer(h[1]);
            a.branch_codes = pointer(h[2]), a.branch_exps = pointer(h[3]);
            a.gate_codes = pointer(h[4]), a.gate_exps = pointer(h[5]);
        } else {
            x = rows_of(h[0], width), b = rows_of(h[1], width), g = rows_of(h[2], width);
            a.x = pointer(x.t), a.branch = pointer(b.t), a.gate = pointer(g.t);
            a.x_stride = x.stride, a.branch_stride = b.stride, a.gate_stride = g.stride;
        }
        const Rows ry = rows_of(dy, width), rh = rows_of(dh, width);
        a.dy = pointer(ry.t), a.dh = pointer(rh.t);
        a.dy_stride = ry.stride, a.dh_stride = rh.stride;
        for (int i = 0; i < 3; ++i)
            if (want[i]) out[i] = at::empty(shape, options);
        a.dx = pointer(out[0]), a.dbranch = pointer(out[1]), a.dgate = pointer(out[2]);
        void *into[5] = {};
        for (int i = 0; i < 5; ++i) columns |= want[3 + i] && c.params[i].defined();
        if (columns) {
            Tensor lines;                                    // one allocation for the parameters' gradients
            for (const Tensor &p : c.params)
                if (p.defined()) { lines = empty({5, width}, p, p.scalar_type()); break; }
            for (int i = 0; i < 5; ++i) {
                if (!want[3 + i] || !c.params[i].defined()) continue;
                out[3 + i] = lines.select(0, i);
                if (i >= 3 && !dh.defined()) out[3 + i].zero_();             // the norm before the next block took no part
                else into[i] = pointer(out[3 + i]);
            }
        }
        a.dscale = into[0], a.dpost_weight = into[1], a.dpost_bias = into[2], a.dpre_weight = into[3], a.dpre_bias = into[4];
        a.workspace_bytes = lib.norms_workspace(rows, (int)width);
        const Tensor workspace = empty({(int64_t)a.workspace_bytes}, any, at::kByte);
        a.workspace = pointer(workspace);
        check(lib.norms_backward(&a, stream_of(any)), "sn_block_norms_backward");
    }
};

struct NormsResult { Tensor y, h, stats, kept[6]; };
NormsResult norms_forward(const NormsCall &c, const Tensor &x, const Tensor &branch, const Tensor &gate, bool train, bool keep8)
{
    at::AutoDispatchBelowADInplaceOrView raw;
    NormsResult r;
    const int64_t width = x.size(-1), rows = x.numel() / width, npad = (width + 31) / 32 * 32;
    const c10::DeviceGuard device(x.device());
    r.y = empty(x.sizes(), x, x.scalar_type());
    if (c.params[3].defined()) r.h = empty(x.sizes(), x, x.scalar_type());
    if (rows == 0) return r;
    before_launch();
    const Rows rx = rows_of(x, width), rb = rows_of(branch, width), rg = rows_of(gate, width);
    sn_block_norms_args a = norms_args(c, type_of(x), x.sizes(), rows);
    a.x = pointer(rx.t), a.branch = pointer(rb.t), a.gate = pointer(rg.t);
    a.x_stride = rx.stride, a.branch_stride = rb.stride, a.gate_stride = rg.stride;
    a.y = pointer(r.y), a.h = pointer(r.h);
    if (train) {
        r.stats = empty({rows, 4}, x, at::kFloat);
        a.stats = (float *)pointer(r.stats);
        if (keep8) {
            for (int i = 0; i < (gate.defined() ? 3 : 2); ++i) {
                r.kept[2 * i] = empty({rows, npad}, x, at::kChar);
                r.kept[2 * i + 1] = empty({rows, npad / 32}, x, at::kByte);
            }
            a.x_codes = pointer(r.kept[0]), a.x_exps = pointer(r.kept[1]);
            a.branch_codes = pointer(r.kept[2]), a.branch_exps = pointer(r.kept[3]);
            a.gate_codes = pointer(r.kept[4]), a.gate_exps = pointer(r.kept[5]);
        }
    }
    check(lib.norms_forward(&a, stream_of(x)), "sn_block_norms_forward");
    return r;
}

std::pair<Tensor, Tensor> gated_residual_norms(const Tensor &x, const Tensor &branch, const Tensor &gate, NormsCall c, bool keep8)
{
    Tensor(&p)[5] = c.params;
    if (!x.defined() || type_of(x) < 0 || x.dim() < 1) refuse("gated_residual_norms: expected a float32, bfloat16 or float16 tensor");
    const int64_t width = x.size(-1);
    if (width < 1 || width > SN_BLOCK_NORMS_MAX_WIDTH) refuse("gated_residual_norms: width %lld outside 1 .. %d", (long long)width, SN_BLOCK_NORMS_MAX_WIDTH);
    auto like_x = [&](const Tensor &t) { return t.defined() && t.scalar_type() == x.scalar_type() && t.sizes() == x.sizes(); };
    if (!like_x(branch)) refuse("gated_residual_norms: branch must have x's shape %s and type", shown(x.sizes()).c_str());
    if (gate.defined() && !like_x(gate)) refuse("gated_residual_norms: gate must have x's shape %s and type", shown(x.sizes()).c_str());
    const Tensor *first = nullptr;
    bool mixed = false;
    for (Tensor &t : p) {
        if (!t.defined()) continue;
        if (type_of(t) < 0 || t.dim() != 1 || t.size(0) != width) refuse("gated_residual_norms: parameters must be [%lld]", (long long)width);
        if (!first) first = &t;
        mixed |= t.scalar_type() != first->scalar_type();
    }
    if (c.eps < 0) refuse("gated_residual_norms: eps %g", c.eps);
    const Tensor &v = c.n_valid;
    if (v.defined() && !(x.dim() == 3 && v.scalar_type() == at::kInt && v.dim() == 1 && v.size(0) == x.size(0) && v.is_contiguous()))
        refuse("gated_residual_norms: n_valid must be int32 [G] with x [G, n, width]");
    if (v.defined() && x.size(1) > INT32_MAX) refuse("gated_residual_norms: %lld vertices a graph (under 2^31 with n_valid)", (long long)x.size(1));
    no_tangents({&x, &branch, &gate, &p[0], &p[1], &p[2], &p[3], &p[4]}, "gated_residual_norms");
    one_device({&x, &branch, &gate, &v, &p[0], &p[1], &p[2], &p[3], &p[4]});
    for (Tensor &t : p)
        if (t.defined()) t = (mixed ? t.to(at::kFloat) : t).resolve_neg().contiguous();
    bool train = false;
    if (at::GradMode::is_enabled()) {
        for (const Tensor *t : {&x, &branch, &gate}) train |= t->defined() && t->requires_grad();
        for (const Tensor &t : p) train |= t.defined() && t.requires_grad();
    }
    std::shared_ptr<GatedResidualNormsBackward> node;
    if (train) {
        node = std::shared_ptr<GatedResidualNormsBackward>(new GatedResidualNormsBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(x, branch, gate, p[0], p[1], p[2], p[3], p[4]));
        before_capture(node->next_edges(), "gated_residual_norms");
    }
    NormsResult r = norms_forward(c, x, branch, gate, train, keep8);
    if (train) {
        const bool kept = r.kept[0].defined();
        for (int i = 0; i < 5; ++i) node->params[i] = SavedVariable(p[i], false);
        node->n_valid = SavedVariable(v, false);
        node->stats = SavedVariable(r.stats, false);
        const Tensor given[3] = {x, branch, gate};
        for (int i = 0; i < (kept ? 6 : 3); ++i) node->held[i] = SavedVariable(kept ? r.kept[i] : given[i], false);
        node->shape = at::DimVector(x.sizes());
        node->options = x.options().requires_grad(false);
        if (first) node->param_type = mixed ? at::kFloat : first->scalar_type();
        node->rms = c.rms, node->eps = c.eps, node->kept = kept, node->gated = gate.defined(), node->empty_rows = !r.stats.defined();
        torch::autograd::set_history(r.y, node);
        if (r.h.defined()) torch::autograd::set_history(r.h, node);
    }
    return {r.y, r.h};
}

// ------------------------------------------------------------------------------------------------------------------- scores
struct LabelLogProbsBackward : torch::autograd::Node {
    SavedVariable logits, target, stats;
    at::DimVector shape;
    at::TensorOptions options;
    int64_t ignore = 0;

    std::string name() const override { return "LabelLogProbsBackward"; }
    void release_variables() override
    {
        std::lock_guard<std::mutex> lock(mutex_);
        logits.reset_data();
        target.reset_data();
        stats.reset_data();
    }
    variable_list apply(variable_list &&grads) override
    {
        std::lock_guard<std::mutex> lock(mutex_);
        no_tangents({&grads[0], &grads[1]}, "label_log_probs (backward)");
        variable_list out(1);
        if ((grads[0].defined() || grads[1].defined()) && task_should_compute_output(0)) {
            at::AutoDispatchBelowADInplaceOrView raw;
            const char *const who = "label_log_probs (backward)";
            const c10::Device place = options.device();
            const int64_t n = shape.back(), rows = rows_in(shape);
            const Tensor x = unpack(logits, at::typeMetaToScalarType(options.dtype()), shape, place, who);
            const Tensor t = unpack_whole(target, at::kLong, at::IntArrayRef(shape).slice(0, shape.size() - 1), place, who);
            const Tensor s = unpack_whole(stats, at::kFloat, {rows, 3}, place, who);
            const c10::DeviceGuard device(x.device());
            out[0] = empty(x.sizes(), x, x.scalar_type());
            if (rows) {
                Tensor g[2];
                for (int i = 0; i < 2; ++i)
                    if (grads[i].defined()) g[i] = grads[i].to(at::kFloat).resolve_neg().contiguous();
                const Rows r = rows_of(x, n);
                check(lib.scores_backward(pointer(r.t), type_of(x), rows, n, r.stride, (const int64_t *)pointer(t), ignore, (const float *)pointer(s),
                                          (const float *)pointer(g[0]), (const float *)pointer(g[1]), pointer(out[0]), stream_of(x)),
                      "sn_label_log_probs_backward");
            }
        }
        return without_second(*this, grads, std::move(out));
    }
};

struct Scores { Tensor log_probs, entropy, top_log_probs, top_ids; };
Scores label_log_probs(const Tensor &logits, const Tensor &given, int64_t topk, int64_t ignore)
{
    if (!logits.defined() || type_of(logits) < 0 || logits.dim() < 1) refuse("label_log_probs: expected float32, bfloat16 or float16 logits");
    const at::IntArrayRef lead = logits.sizes().slice(0, logits.dim() - 1);
    if (!given.defined() || given.scalar_type() != at::kLong || given.sizes() != lead)
        refuse("label_log_probs: expected an int64 target of shape %s", shown(lead).c_str());
    const int64_t n = logits.size(-1), rows = given.numel();
    if (n < 1 || n >= 1 << 30 || rows >= 1 << 24) refuse("label_log_probs: %lld rows of %lld entries", (long long)rows, (long long)n);
    if (topk < 0 || topk > n || topk > SN_SCORES_MAX_TOP)
        refuse("label_log_probs: %lld alternatives of %lld entries (at most %d)", (long long)topk, (long long)n, SN_SCORES_MAX_TOP);
    no_tangents({&logits}, "label_log_probs");
    one_device({&logits, &given});
    std::shared_ptr<LabelLogProbsBackward> node;
    if (at::GradMode::is_enabled() && logits.requires_grad()) {
        node = std::shared_ptr<LabelLogProbsBackward>(new LabelLogProbsBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(logits));
        before_capture(node->next_edges(), "label_log_probs");
    }
    Scores o;
    Tensor target, stats;
    {
        at::AutoDispatchBelowADInplaceOrView raw;
        const c10::DeviceGuard device(logits.device());
        target = given.contiguous();
        o.log_probs = empty(lead, logits, at::kFloat);
        o.entropy = empty(lead, logits, at::kFloat);
        if (node) stats = empty({rows, 3}, logits, at::kFloat);             // what the backward pass reads
        if (topk) {
            std::vector<int64_t> sizes = lead.vec();
            sizes.push_back(topk);
            o.top_log_probs = empty(sizes, logits, at::kFloat);
            o.top_ids = empty(sizes, logits, at::kLong);
        }
        if (rows) {
            before_launch();
            const Rows r = rows_of(logits, n);
            const size_t size = lib.scores_workspace(rows, n, (int)topk);
            Tensor workspace;
            if (size) workspace = empty({(int64_t)size}, logits, at::kByte);
            check(lib.scores(pointer(r.t), type_of(logits), rows, n, r.stride, (const int64_t *)pointer(target), ignore, (int)topk, (float *)pointer(o.log_probs),
                             (float *)pointer(o.entropy), (float *)pointer(stats), (float *)pointer(o.top_log_probs), (int64_t *)pointer(o.top_ids),
                             pointer(workspace), size, stream_of(logits)),
                  "sn_label_log_probs");
        }
    }
    if (node) {
        node->logits = SavedVariable(logits, false);
        node->target = SavedVariable(target, false);
        node->stats = SavedVariable(stats, false);
        node->shape = at::DimVector(logits.sizes());
        node->options = logits.options().requires_grad(false);
        node->ignore = ignore;
        torch::autograd::set_history(o.log_probs, node);
        torch::autograd::set_history(o.entropy, node);
    }
    return o;
}

// ------------------------------------------------------------------------------------------------------- 8-bit checkpoints
// the entry points' own limits, tested here too: they see the numbers as 32-bit ones
constexpr int64_t kMostFeatures = 1 << 30, kMostProduct = 1 << 20;

std::pair<Tensor, Tensor> checkpoint8(const Tensor &x)
{
    if (!x.defined() || type_of(x) < 0) refuse("checkpoint8: expected a float32, bfloat16 or float16 tensor");
    if (x.dim() < 1 || x.size(-1) < 1) refuse("checkpoint8: expected at least one feature, got shape %s", shown(x.sizes()).c_str());
    if (x.size(-1) > kMostFeatures) refuse("checkpoint8: %lld features (at most 2^30)", (long long)x.size(-1));
    one_device({&x});
    at::AutoDispatchBelowADInplaceOrView raw;
    const c10::DeviceGuard device(x.device());
    const int64_t n = x.size(-1), rows = rows_in(x.sizes()), npad = (n + 31) / 32 * 32;
    std::pair<Tensor, Tensor> kept(empty({rows, npad}, x, at::kChar), empty({rows, npad / 32}, x, at::kByte));
    if (rows) {
        before_launch();
        const Rows r = rows_of(x, n);
        check(lib.checkpoint8(pointer(r.t), type_of(x), rows, (int)n, r.stride, pointer(kept.first), pointer(kept.second), stream_of(x)), "sn_checkpoint8");
    }
    return kept;
}

Tensor restore(const Tensor &codes, const Tensor &exps, at::IntArrayRef shape, at::ScalarType type)
{
    if (type_of(type) < 0) refuse("checkpoint8: cannot restore to %s", c10::toString(type));
    if (shape.back() > kMostFeatures) refuse("checkpoint8: %lld features (at most 2^30)", (long long)shape.back());
    check_kept(codes, exps, shape);
    one_device({&codes, &exps});
    at::AutoDispatchBelowADInplaceOrView raw;
    const c10::DeviceGuard device(codes.device());
    Tensor out = empty(shape, codes, type);
    if (out.numel()) {
        before_launch();
        check(lib.restore(pointer(codes), pointer(exps), codes.size(0), (int)shape.back(), pointer(out), type_of(type), stream_of(codes)),
              "sn_checkpoint8_restore");
    }
    return out;
}

std::pair<Tensor, Tensor> weight_grad(const Tensor &dy, const Tensor &codes, const Tensor &exps, at::IntArrayRef shape, bool bias, std::optional<at::ScalarType> wanted)
{
    if (!dy.defined() || type_of(dy) < 0) refuse("checkpoint8_weight_grad: expected float32, bfloat16 or float16 gradients");
    const at::ScalarType type = wanted ? *wanted : dy.scalar_type();
    if (type_of(type) < 0) refuse("checkpoint8_weight_grad: cannot write %s", c10::toString(type));
    if (dy.dim() < 2 || dy.size(-1) < 1 || dy.sizes().slice(0, dy.dim() - 1) != shape.slice(0, shape.size() - 1))
        refuse("checkpoint8_weight_grad: gradients %s do not fit the activation %s", shown(dy.sizes()).c_str(), shown(shape).c_str());
    if (dy.size(-1) > kMostProduct || shape.back() > kMostProduct)
        refuse("checkpoint8_weight_grad: %lld x %lld features (at most 2^20 each)", (long long)dy.size(-1), (long long)shape.back());
    if (rows_in(shape) > INT32_MAX) refuse("checkpoint8_weight_grad: %lld rows (under 2^31)", (long long)rows_in(shape));
    check_kept(codes, exps, shape);
    no_tangents({&dy}, "checkpoint8_weight_grad");
    one_device({&dy, &codes, &exps});
    at::AutoDispatchBelowADInplaceOrView raw;
    const c10::DeviceGuard device(dy.device());
    const int64_t out_f = dy.size(-1), in_f = shape.back(), rows = codes.size(0);
    Tensor dw = empty({out_f, in_f}, dy, type), db;
    if (bias) db = empty({out_f}, dy, type);
    if (rows == 0) {
        dw.zero_();
        if (bias) db.zero_();
        return {dw, db};
    }
    before_launch();
    const Rows r = rows_of(dy, out_f);
    const size_t size = lib.weight_grad_workspace(rows, (int)out_f, (int)in_f, type_of(dy));
    const Tensor workspace = empty({(int64_t)std::max<size_t>(size, 16)}, dy, at::kByte);
    check(lib.weight_grad(pointer(r.t), type_of(dy), r.stride, pointer(codes), pointer(exps), rows, (int)out_f, (int)in_f, pointer(dw), pointer(db), type_of(type),
                          pointer(workspace), size, stream_of(dy)),
          "sn_checkpoint8_weight_grad");
    return {dw, db};
}

// ------------------------------------------------------------------------------------------------------- Python's side of it
// (None, or whatever is no tensor: undefined; `what`: what is refused then, nullptr: left to the operator's own check)
Tensor tensor(PyObject *o, const char *what = nullptr)
{
    if (THPVariable_Check(o)) return THPVariable_Unpack(o);
    if (o != Py_None && what) refuse("%s", what);
    return Tensor();
}
PyObject *python(const Tensor &t)
{
    if (!t.defined()) Py_RETURN_NONE;
    PyObject *o = THPVariable_Wrap(t);
    if (!o) throw python_error();
    return o;
}
template <class... T> PyObject *python_tuple(const T &...ts)
{
    PyObject *all = PyTuple_New(sizeof...(ts));
    if (!all) throw python_error();
    Py_ssize_t i = 0;
    try {
        (PyTuple_SET_ITEM(all, i++, python(ts)), ...);
    } catch (...) {
        Py_DECREF(all);
        throw;
    }
    return all;
}
int64_t integer(PyObject *o)
{
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
}
bool truth(PyObject *o)
{
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw python_error();
    return v != 0;
}
std::vector<int64_t> sizes(PyObject *o)
{
    if (!PyTuple_Check(o)) refuse("expected a tuple of sizes");
    std::vector<int64_t> v;
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(o); ++i) v.push_back(integer(PyTuple_GET_ITEM(o, i)));
    return v;
}
std::optional<at::ScalarType> scalar_type(PyObject *o)
{
    if (o == Py_None) return std::nullopt;
    if (!THPDtype_Check(o)) refuse("expected a torch.dtype");
    return reinterpret_cast<THPDtype *>(o)->scalar_type;
}

// (count: what the Python side passes; C++ exceptions end here, each as the Python one that torch makes of it: torch.OutOfMemoryError,
// whatever a hook for saved tensors raised, NotImplementedError, RuntimeError)
template <class F> PyObject *guarded(Py_ssize_t got, Py_ssize_t count, F body)
{
    HANDLE_TH_ERRORS
    if (got != count) refuse("expected %d arguments, got %d", (int)count, (int)got);
    return body();
    END_HANDLE_TH_ERRORS
}

PyObject *py_norms(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    return guarded(n, 12, [&] {
        const char *const parameters = "gated_residual_norms: parameters must be tensors";
        NormsCall c;
        c.rms = truth(a[8]);
        const double eps = PyFloat_AsDouble(a[9]);
        if (eps == -1.0 && PyErr_Occurred()) throw python_error();
        c.eps = (float)eps;
        c.n_valid = tensor(a[10], "gated_residual_norms: n_valid must be int32 [G] with x [G, n, width]");
        for (int i = 0; i < 5; ++i) c.params[i] = tensor(a[3 + i], parameters);
        const auto r = gated_residual_norms(tensor(a[0]), tensor(a[1]), tensor(a[2], "gated_residual_norms: gate must be a tensor of x's shape and type"), c, truth(a[11]));
        return python_tuple(r.first, r.second);
    });
}
PyObject *py_scores(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    return guarded(n, 4, [&] {
        const Scores s = label_log_probs(tensor(a[0]), tensor(a[1]), integer(a[2]), integer(a[3]));
        return python_tuple(s.log_probs, s.entropy, s.top_log_probs, s.top_ids);
    });
}
PyObject *py_checkpoint8(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    return guarded(n, 1, [&] {
        const auto kept = checkpoint8(tensor(a[0]));
        return python_tuple(kept.first, kept.second);
    });
}
PyObject *py_restore(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    return guarded(n, 4, [&] {
        const auto type = scalar_type(a[3]);
        if (!type) refuse("expected a torch.dtype");
        return python(restore(tensor(a[0]), tensor(a[1]), sizes(a[2]), *type));
    });
}
PyObject *py_weight_grad(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    return guarded(n, 6, [&] {
        const auto r = weight_grad(tensor(a[0]), tensor(a[1]), tensor(a[2]), sizes(a[3]), truth(a[4]), scalar_type(a[5]));
        return python_tuple(r.first, r.second);
    });
}

// before_capture(x, weight, bias) of linear_checkpoint8, whose node is Python's
PyObject *py_before_capture(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    return guarded(n, 3, [&]() -> PyObject * {
        if (at::GradMode::is_enabled()) before_capture(torch::autograd::collect_next_edges(tensor(a[0]), tensor(a[1]), tensor(a[2])), "linear_checkpoint8");
        Py_RETURN_NONE;
    });
}

// bind(addresses of the entry points in Library's order, what to call before the first launch)
PyObject *py_bind(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    return guarded(n, 2, [&]() -> PyObject * {
        if (!PyTuple_Check(a[0]) || PyTuple_GET_SIZE(a[0]) != kEntries) refuse("bind: expected %d entry points", (int)kEntries);
        void *entries[kEntries];
        for (Py_ssize_t i = 0; i < kEntries; ++i) entries[i] = (void *)integer(PyTuple_GET_ITEM(a[0], i));
        memcpy(&lib, entries, sizeof lib);
        Py_INCREF(a[1]);
        Py_XSETREF(require_gpu, a[1]);
        Py_RETURN_NONE;
    });
}

#define SN_METHOD(name, function) {name, (PyCFunction)(void (*)(void))function, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {SN_METHOD("bind", py_bind),
                         SN_METHOD("gated_residual_norms", py_norms),
                         SN_METHOD("label_log_probs", py_scores),
                         SN_METHOD("checkpoint8", py_checkpoint8),
                         SN_METHOD("restore", py_restore),
                         SN_METHOD("weight_grad", py_weight_grad),
                         SN_METHOD("before_capture", py_before_capture),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_schemanet_blocks", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__schemanet_blocks() { return PyModule_Create(&module); }
