// torch_binding.cpp — the 8-bit training operators on torch tensors (siren_amd/_native.so): argument checks, memory from
// torch's caching allocator, the current stream, and the layer's autograd node, over the C ABI of libsiren_amd.so.
//
// Why not ctypes, as the other entry points: these calls are short. A layer's training step took 233 us of host time
// through Python (of 110 us of kernels: the engine's own thread has to take the interpreter's lock for a Python node),
// an AdamW step over ten tensors 29 us (of 9), a layer for one row 19 us. No kernel is here, and no copy of the C ABI: the
// functions are taken from the library that siren_amd/_lib.py loaded (bind).
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>

#include "../../include/siren_amd.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> MaybeTensor;

struct Library {
    decltype(&siren_last_error) last_error;
    decltype(&siren_fp8_quantize_sources) quantize;
    decltype(&siren_fp8_matmul_ws_bytes) matmul_ws_bytes;
    decltype(&siren_fp8_matmul) matmul;
    decltype(&siren_fp8_linear_ws_bytes) linear_ws_bytes;
    decltype(&siren_fp8_linear) linear;
    decltype(&siren_adamw_scratch_bytes) adamw_scratch_bytes;
    decltype(&siren_adamw_step_each) adamw_step;
} lib;

void bind(const std::map<std::string, uintptr_t>& f) {
#define SIREN_BIND(field, name) lib.field = reinterpret_cast<decltype(lib.field)>(f.at(name))
    SIREN_BIND(last_error, "siren_last_error");
    SIREN_BIND(quantize, "siren_fp8_quantize_sources");
    SIREN_BIND(matmul_ws_bytes, "siren_fp8_matmul_ws_bytes");
    SIREN_BIND(matmul, "siren_fp8_matmul");
    SIREN_BIND(linear_ws_bytes, "siren_fp8_linear_ws_bytes");
    SIREN_BIND(linear, "siren_fp8_linear");
    SIREN_BIND(adamw_scratch_bytes, "siren_adamw_scratch_bytes");
    SIREN_BIND(adamw_step, "siren_adamw_step_each");
#undef SIREN_BIND
}

// a status of the C ABI as the exception that siren_amd/_lib.py raises for it
void check(int32_t rc, const char* what) {
    if (rc == SIREN_OK) return;
    TORCH_CHECK_VALUE(rc != SIREN_EINVAL, what, ": ", lib.last_error());
    TORCH_CHECK(false, what, " failed (", rc, "): ", lib.last_error());
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

int type_code(at::ScalarType t) {
    return t == at::kFloat ? 0 : t == at::kBFloat16 ? 1 : t == at::kHalf ? 2 : -1;
}
int format_code(at::ScalarType t) { return t == at::kFloat8_e4m3fn ? 0 : t == at::kFloat8_e5m2 ? 1 : -1; }

void check_input(const Tensor& x, const char* what) {
    TORCH_CHECK(x.is_cuda(), "siren_amd.fp8 runs on ROCm devices (MI355X) only; got a ", x.device().type(), " tensor as ", what);
    TORCH_CHECK_TYPE(type_code(x.scalar_type()) >= 0, what, " must be fp32, bf16 or fp16; got ", x.scalar_type());
    TORCH_CHECK_TYPE(x.layout() == at::kStrided, what, " must be a dense tensor");
    TORCH_CHECK(!x._fw_grad(0).defined(), "siren_amd.fp8 has no forward-mode derivatives; ", what, " carries a tangent");
}

int64_t blocks(int64_t n) { return (n + 127) / 128; }
int64_t padded(int64_t n) { return blocks(n) * 128; }
int64_t words(int64_t n) { return (blocks(n) + 3) / 4 * 4; }

// A quantised (rows, cols) tensor in memory that someone holds: values in rows (rows, padded cols) or in panels (padded
// cols / 64, rows, 64), and its scales
struct Blocks {
    char *values = nullptr, *scales = nullptr;
    int64_t rows = 0, cols = 0;
    int layout = 0, fmt = 0;
    int64_t value_bytes() const { return rows * padded(cols); }
    int64_t scale_bytes() const { return ((layout & SIREN_FP8_TILES) ? blocks(rows) : rows) * words(cols); }
};

// What the layer makes for itself lies in one allocation, each tensor's values before its scales; those that are not wanted
// (no rows) take nothing
Tensor hold(const Tensor& like, std::initializer_list<Blocks*> all, Tensor memory = Tensor()) {
    int64_t size = 0;
    for (const Blocks* b : all) size += b->value_bytes() + (b->scale_bytes() + 15) / 16 * 16;
    if (!memory.defined() && size > 0) memory = at::empty({size}, like.options().dtype(at::kByte));
    char* at = size > 0 ? (char*)memory.data_ptr() : nullptr;
    for (Blocks* b : all) {
        if (b->rows == 0) continue;
        b->values = at;
        b->scales = at + b->value_bytes();
        at = b->scales + (b->scale_bytes() + 15) / 16 * 16;
    }
    return memory;
}

Blocks plan(int64_t rows, int64_t cols, int layout, int fmt = 0) {
    Blocks b;
    b.rows = rows;
    b.cols = cols;
    b.layout = layout;
    b.fmt = fmt;
    return b;
}

// x as the kernels read it: columns one element apart, rows any distance that does not overlap
Tensor rows_of(const Tensor& x0, int64_t& ld) {
    const Tensor x = x0.is_neg() ? x0.resolve_neg() : x0;  // what a view negates is not so in memory
    const int64_t r = x.size(0), c = x.size(1);
    Tensor y = (c <= 1 || x.stride(1) == 1) && (r <= 1 || x.stride(0) >= c) ? x : x.contiguous();
    ld = r > 1 ? y.stride(0) : c;
    return y;
}

// One pass over x (times mult): its rows (q), its transpose's rows (qt), its column sums, those that have memory
struct Source {
    Tensor x, ws;
    siren_fp8_source arg = {};
    Source(const Tensor& x0, const Blocks& q, const Blocks& qt, const Tensor& mult, Tensor* colsum) {
        x = rows_of(x0, arg.ld);
        const Blocks& any = q.values ? q : qt;
        arg.x = x.data_ptr();
        arg.dtype = type_code(x.scalar_type());
        arg.rows = x.size(0);
        arg.cols = x.size(1);
        arg.mult = mult.defined() ? mult.data_ptr() : nullptr;
        arg.format = any.fmt;
        arg.tiles = (any.layout & SIREN_FP8_TILES) != 0;
        arg.panels = ((q.layout & SIREN_FP8_PANELS) ? 1 : 0) | ((qt.layout & SIREN_FP8_PANELS) ? 2 : 0);
        arg.q = q.values;
        arg.s = q.scales;
        arg.qt = qt.values;
        arg.st = qt.scales;
        if (colsum) {
            const auto f32 = x.options().dtype(at::kFloat);
            if (arg.rows > 128) ws = at::empty({blocks(arg.rows), arg.cols}, f32);
            *colsum = at::empty({arg.cols}, f32);
            arg.colsum_ws = ws.defined() ? ws.data_ptr<float>() : nullptr;
            arg.colsum = colsum->data_ptr<float>();
        }
    }
};

void quantize_into(const Source& a) { check(lib.quantize(&a.arg, 1, stream_of(a.x)), "siren_fp8_quantize"); }
void quantize_into(const Source& a, const Source& b) {
    const siren_fp8_source both[2] = {a.arg, b.arg};
    check(lib.quantize(both, 2, stream_of(a.x)), "siren_fp8_quantize");
}

Tensor product(const Tensor& like, const Blocks& a, const Blocks& b, const Tensor& bias, int act, double omega, at::ScalarType type,
               Tensor* deriv) {
    const auto opt = like.options().dtype(at::kByte);
    Tensor out = at::empty({a.rows, b.rows}, opt.dtype(type));
    // The sine's derivative is kept in 8 bits of mantissa (bf16), half the bytes of fp32 both ways. In dx and dW it meets a
    // gradient that is rounded to 3 bits next. A bias's gradient is not rounded so: each of its terms is off by 2^-8 of itself
    // at most, their sum (in fp32 over 128 rows, in 64 bits over those) by no more.
    if (deriv) *deriv = at::empty({a.rows, b.rows}, opt.dtype(at::kBFloat16));
    int64_t need = 0;
    check(lib.matmul_ws_bytes(a.rows, b.rows, a.cols, &need), "siren_fp8_matmul_ws_bytes");
    Tensor ws;
    if (need) ws = at::empty({need}, opt);
    check(lib.matmul(a.values, a.scales, a.rows, a.layout, a.fmt, b.values, b.scales, b.rows, b.layout, a.cols,
                     bias.defined() ? bias.data_ptr<float>() : nullptr, act, (float)omega, out.data_ptr(), type_code(type),
                     deriv ? deriv->data_ptr() : nullptr, need ? ws.data_ptr() : nullptr, stream_of(like)),
          "siren_fp8_matmul");
    return out;
}

// act(x w^T + bias) in one call of the C ABI; w: rows, tiles
Tensor serve(const Tensor& x0, const Blocks& w, const Tensor& bias, int act, double omega, Tensor* deriv) {
    int64_t ld;
    const Tensor x = rows_of(x0, ld);
    const int64_t m = x.size(0), k = x.size(1);
    Tensor y = at::empty({m, w.rows}, x.options());
    if (deriv) *deriv = at::empty({m, w.rows}, x.options().dtype(at::kBFloat16));
    int64_t need = 0;
    check(lib.linear_ws_bytes(m, w.rows, k, &need), "siren_fp8_linear_ws_bytes");
    Tensor ws;
    if (need) ws = at::empty({need}, x.options().dtype(at::kByte));
    check(lib.linear(x.data_ptr(), type_code(x.scalar_type()), m, k, ld, w.values, w.scales, w.rows,
                     bias.defined() ? bias.data_ptr<float>() : nullptr, act, (float)omega, y.data_ptr(),
                     deriv ? deriv->data_ptr() : nullptr, need ? ws.data_ptr() : nullptr, stream_of(x)),
          "siren_fp8_linear");
    return y;
}

Tensor bias32(const Tensor& bias) {
    if (!bias.defined()) return bias;
    const Tensor b = bias.detach();
    return (b.is_neg() ? b.resolve_neg() : b).to(at::kFloat).contiguous();
}

// Gradients of gradients: the values pass, a backward through them says why there is none
struct NotTwice : torch::autograd::Function<NotTwice> {
    static Tensor forward(AutogradContext*, const Tensor& g, const Tensor&) { return g.detach(); }
    static variable_list backward(AutogradContext*, const variable_list&) {
        TORCH_CHECK(false, "fp8.linear: its gradients are not differentiable again (second derivatives need the fp32 kernels)");
    }
};

// A backward that is captured while an eager graph of the same leaf lives would make the engine wait for that graph's
// stream, which a capture may not: the process ends. The leaf's accumulator tells, so the call is refused instead.
void check_capture(std::initializer_list<const Tensor*> leaves) {
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    for (const Tensor* t : leaves) {
        if (!t->defined() || !t->requires_grad() || t->grad_fn()) continue;
        const auto accumulator = torch::autograd::impl::try_get_grad_accumulator(*t);
        const auto stream = accumulator ? accumulator->stream() : std::nullopt;
        TORCH_CHECK(!stream || stream->id() == c10::hip::getCurrentHIPStream(t->device().index()).id(),
                    "fp8.linear: this capture uses a leaf that an eager graph made on another stream still holds; its backward "
                    "cannot be captured. Delete what that graph returned first, or warm up on the stream that captures");
    }
}

// The backward of y = act(x W^T + b): x was read once in the forward, dy is read once here, each quantised both along its
// rows and along its columns in that pass; the weight's tiles serve both directions. A Node of its own rather than a
// torch::autograd::Function, whose dictionary and bookkeeping cost 4 us of the 88 that a training step of 8 x 128 x 128
// then took (all of it host time, half the engine's own; 76 since x and the weight are one launch and two allocations).
struct LinearBackward : torch::autograd::Node {
    int64_t m = 0, n = 0, k = 0, fmt = 0, kept_bytes = 0;
    at::ScalarType tx = at::kFloat, tw = at::kFloat, tb = at::kFloat;
    Blocks qxt, qwt;                             // x and the weight by their columns, in kept's memory
    torch::autograd::SavedVariable kept, deriv;  // saved as torch saves, so that its hooks (checkpointing) see them

    std::string name() const override { return "Fp8LinearBackward"; }

    void release_variables() override {
        const std::lock_guard<std::mutex> lock(mutex_);
        kept.reset_data();
        deriv.reset_data();
    }

    variable_list apply(variable_list&& grads) override {
        const std::lock_guard<std::mutex> lock(mutex_);
        const bool nx = task_should_compute_output(0), nw = task_should_compute_output(1), nb = task_should_compute_output(2);
        Tensor dx, dw, db;
        const Tensor& dy = grads[0];
        if (!dy.defined() || !(nx || nw || nb)) return {dx, dw, db};
        const auto opt = dy.options();
        if (m == 0) {
            if (nx) dx = at::empty({0, k}, opt.dtype(tx));
            if (nw) dw = at::zeros({n, k}, opt.dtype(tw));
            if (nb) db = at::zeros({n}, opt.dtype(tb));
            return {dx, dw, db};
        }
        const c10::DeviceGuard guard(dy.device());
        const bool create_graph = at::GradMode::is_enabled();
        {
            const at::NoGradGuard no_grad;
            const Tensor g = dy.detach(), memory = kept.unpack(), factor = deriv.unpack();
            Blocks xt = qxt, wt = qwt;
            // a hook may have held them in between
            for (const Tensor* t : {&memory, &factor})
                TORCH_CHECK(!t->defined() || (t->device() == g.device() && t->is_contiguous() && (uintptr_t)t->data_ptr() % 16 == 0),
                            "fp8.linear: a saved tensor came back on ", t->device(), ", or not as it was saved");
            TORCH_CHECK((!memory.defined() || (memory.scalar_type() == at::kByte && memory.numel() == kept_bytes)) &&
                            (!factor.defined() || (factor.scalar_type() == at::kBFloat16 && factor.numel() == m * n)),
                        "fp8.linear: a saved tensor came back with another type or size");
            if (memory.defined()) hold(g, {&xt, &wt}, memory);
            Blocks q = plan(nx ? m : 0, n, SIREN_FP8_PANELS, (int)fmt), qt = plan(nw ? n : 0, m, SIREN_FP8_PANELS, (int)fmt);
            const Tensor own = hold(g, {&q, &qt});
            Tensor sums;
            quantize_into(Source(g, q, qt, factor, nb ? &sums : nullptr));
            if (nx) dx = product(g, q, wt, Tensor(), 0, 0., tx, nullptr);
            if (nw) dw = product(g, qt, xt, Tensor(), 0, 0., tw, nullptr);
            if (nb) db = sums.to(tb);
        }
        if (create_graph) {
            const Tensor anchor = at::empty({0}, opt.dtype(at::kFloat)).requires_grad_(true);
            for (Tensor* g : {&dx, &dw, &db})
                if (g->defined()) *g = NotTwice::apply(*g, anchor);
        }
        return {dx, dw, db};
    }
};

// The backward's products have limits of their own (a sum's length is the forward's rows or outputs, a result's columns its
// inputs): a layer whose gradients the library would refuse is refused before its forward
void check_backward(const Tensor& x, const Tensor& weight) {
    const int64_t m = x.size(0), n = weight.size(0), k = weight.size(1);
    int64_t bytes;
    if (m > 0 && x.requires_grad()) check(lib.matmul_ws_bytes(m, k, n, &bytes), "fp8.linear: the gradient of x");
    if (m > 0 && weight.requires_grad()) check(lib.matmul_ws_bytes(n, k, m, &bytes), "fp8.linear: the gradient of the weight");
}

// y = act(x W^T + b) with gradients
Tensor train(const Tensor& x, const Tensor& weight, const Tensor& bias, int64_t act, double omega, int64_t fmt) {
    const bool nx = x.requires_grad(), nw = weight.requires_grad();
    const std::shared_ptr<LinearBackward> node(new LinearBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x, weight, bias));
    node->m = x.size(0);
    node->n = weight.size(0);
    node->k = weight.size(1);
    node->fmt = fmt;
    node->tx = x.scalar_type();
    node->tw = weight.scalar_type();
    if (bias.defined()) node->tb = bias.scalar_type();
    Tensor y;
    {
        const at::NoGradGuard no_grad;
        if (node->m == 0) {  // no products, gradients of zero
            y = x.new_empty({0, node->n});
        } else {
            const c10::DeviceGuard guard(x.device());
            const Tensor b32 = bias32(bias);
            const int64_t m = node->m, n = node->n, k = node->k;
            int64_t ws = 0;
            check(lib.linear_ws_bytes(m, n, k, &ws), "siren_fp8_linear_ws_bytes");
            const bool few = ws == 0;  // the product quantises its rows itself, and reads the weight in rows
            Blocks qx = plan(few ? 0 : m, k, SIREN_FP8_PANELS), qw = plan(n, k, SIREN_FP8_TILES | (few ? 0 : SIREN_FP8_PANELS));
            const Tensor own = hold(x, {&qx, &qw});
            Blocks &qxt = node->qxt, &qwt = node->qwt;
            qxt = plan(nw ? k : 0, m, SIREN_FP8_PANELS);
            qwt = plan(nx ? k : 0, n, SIREN_FP8_TILES | SIREN_FP8_PANELS);
            const Tensor kept = hold(x, {&qxt, &qwt});
            const Source from_w(weight, qw, qwt, Tensor(), nullptr);
            if (few && !nw)
                quantize_into(from_w);
            else
                quantize_into(Source(x, qx, qxt, Tensor(), nullptr), from_w);
            Tensor d;
            Tensor* deriv = act ? &d : nullptr;
            y = few ? serve(x, qw, b32, (int)act, omega, deriv) : product(x, qx, qw, b32, (int)act, omega, x.scalar_type(), deriv);
            node->kept = torch::autograd::SavedVariable(kept, false);
            node->kept_bytes = kept.defined() ? kept.numel() : 0;
            node->deriv = torch::autograd::SavedVariable(d, false);
        }
    }
    torch::autograd::set_history(y, node);
    return y;
}

Tensor check_layer(const Tensor& x, const Tensor& bias, int64_t n, int64_t k, double omega) {
    check_input(x, "x");
    TORCH_CHECK_VALUE(x.dim() >= 1, "x must be (..., in)");
    TORCH_CHECK_VALUE(n >= 1 && k >= 1, "weight must have rows and columns; got (", n, ", ", k, ")");
    TORCH_CHECK_VALUE(x.size(-1) == k, "x must be (..., ", k, ") for this weight; got ", x.sizes());
    TORCH_CHECK_VALUE(std::isfinite(omega), "omega must be finite");
    if (bias.defined()) {
        check_input(bias, "bias");
        TORCH_CHECK_VALUE(bias.dim() == 1 && bias.size(0) == n && bias.device() == x.device(), "bias must be (", n, ",) on ",
                          x.device(), "; got ", bias.sizes(), " on ", bias.device());
    }
    return x.dim() == 2 ? x : x.reshape({-1, k});
}

Tensor like_input(const Tensor& x, const Tensor& y) {
    if (x.dim() == 2) return y;
    auto shape = x.sizes().vec();
    shape.back() = y.size(1);
    return y.view(shape);
}

Blocks packed_operand(const Tensor& data, const Tensor& scale, int64_t cols, const at::Device& dev, bool tiles_only) {
    TORCH_CHECK(data.is_cuda(), "siren_amd.fp8 runs on ROCm devices (MI355X) only; got a ", data.device().type(), " tensor");
    TORCH_CHECK_TYPE(format_code(data.scalar_type()) >= 0 && scale.scalar_type() == at::kByte,
                     "Blocks are e4m3 or e5m2 with uint8 scales; got ", data.scalar_type(), " and ", scale.scalar_type());
    TORCH_CHECK_VALUE(data.dim() == 2 && scale.dim() == 2 && cols >= 1 && data.size(1) == padded(cols) &&
                          scale.size(1) == words(cols) &&
                          (scale.size(0) == blocks(data.size(0)) || (!tiles_only && scale.size(0) == data.size(0))),
                      "Blocks of ", cols, " columns are quantize()'s: data (rows, ", padded(cols), "), scale (rows or ceil(rows / 128), ",
                      words(cols), ")", tiles_only ? "; a weight is quantize(weight, 'tile')" : "", "; got ", data.sizes(), " and ",
                      scale.sizes());
    TORCH_CHECK_VALUE(data.is_contiguous() && scale.is_contiguous() && (uintptr_t)data.data_ptr() % 16 == 0 &&
                          (uintptr_t)scale.data_ptr() % 4 == 0,
                      "Blocks must be contiguous, their data 16-byte and their scales 4-byte aligned");
    TORCH_CHECK_VALUE(data.device() == dev && scale.device() == dev, "Blocks on ", data.device(), " but the other operand on ", dev);
    // one row is both: its tile is its row block
    Blocks b = plan(data.size(0), cols, tiles_only || scale.size(0) != data.size(0) ? SIREN_FP8_TILES : 0,
                    format_code(data.scalar_type()));
    b.values = (char*)data.data_ptr();
    b.scales = (char*)scale.data_ptr();
    return b;
}

// what the user holds: two tensors
Blocks tensors(const Tensor& like, int64_t rows, int64_t cols, bool tiles, int64_t fmt, Tensor& data, Tensor& scale) {
    Blocks b = plan(rows, cols, tiles ? SIREN_FP8_TILES : 0, (int)fmt);
    data = at::empty({rows, padded(cols)}, like.options().dtype(fmt ? at::kFloat8_e5m2 : at::kFloat8_e4m3fn));
    scale = at::empty({tiles ? blocks(rows) : rows, words(cols)}, like.options().dtype(at::kByte));
    b.values = (char*)data.data_ptr();
    b.scales = (char*)scale.data_ptr();
    return b;
}

void check_matrix(const Tensor& x) {
    check_input(x, "x");
    TORCH_CHECK_VALUE(x.dim() == 2, "x must be (rows, cols); got ", x.sizes());
}

std::pair<Tensor, Tensor> quantize(const Tensor& x, bool tiles, int64_t fmt) {
    check_matrix(x);
    const c10::DeviceGuard guard(x.device());
    Tensor data, scale;
    const Blocks q = tensors(x, x.size(0), x.size(1), tiles, fmt, data, scale);
    quantize_into(Source(x.detach(), q, Blocks(), Tensor(), nullptr));
    return {data, scale};
}

std::vector<Tensor> quantize_both(const Tensor& x, bool tiles, int64_t fmt) {
    check_matrix(x);
    const c10::DeviceGuard guard(x.device());
    Tensor data, scale, tdata, tscale;
    const Blocks q = tensors(x, x.size(0), x.size(1), tiles, fmt, data, scale);
    const Blocks qt = tensors(x, x.size(1), x.size(0), tiles, fmt, tdata, tscale);
    quantize_into(Source(x.detach(), q, qt, Tensor(), nullptr));
    return {data, scale, tdata, tscale};
}

std::pair<Tensor, MaybeTensor> matmul(const Tensor& a, const Tensor& sa, const Tensor& b, const Tensor& sb, int64_t cols,
                                      const MaybeTensor& bias, int64_t act, double omega, at::ScalarType type, bool derivative) {
    const Blocks qa = packed_operand(a, sa, cols, a.device(), false), qb = packed_operand(b, sb, cols, a.device(), false);
    TORCH_CHECK_TYPE(b.scalar_type() == at::kFloat8_e4m3fn, "the second operand must be e4m3; got ", b.scalar_type());
    TORCH_CHECK_TYPE(type_code(type) >= 0, "dtype must be fp32, bf16 or fp16; got ", type);
    TORCH_CHECK_VALUE(std::isfinite(omega), "omega must be finite");
    Tensor b32;
    if (bias) {
        check_input(*bias, "bias");
        TORCH_CHECK_VALUE(bias->dim() == 1 && bias->size(0) == qb.rows && bias->device() == a.device(), "bias must be (", qb.rows, ",)");
        b32 = bias32(*bias);
    }
    const c10::DeviceGuard guard(a.device());
    Tensor d;
    Tensor y = product(a, qa, qb, b32, (int)act, omega, type, derivative ? &d : nullptr);
    return {y, derivative ? MaybeTensor(d) : std::nullopt};
}

Tensor linear_packed(const Tensor& x, const Tensor& data, const Tensor& scale, int64_t cols, const MaybeTensor& maybe_bias,
                     int64_t act, double omega) {
    const Tensor bias = maybe_bias.value_or(Tensor());
    check_input(x, "x");
    const Blocks w = packed_operand(data, scale, cols, x.device(), true);
    TORCH_CHECK_TYPE(data.scalar_type() == at::kFloat8_e4m3fn, "a weight in 8 bits is e4m3; got ", data.scalar_type());
    const Tensor x2 = check_layer(x, bias, w.rows, cols, omega);
    TORCH_CHECK(!(at::GradMode::is_enabled() && (x.requires_grad() || (bias.defined() && bias.requires_grad()))),
                "fp8.linear: a weight held in 8 bits is forward only; use torch.no_grad(), or pass the weight itself to train");
    const c10::DeviceGuard guard(x.device());
    return like_input(x, serve(x2.detach(), w, bias32(bias), (int)act, omega, nullptr));
}

Tensor linear(const Tensor& x, const Tensor& weight, const MaybeTensor& maybe_bias, int64_t act, double omega, int64_t fmt) {
    const Tensor bias = maybe_bias.value_or(Tensor());
    check_input(x, "x");
    check_input(weight, "weight");
    TORCH_CHECK_VALUE(weight.dim() == 2, "weight must be (out, in); got ", weight.sizes());
    TORCH_CHECK_VALUE(weight.device() == x.device(), "weight on ", weight.device(), " but x on ", x.device());
    const Tensor x2 = check_layer(x, bias, weight.size(0), weight.size(1), omega);
    if (at::GradMode::is_enabled() && (x.requires_grad() || weight.requires_grad() || (bias.defined() && bias.requires_grad()))) {
        check_backward(x2, weight);
        check_capture({&x, &weight, &bias});
        return like_input(x, train(x2, weight, bias, act, omega, fmt));
    }
    const c10::DeviceGuard guard(x.device());
    Blocks w = plan(weight.size(0), weight.size(1), SIREN_FP8_TILES);
    const Tensor own = hold(weight, {&w});
    quantize_into(Source(weight.detach(), w, Blocks(), Tensor(), nullptr));
    return like_input(x, serve(x2.detach(), w, bias32(bias), (int)act, omega, nullptr));
}

MaybeTensor adamw_step(const std::vector<Tensor>& params, const std::vector<MaybeTensor>& grads, const Tensor& m, const Tensor& v,
                       const Tensor& step, double lr, double b1, double b2, double eps, double weight_decay,
                       std::optional<double> max_norm, uint64_t seed, const MaybeTensor& sm, const MaybeTensor& sv,
                       const MaybeTensor& counts) {
    const size_t n = params.size();
    TORCH_CHECK_VALUE(n >= 1 && grads.size() == n, "adamw_step needs as many gradients as parameters, one at least; got ",
                      grads.size(), " and ", n);
    const at::Device dev = params[0].device();
    TORCH_CHECK(dev.is_cuda(), "adamw_step runs on ROCm devices (MI355X) only; got a ", dev.type(), " tensor");
    std::vector<void*> ps(n);
    std::vector<const void*> gs(n);
    std::vector<int64_t> numels(n);
    std::vector<int32_t> types(n);
    std::vector<std::pair<uintptr_t, uintptr_t>> spans;
    spans.reserve(n + 6);
    std::vector<Tensor> keep;
    int64_t size = 0;
    for (size_t i = 0; i < n; ++i) {
        const Tensor& p = params[i];
        types[i] = type_code(p.scalar_type());
        TORCH_CHECK(types[i] >= 0 && p.device() == dev, "adamw_step needs fp32, bf16 or fp16 parameters on one device; got ",
                    p.scalar_type(), " on ", p.device());
        TORCH_CHECK_VALUE(p.is_contiguous() && !p.is_neg(), "adamw_step needs contiguous parameters; parameter ", i,
                          " has strides ", p.strides(), p.is_neg() ? " and is a negated view" : "");
        ps[i] = p.data_ptr();
        gs[i] = nullptr;
        if (grads[i]) {
            const Tensor& g = *grads[i];
            TORCH_CHECK_VALUE(g.layout() == at::kStrided && g.sizes() == p.sizes() && g.scalar_type() == p.scalar_type() &&
                                  g.device() == dev,
                              "gradient ", i, " must be ", p.sizes(), " ", p.scalar_type(), " on ", dev, "; got ", g.sizes(), " ",
                              g.scalar_type(), " on ", g.device());
            if (g.is_contiguous() && !g.is_neg()) {
                gs[i] = g.data_ptr();
            } else {
                keep.push_back(g.resolve_neg().contiguous());
                gs[i] = keep.back().data_ptr();
            }
        }
        numels[i] = p.numel();
        if (numels[i] > 0) spans.emplace_back((uintptr_t)ps[i], (uintptr_t)ps[i] + p.nbytes());
        size += padded(numels[i]);
    }
    TORCH_CHECK_VALUE(bool(sm) == bool(sv), "scales must be two tensors");
    const auto want = sm ? at::kFloat8_e4m3fn : at::kFloat;
    const std::pair<const char*, const Tensor*> states[2] = {{"exp_avg", &m}, {"exp_avg_sq", &v}};
    for (const auto& s : states)
        TORCH_CHECK_VALUE(s.second->scalar_type() == want && s.second->numel() == size && s.second->device() == dev &&
                              s.second->is_contiguous() && (uintptr_t)s.second->data_ptr() % 16 == 0,
                          s.first, " must be ", size, " contiguous 16-byte aligned values of ", want, " on ", dev, "; got ",
                          s.second->numel(), " of ", s.second->scalar_type(), " on ", s.second->device());
    if (sm)
        for (const Tensor* s : {&*sm, &*sv})
            TORCH_CHECK_VALUE(s->scalar_type() == at::kByte && s->numel() == size / 128 && s->device() == dev && s->is_contiguous(),
                              "scales must be two tensors of ", size / 128, " contiguous uint8 on ", dev);
    TORCH_CHECK_VALUE(step.scalar_type() == at::kLong && step.numel() == 1 && step.device() == dev, "step must be one int64 on ", dev);
    TORCH_CHECK_VALUE(!counts || (counts->scalar_type() == at::kLong && counts->numel() == (int64_t)n && counts->device() == dev &&
                                  counts->is_contiguous()),
                      "counts must be ", n, " contiguous int64 on ", dev);
    // what is written lies apart: one thread's store must not be another's load
    const auto span = [&](const Tensor& t) {
        if (t.numel() > 0) spans.emplace_back((uintptr_t)t.data_ptr(), (uintptr_t)t.data_ptr() + t.nbytes());
    };
    span(m), span(v), span(step);
    if (sm) span(*sm), span(*sv);
    if (counts) span(*counts);
    std::sort(spans.begin(), spans.end());
    for (size_t i = 1; i < spans.size(); ++i)
        TORCH_CHECK_VALUE(spans[i - 1].second <= spans[i].first,
                          "adamw_step: parameters or states overlap (is a parameter listed twice, a state given for two?)");
    TORCH_CHECK_VALUE(!max_norm || *max_norm > 0., "max_norm must be positive or None; got ", max_norm.value_or(0.));
    int64_t need = 0;
    check(lib.adamw_scratch_bytes((int64_t)n, &need), "siren_adamw_scratch_bytes");
    const c10::DeviceGuard guard(dev);
    const Tensor scratch = at::empty({need / 4}, step.options().dtype(at::kFloat));
    // Written behind autograd's back: a graph that saved a parameter must notice. Before the launch: this is what refuses
    // a parameter made in inference mode
    for (size_t i = 0; i < n; ++i)
        if (gs[i]) torch::autograd::impl::bump_version(params[i]);
    check(lib.adamw_step((int64_t)n, ps.data(), gs.data(), numels.data(), types.data(), sm ? 8 : 32, m.data_ptr(), v.data_ptr(),
                         sm ? sm->data_ptr() : nullptr, sv ? sv->data_ptr() : nullptr, step.data_ptr<int64_t>(),
                         counts ? counts->data_ptr<int64_t>() : nullptr, lr, b1, b2, eps,
                         weight_decay, max_norm.value_or(0.), seed, scratch.data_ptr(), stream_of(step)),
          "siren_adamw_step");
    return max_norm ? MaybeTensor(scratch.select(0, 8)) : std::nullopt;
}

}  // namespace

PYBIND11_MODULE(_native, m) {
    m.def("bind", &bind);
    m.def("quantize", &quantize);
    m.def("quantize_both", &quantize_both);
    m.def("matmul", [](const Tensor& a, const Tensor& sa, const Tensor& b, const Tensor& sb, int64_t cols, const MaybeTensor& bias,
                       int64_t act, double omega, py::object dtype, bool derivative) {
        return matmul(a, sa, b, sb, cols, bias, act, omega, torch::python::detail::py_object_to_dtype(dtype), derivative);
    });
    m.def("linear_packed", &linear_packed);
    m.def("linear", &linear);
    m.def("adamw_step", &adamw_step);
}
