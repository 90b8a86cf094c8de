// The host's side of the calls whose launches take less time than Python's share of them: int8 linear layers with their
// autograd node, and the AdamW step with its look at every weight and gradient.  A Python extension on torch's C++ interface
// over the C ABI of the library; it allocates, checks and launches, and keeps nothing from one call for the next but an
// optimizer's plan.  (From Python over ctypes: one token through a 4096 x 4096 layer 12.3 us a call of which the GPU works 8.5,
// a small training step 139 us, a step over 62 tensors 51 us.)
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <cstdlib>
#include <cstring>

#include "../../include/rexsc_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

int code_of(at::ScalarType t)
{
    return t == at::kFloat ? REXSC_F32 : t == at::kHalf ? REXSC_F16 : t == at::kBFloat16 ? REXSC_BF16 : -1;
}
at::ScalarType kept_type(at::ScalarType t) { return code_of(t) < 0 ? at::kFloat : t; }

void check(int rc, const char *what)
{
    if (rc == REXSC_OK) return;
    const char *name = rc == REXSC_E_BAD_ARG       ? "REXSC_E_BAD_ARG"
                       : rc == REXSC_E_UNSUPPORTED ? "REXSC_E_UNSUPPORTED"
                       : rc == REXSC_E_WORKSPACE   ? "REXSC_E_WORKSPACE"
                       : rc == REXSC_E_TOO_LONG    ? "REXSC_E_TOO_LONG"
                       : rc == REXSC_E_CUDA        ? "REXSC_E_CUDA"
                       : rc == REXSC_E_DEVICE_TIMEOUT ? "REXSC_E_DEVICE_TIMEOUT"
                                                      : "error";
    TORCH_CHECK_VALUE(rc != REXSC_E_BAD_ARG && rc != REXSC_E_UNSUPPORTED && rc != REXSC_E_TOO_LONG, what, ": ", name);
    TORCH_CHECK(false, what, ": ", name, rc == REXSC_E_CUDA ? ": " : "", rc == REXSC_E_CUDA ? rexsc_last_cuda_error() : "");
}

// Whether two sets of strides put the elements of a tensor in the same places (those of dimensions of one element do not matter)
bool same_places(at::IntArrayRef sizes, at::IntArrayRef a, at::IntArrayRef b)
{
    if (sizes.size() != a.size() || a.size() != b.size()) return false;
    for (size_t i = 0; i < a.size(); i++)
        if (sizes[i] != 1 && a[i] != b[i]) return false;
    return true;
}

void *stream_of(const at::Device &d) { return c10::cuda::getCurrentCUDAStream(d.index()).stream(); }

// (views that stand for the negative of what lies in memory, as the imaginary part of a conjugate does, are written out)
Tensor as_stored(const Tensor &t) { return t.is_neg() ? t.resolve_neg() : t; }

// t as [rows, cols] whose rows are dense, in a type that the kernels read (a view where that is possible)
Tensor rows_of(const Tensor &given, int64_t cols)
{
    const Tensor t = as_stored(given);
    if (t.dim() == 2 && code_of(t.scalar_type()) >= 0 && (t.stride(1) == 1 || cols == 1)) return t;
    Tensor r = code_of(t.scalar_type()) >= 0 ? t : t.to(at::kFloat);
    if (r.dim() != 2) r = r.reshape({-1, cols});
    return r.stride(1) == 1 || cols == 1 ? r : r.contiguous();
}

// With REXSC_B200_DEBUG=1, behind a product: whether a bounded wait gave up (the call synchronises; not during a capture)
void check_waits(const at::Device &d, const char *what)
{
    static const bool debug = [] {
        const char *v = std::getenv("REXSC_B200_DEBUG");
        return v && std::strcmp(v, "1") == 0;
    }();
    if (debug && c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None)
        check(rexsc_int8_status(stream_of(d)), what);
}

int64_t tile_bytes(int64_t rows, int64_t cols) { return (rows + 127) / 128 * ((cols + 127) / 128) * 16384; }
int64_t scale_bytes(int64_t rows) { return (rows + 63) / 64 * 256; }

Tensor bytes(int64_t n, const at::Device &d) { return at::empty({n}, at::TensorOptions().dtype(at::kByte).device(d)); }

struct Bias {
    Tensor kept;
    const void *ptr = nullptr;
    int dtype = 0;
    Bias(const Tensor &bias, int64_t n, const at::Device &d)
    {
        if (!bias.defined()) return;
        TORCH_CHECK_VALUE(bias.device() == d && bias.dim() == 1 && bias.size(0) == n && bias.is_floating_point(),
                          "int8_linear: expected a floating-point bias [", n, "] on ", d);
        kept = as_stored(code_of(bias.scalar_type()) >= 0 ? bias : bias.to(at::kFloat)).contiguous();
        ptr = kept.data_ptr();
        dtype = code_of(kept.scalar_type());
    }
};

std::vector<int64_t> with_last(const Tensor &x, int64_t n)
{
    std::vector<int64_t> s = x.sizes().vec();
    s.back() = n;
    return s;
}

// ---- training: both operands quantised in the call, gradients as products of 8-bit integers -------------------------
struct Int8Linear : public torch::autograd::Function<Int8Linear> {
    // no weight: prepared weights (data, scale)
    using Maybe = std::optional<Tensor>;
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Maybe &weight_, const Maybe &data_, const Maybe &scale_,
                          const Maybe &bias_, int64_t n, int64_t k, int64_t kernel)
    {
        const Tensor weight = weight_.value_or(Tensor()), data = data_.value_or(Tensor()), scale = scale_.value_or(Tensor());
        const Tensor bias = bias_.value_or(Tensor());
        const at::Device dev = x.device();
        const bool want_x = x.requires_grad(), want_w = weight.defined() && weight.requires_grad();
        const bool want_b = bias.defined() && bias.requires_grad();
        const Tensor x2 = rows_of(x, k);
        const int64_t m = x2.size(0), code = code_of(x2.scalar_type());
        // (made in its final shape: a view made here could not be written to in place)
        Tensor y = at::empty(with_last(x, n), x2.options());
        Tensor buf;
        int64_t at_w = 0;
        if (m > 0) {
            // both quantised operands with their scales in one buffer
            at_w = tile_bytes(m, k) + scale_bytes(m);
            buf = bytes(at_w + (weight.defined() ? tile_bytes(n, k) + scale_bytes(n) : 0), dev);
            int8_t *const base = reinterpret_cast<int8_t *>(buf.data_ptr());
            const Tensor w2 = weight.defined() ? rows_of(weight, k) : Tensor();
            const Bias b(bias, n, dev);
            int8_t *const wq = weight.defined() ? base + at_w : reinterpret_cast<int8_t *>(data.data_ptr());
            float *const ws = weight.defined() ? reinterpret_cast<float *>(wq + tile_bytes(n, k)) : scale.data_ptr<float>();
            check(rexsc_int8_linear_train_fwd(x2.data_ptr(), code, m, k, x2.stride(0), weight.defined() ? w2.data_ptr() : nullptr,
                                              weight.defined() ? code_of(w2.scalar_type()) : 0, n,
                                              weight.defined() ? w2.stride(0) : 0, b.ptr, b.dtype, base,
                                              reinterpret_cast<float *>(base + tile_bytes(m, k)), wq, ws, y.data_ptr(), code,
                                              (int)kernel, stream_of(dev)),
                  "rexsc_int8_linear_train_fwd");
            check_waits(dev, "int8_linear (device status)");
            if (weight.defined() && want_x && !want_w) { // the activations are not needed again: only the weights stay
                buf = buf.slice(0, at_w).clone();
                at_w = 0;
            }
        }
        ctx->save_for_backward({buf, weight.defined() ? Tensor() : data, weight.defined() ? Tensor() : scale});
        ctx->saved_data["sizes"] = std::vector<int64_t>{m, n, k, kernel, at_w, want_x, want_w, want_b,
                                                        (int64_t)x.scalar_type(),
                                                        (int64_t)(weight.defined() ? weight.scalar_type() : at::kFloat),
                                                        (int64_t)(bias.defined() ? bias.scalar_type() : at::kFloat)};
        ctx->saved_data["shape"] = x.sizes().vec();
        return y;
    }

    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        const auto sizes = ctx->saved_data["sizes"].toIntVector();
        const int64_t m = sizes[0], n = sizes[1], k = sizes[2], kernel = sizes[3], at_w = sizes[4];
        const bool want_x = sizes[5], want_w = sizes[6], want_b = sizes[7];
        const auto xt = (at::ScalarType)sizes[8], wt = (at::ScalarType)sizes[9], bt = (at::ScalarType)sizes[10];
        const auto shape = ctx->saved_data["shape"].toIntVector();
        variable_list out(8);
        Tensor &dx = out[0], &dw = out[1], &db = out[4];
        {
            at::NoGradGuard no_grad;
            const Tensor &dy = grads[0];
            const at::Device dev = dy.device();
            c10::cuda::CUDAGuard guard(dev);
            const auto options = [&](at::ScalarType t) { return at::TensorOptions().dtype(kept_type(t)).device(dev); };
            if (m == 0) {
                if (want_x) dx = at::zeros(shape, options(xt));
                if (want_w) dw = at::zeros({n, k}, options(wt));
                if (want_b) db = at::zeros({n}, options(bt));
            } else {
                const auto saved = ctx->get_saved_variables();
                const int8_t *const base = static_cast<const int8_t *>(saved[0].data_ptr());
                const int8_t *wq = base + at_w;
                const float *ws = reinterpret_cast<const float *>(wq + tile_bytes(n, k));
                if (saved[1].defined()) wq = static_cast<const int8_t *>(saved[1].data_ptr()), ws = saved[2].data_ptr<float>();
                const Tensor g = rows_of(dy, n);
                if (want_x) dx = at::empty(shape, options(xt));
                if (want_w) dw = at::empty({n, k}, options(wt));
                if (want_b) db = at::empty({n}, options(bt));
                const auto ptr = [](const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; };
                const auto code = [](const Tensor &t) { return t.defined() ? code_of(t.scalar_type()) : 0; };
                const size_t nbytes = rexsc_int8_linear_bwd_workspace_size(m, n, want_x, want_w, want_b);
                const Tensor scratch = bytes((int64_t)nbytes, dev);
                check(rexsc_int8_linear_bwd(g.data_ptr(), code_of(g.scalar_type()), m, n, k, g.stride(0), base,
                                            reinterpret_cast<const float *>(base + tile_bytes(m, k)), wq, ws, ptr(dx), code(dx),
                                            ptr(dw), code(dw), ptr(db), code(db), (int)kernel, scratch.data_ptr(), nbytes,
                                            stream_of(dev)),
                      "rexsc_int8_linear_bwd");
                check_waits(dev, "int8_linear's gradients (device status)");
            }
            if (want_x && dx.scalar_type() != xt) dx = dx.to(xt);
            if (want_w && dw.scalar_type() != wt) dw = dw.to(wt);
            if (want_b && db.scalar_type() != bt) db = db.to(bt);
        }
        if (at::GradMode::is_enabled()) { // a graph of the backward pass is asked for: its nodes raise when they are used
            variable_list some;
            for (auto &t : out)
                if (t.defined()) some.push_back(t.detach().set_requires_grad(true));
            auto later = std::make_shared<torch::autograd::DelayedError>("int8_linear has no second derivative", (int64_t)some.size());
            some = (*later)(std::move(some));
            size_t i = 0;
            for (auto &t : out)
                if (t.defined()) t = some[i++];
        }
        return out;
    }
};

bool has_tangent(const Tensor &t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }

// weight: floating point [n, k], or undefined with data and scale of weights quantised before
Tensor int8_linear(const Tensor &x, const std::optional<Tensor> &weight_, const std::optional<Tensor> &data_,
                   const std::optional<Tensor> &scale_, int64_t n, int64_t k, const std::optional<Tensor> &bias_, int64_t kernel)
{
    const Tensor weight = weight_.value_or(Tensor()), data = data_.value_or(Tensor()), scale = scale_.value_or(Tensor());
    const Tensor bias = bias_.value_or(Tensor());
    const bool prepared = data.defined();
    // a trace would record the output's allocation and not the launches; a tangent would be lost, which reads as a slope of 0
    TORCH_CHECK_NOT_IMPLEMENTED(!torch::jit::tracer::isTracing(), "int8_linear cannot be traced");
    TORCH_CHECK_NOT_IMPLEMENTED(!c10::AutogradState::get_tls_state().get_fw_grad_mode() ||
                                    !(has_tangent(x) || has_tangent(weight) || has_tangent(bias)),
                                "int8_linear has no forward-mode derivative");
    TORCH_CHECK(x.is_cuda(), "int8_linear: expected a CUDA tensor (rexsc_b200 has no CPU path)");
    if (!prepared) {
        TORCH_CHECK(weight.is_cuda(), "int8_linear: expected a CUDA tensor (rexsc_b200 has no CPU path)");
        TORCH_CHECK_VALUE(weight.dim() == 2 && weight.is_floating_point(),
                          "int8_linear: expected a floating-point weight [n, k] or an Int8Matrix");
        n = weight.size(0), k = weight.size(1);
    } else {
        TORCH_CHECK_VALUE(n > 0 && k > 0 && data.is_cuda() && data.scalar_type() == at::kChar && data.is_contiguous() &&
                              data.numel() >= tile_bytes(n, k) && scale.defined() && scale.device() == data.device() &&
                              scale.scalar_type() == at::kFloat && scale.is_contiguous() && scale.numel() >= n,
                          "int8_linear: an Int8Matrix whose data or scale does not fit its size");
    }
    const at::Device dev = (prepared ? data : weight).device();
    TORCH_CHECK_VALUE(x.device() == dev, "int8_linear: x is on ", x.device(), ", the weights are on ", dev);
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) == k && n > 0 && k > 0 && x.is_floating_point(),
                      "int8_linear: expected floating-point x [..., ", k, "] for weights [", n, ", ", k, "], neither of them 0");
    TORCH_CHECK_VALUE(k <= REXSC_INT8_MAX_DOT, "int8_linear: sums of more than ", REXSC_INT8_MAX_DOT,
                      " products are not supported (k = ", k, ")");
    c10::cuda::CUDAGuard guard(dev);
    const bool wx = x.requires_grad(), ww = !prepared && weight.requires_grad(), wb = bias.defined() && bias.requires_grad();
    if (at::GradMode::is_enabled() && (wx || ww || wb)) {
        TORCH_CHECK_VALUE(!wx || n <= REXSC_INT8_MAX_DOT, "int8_linear: the gradient of x sums over ", n,
                          " output channels, at most ", REXSC_INT8_MAX_DOT);
        TORCH_CHECK_VALUE(!ww || x.numel() / k <= REXSC_INT8_MAX_DOT, "int8_linear: the weight's gradient sums over ",
                          x.numel() / k, " tokens, at most ", REXSC_INT8_MAX_DOT);
        const Bias valid(bias, n, dev);
        return Int8Linear::apply(x, weight_, data_, scale_, bias_, n, k, kernel);
    }
    at::NoGradGuard no_grad;
    const Tensor x2 = rows_of(x, k);
    const int64_t m = x2.size(0);
    const int code = code_of(x2.scalar_type());
    const Bias b(bias, n, dev);
    Tensor y = at::empty(with_last(x, n), x2.options());
    if (m > 0) {
        void *const st = stream_of(dev);
        Tensor kept;
        const int8_t *wq;
        const float *ws;
        if (prepared) {
            wq = static_cast<const int8_t *>(data.data_ptr()), ws = scale.data_ptr<float>();
        } else {
            const Tensor w2 = rows_of(weight, k);
            kept = bytes(tile_bytes(n, k) + scale_bytes(n), dev);
            int8_t *const q = reinterpret_cast<int8_t *>(kept.data_ptr());
            float *const s = reinterpret_cast<float *>(q + tile_bytes(n, k));
            check(rexsc_int8_quantize(w2.data_ptr(), code_of(w2.scalar_type()), n, k, w2.stride(0), q, s, st), "rexsc_int8_quantize");
            wq = q, ws = s;
        }
        const size_t nbytes = rexsc_int8_linear_workspace_size(m, n, k, (int)kernel);
        const Tensor scratch = nbytes ? bytes((int64_t)nbytes, dev) : Tensor();
        check(rexsc_int8_linear_fwd(x2.data_ptr(), code, m, k, x2.stride(0), wq, ws, n, b.ptr, b.dtype, y.data_ptr(), code,
                                    (int)kernel, nbytes ? scratch.data_ptr() : nullptr, nbytes, st),
              "rexsc_int8_linear_fwd");
        check_waits(dev, "int8_linear (device status)");
    }
    return y;
}

// ---- AdamW ----------------------------------------------------------------------------------------------------------
// Pieces of memory [first, second) in rising order
using Spans = std::vector<std::pair<uintptr_t, uintptr_t>>;

bool touches(const Spans &spans, uintptr_t begin, uintptr_t end)
{
    const auto at = std::upper_bound(spans.begin(), spans.end(), begin, [](uintptr_t b, const auto &s) { return b < s.second; });
    return at != spans.end() && at->first < end; // (the first one that ends behind `begin`)
}

// What stays of a parameter group between its steps: each parameter's size, strides and place in the flat moment buffers, and
// those buffers.  Pointers, types, sizes and strides of weights and gradients are looked at anew in every step.
class AdamWPlan {
public:
    AdamWPlan(const std::vector<Tensor> &params, int state_bits, const Tensor &step, const Tensor &exp_avg, const Tensor &second,
              const std::optional<Tensor> &scale, const std::optional<Tensor> &second_scale)
        : device_(step.device()), kept_{step, exp_avg, second}
    {
        int64_t first = 0;
        for (const Tensor &p : params) {
            shapes_.push_back({p.numel(), first, p.strides().vec()});
            first += (p.numel() + 255) / 256;
        }
        for (size_t i = 0; i < params.size(); i++) by_address_.push_back((uint32_t)i);
        std::sort(by_address_.begin(), by_address_.end(), [&](uint32_t a, uint32_t b) {
            return reinterpret_cast<uintptr_t>(params[a].data_ptr()) < reinterpret_cast<uintptr_t>(params[b].data_ptr());
        });
        d_.state_bits = state_bits;
        d_.d_step = step.data_ptr<int64_t>();
        d_.d_exp_avg = exp_avg.data_ptr();
        d_.d_exp_avg_sq = second.data_ptr();
        if (scale) {
            kept_.push_back(*scale);
            kept_.push_back(*second_scale);
            d_.d_exp_avg_scale = scale->data_ptr<float>();
            d_.d_exp_avg_sq_scale = second_scale->data_ptr<float>();
        }
    }

    void step(const std::vector<Tensor> &params, double lr, const std::optional<Tensor> &lr_tensor, double beta1, double beta2,
              double eps, double weight_decay, const std::optional<Tensor> &grad_scale, const std::optional<Tensor> &found_inf) const
    {
        at::NoGradGuard no_grad;
        c10::cuda::CUDAGuard guard(device_);
        std::vector<Tensor> kept, changed;
        std::vector<int> place(params.size(), -1); // in the table
        bool lone = true;                          // no gradient shares its storage with any other tensor
        std::vector<rexsc_adamw_tensor> table;
        std::vector<int> kinds;
        table.reserve(params.size());
        changed.reserve(params.size());
        kinds.reserve(params.size());
        TORCH_CHECK_VALUE(params.size() == shapes_.size(), "AdamW: a parameter group has changed");
        for (size_t i = 0; i < params.size(); i++) {
            const Tensor &p = params[i];
            const Shape &s = shapes_[i];
            Tensor g = p.grad();
            if (!g.defined() || s.numel == 0) continue;
            TORCH_CHECK_VALUE(p.layout() == at::kStrided && p.numel() == s.numel && same_places(p.sizes(), p.strides(), s.strides) &&
                                  p.device() == device_ && !p.is_neg(),
                              "AdamW: a parameter has changed its size, memory format or device");
            const int p_code = code_of(p.scalar_type());
            TORCH_CHECK_VALUE(p_code >= 0, "AdamW: parameters must be float32, float16 or bfloat16 (got ", p.scalar_type(), ")");
            TORCH_CHECK_VALUE(g.layout() == at::kStrided, "AdamW: sparse gradients are not supported");
            if (code_of(g.scalar_type()) < 0) g = g.to(at::kFloat);
            g = as_stored(g);
            if (!same_places(p.sizes(), g.strides(), s.strides) || g.sizes() != p.sizes() || g.device() != device_)
                g = at::empty_strided(p.sizes(), s.strides, g.options().device(device_)).copy_(g);
            table.push_back({p.data_ptr(), g.data_ptr(), s.numel, s.first});
            kinds.push_back(p_code * 4 + code_of(g.scalar_type()));
            place[i] = (int)table.size() - 1;
            lone = lone && g.storage().use_count() == 1;
            kept.push_back(std::move(g)); // (until the launch is on the stream)
            changed.push_back(p);
        }
        if (table.empty()) return;
        keep_apart(table, kinds, place, lone, kept);
        // autograd knows of writes by their versions: a graph that still needs the old weights raises instead of reading new ones
        for (const Tensor &p : changed) torch::autograd::impl::bump_version(p);
        rexsc_adamw_desc d = d_;
        const auto scalar = [&](const std::optional<Tensor> &t) -> const float * {
            if (!t) return nullptr;
            TORCH_CHECK_VALUE(t->numel() == 1, "AdamW: expected one element");
            kept.push_back(as_stored(t->to(device_, at::kFloat)));
            return kept.back().data_ptr<float>();
        };
        d.lr = lr, d.beta1 = beta1, d.beta2 = beta2, d.eps = eps, d.weight_decay = weight_decay;
        d.d_lr = scalar(lr_tensor), d.d_grad_scale = scalar(grad_scale), d.d_found_inf = scalar(found_inf);
        // one call for each pair of types; the last one counts the step
        std::vector<int> distinct;
        for (int kind : kinds)
            if (std::find(distinct.begin(), distinct.end(), kind) == distinct.end()) distinct.push_back(kind);
        std::vector<rexsc_adamw_tensor> part;
        for (size_t j = 0; j < distinct.size(); j++) {
            const std::vector<rexsc_adamw_tensor> *list = &table;
            if (distinct.size() > 1) {
                part.clear();
                for (size_t i = 0; i < table.size(); i++)
                    if (kinds[i] == distinct[j]) part.push_back(table[i]);
                list = &part;
            }
            d.param_dtype = distinct[j] / 4, d.grad_dtype = distinct[j] % 4;
            d.advance = j + 1 == distinct.size();
            check(rexsc_adamw_step(&d, list->data(), (int32_t)list->size(), stream_of(device_)), "rexsc_adamw_step");
        }
    }

private:
    // One launch updates all weights at once and reads all gradients: no two weights may hold the same element, and a gradient
    // that lies in the memory of any of them is read from a copy.  (One with a storage of its own, as a backward pass leaves
    // it, does not.)
    void keep_apart(std::vector<rexsc_adamw_tensor> &table, const std::vector<int> &kinds, const std::vector<int> &place, bool lone,
                    std::vector<Tensor> &grads) const
    {
        const auto span = [&](int i) {
            const uintptr_t at = reinterpret_cast<uintptr_t>(table[i].d_param);
            return std::make_pair(at, at + (uintptr_t)table[i].numel * (kinds[i] / 4 == REXSC_F32 ? 4 : 2));
        };
        // in the order of their memory, unless weights have been given other memory since
        uintptr_t end = 0;
        bool ordered = true;
        for (uint32_t i : by_address_) {
            if (place[i] < 0) continue;
            const auto s = span(place[i]);
            ordered = ordered && s.first >= end;
            end = s.second;
        }
        if (ordered && lone) return;
        Spans spans;
        spans.reserve(table.size());
        for (uint32_t i : by_address_)
            if (place[i] >= 0) spans.push_back(span(place[i]));
        if (!ordered) std::sort(spans.begin(), spans.end());
        for (size_t i = 1; i < spans.size(); i++)
            TORCH_CHECK_VALUE(spans[i - 1].second <= spans[i].first, "AdamW: two parameters share memory");
        const void *apart = nullptr; // a storage that lies apart from all of them: gradients are often pieces of one buffer
        for (size_t i = 0; i < grads.size(); i++) {
            const at::Storage &storage = grads[i].storage();
            if (storage.unsafeGetStorageImpl() == apart) continue;
            const uintptr_t all = reinterpret_cast<uintptr_t>(storage.data()), at = reinterpret_cast<uintptr_t>(grads[i].data_ptr());
            if (!touches(spans, all, all + storage.nbytes())) {
                apart = storage.unsafeGetStorageImpl();
            } else if (touches(spans, at, at + (uintptr_t)grads[i].numel() * grads[i].element_size())) {
                grads[i] = grads[i].clone(at::MemoryFormat::Preserve);
                table[i].d_grad = grads[i].data_ptr();
            }
        }
    }

    struct Shape {
        int64_t numel, first;
        std::vector<int64_t> strides;
    };
    at::Device device_;
    std::vector<Tensor> kept_;
    std::vector<Shape> shapes_;
    std::vector<uint32_t> by_address_; // the parameters in the order of their memory when the plan was made
    rexsc_adamw_desc d_ = {};
};

} // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m)
{
    namespace py = pybind11;
    m.def("int8_linear", &int8_linear, py::call_guard<py::gil_scoped_release>());
    py::class_<AdamWPlan>(m, "AdamWPlan")
        .def(py::init<const std::vector<Tensor> &, int, const Tensor &, const Tensor &, const Tensor &, const std::optional<Tensor> &,
                      const std::optional<Tensor> &>())
        .def("step", &AdamWPlan::step, py::call_guard<py::gil_scoped_release>());
}
