// Host side of the training operators (group_norm_act, class_log_probs, AdamW): argument checks, output allocation, autograd nodes
// and the walk over an optimizer's parameters, in C++.  A group norm's forward and backward pass through nodes written in Python cost
// about 145 us of host time; these take 66 to 69, of which a trivial operation's pass (autograd's hand-over to its thread and back)
// has 43.  Where the two threads get neighbouring cores it is 36, of 23.  The kernels are reached through the C ABI of libermi355.so
// on the current stream of the tensors' device.
//
// On meta and fake tensors the functions give shapes, types and layouts and launch nothing.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>
#include "../../include/erfnet_mi355.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> OptTensor;

static int dtype_code(const Tensor& t, const char* who) {
    if (t.scalar_type() == at::kFloat) return ERF_F32;
    if (t.scalar_type() == at::kBFloat16) return ERF_BF16;
    TORCH_CHECK_TYPE(false, who, ": float32 or bfloat16 tensors, got ", t.dtype());
}

// Whether there is no memory behind a tensor: meta and fake ones.  Other tensors that dispatch to Python have memory of their own
// making, which the kernels do not see: refused.
static bool shape_only(const Tensor& t) {
    if (t.is_meta()) return true;
    if (!t.key_set().has(c10::DispatchKey::Python)) return false;
    py::gil_scoped_acquire gil;
    const py::object o = py::reinterpret_steal<py::object>(THPVariable_Wrap(t));
    const bool fake = py::isinstance(o, py::module_::import("torch._subclasses.fake_tensor").attr("FakeTensor"));
    TORCH_CHECK_TYPE(fake, "erfnet_pytorch_amd's operators take plain tensors, got ", std::string(py::str(py::type::of(o))));
    return true;
}

static void require_gpu(const Tensor& t, const char* who) {
    TORCH_CHECK(t.is_cuda(), who, ": erfnet_pytorch_amd runs on MI355X (gfx950) device tensors only; got a CPU tensor and there is no CPU path in this package");
}

static void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

static void check_status(int rc, const char* name) {
    TORCH_CHECK(rc == 0, name, " failed: ", rc == -1 ? "invalid argument" : rc == -2 ? "unsupported shape or dtype" : "kernel launch failed");
}

static const OptTensor& on_device(const OptTensor& t, const Tensor& x, const char* who, const char* name) {
    if (t) TORCH_CHECK_VALUE(t->device() == x.device(), who, ": ", name, " is on ", t->device(), ", the input on ", x.device());
    return t;
}

// Views that torch negates when they are read (the imaginary part of a conjugate) hold the negative of their values: resolve_neg()
// copies those, and gives every other tensor as it is.
static void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// backward with create_graph=True would record nothing of what these passes do
static void once_only(const char* who) {
    TORCH_CHECK(!c10::GradMode::is_enabled(), who, " is differentiable once: backward with create_graph=True is not supported");
}

// ... and forward-mode differentiation would find no tangent on the outputs, which counts as a derivative of 0
static void reverse_only(const Tensor& t, const char* who) {
    TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(), who, " has no forward-mode derivative");
}

// ------------------------------------------------------------------------------------------------ group norm + activation
static int64_t activation_code(const std::string& a) {
    const int64_t code = a == "none" ? ERF_ACT_NONE : a == "relu" ? ERF_ACT_RELU : a == "silu" ? ERF_ACT_SILU : -1;
    TORCH_CHECK_VALUE(code >= 0, "group_norm_act: activation is one of none, relu, silu, got '", a, "'");
    return code;
}

// Logical [N, C, ...] as a contiguous [N, ..., C]; zero-copy where the memory is channels-last
static Tensor channels_last(const Tensor& given) {
    const Tensor x = given.resolve_neg();
    Tensor last = x.dim() > 2 ? x.movedim(1, -1) : x;
    if (last.is_contiguous()) return last;
    auto tiles = [](int64_t n) { return (n + 31) / 32; };
    if (x.dim() == 4 && x.is_contiguous() && x.numel() && x.is_cuda() && !shape_only(x) &&
        x.size(0) * tiles(x.size(1)) * tiles(x.size(2) * x.size(3)) < (1 << 24)) {              // what one launch takes
        const int code = dtype_code(x, "group_norm_act");
        Tensor out = at::empty({x.size(0), x.size(2), x.size(3), x.size(1)}, x.options());
        c10::DeviceGuard guard(x.device());
        check_status(erf_nchw_to_nhwc(x.data_ptr(), code, out.data_ptr(), code, (int)x.size(0), (int)x.size(1), (int)x.size(2), (int)x.size(3), stream_of(x)),
                     "erf_nchw_to_nhwc");
        return out;
    }
    return last.contiguous();
}
static Tensor channels_first(const Tensor& y) { return y.dim() > 2 ? y.movedim(-1, 1) : y; }
// [N, C, ...] in channels-last memory.  No view: a view made inside an autograd node may not be written in place.
static Tensor empty_channels_last(at::IntArrayRef sizes, const at::TensorOptions& options) {
    std::vector<int64_t> strides(sizes.size());
    int64_t step = sizes[1];
    for (size_t d = sizes.size() - 1; d >= 2; --d) {
        strides[d] = step;
        step *= std::max<int64_t>(sizes[d], 1);
    }
    strides[0] = std::max<int64_t>(step, 1);
    strides[1] = 1;
    return at::empty_strided(sizes, strides, options);
}

static Tensor fp32(const OptTensor& t) { return t ? t->resolve_neg().to(at::kFloat).contiguous() : Tensor(); }

struct GnShape { int code, n, c; int64_t hw; };
static GnShape gn_check(const Tensor& x, const OptTensor& weight, const OptTensor& bias, int64_t groups) {
    const char* who = "group_norm_act";
    GnShape s;
    s.code = dtype_code(x, who);
    TORCH_CHECK_VALUE(x.dim() >= 2 && x.is_contiguous(), who, ": a contiguous channels-last tensor [N, ..., C], got shape ", x.sizes(), " strides ", x.strides());
    const int64_t c = x.size(-1), n = x.size(0);
    TORCH_CHECK_VALUE(groups >= 1 && c >= 1 && c % groups == 0, who, ": ", c, " channels do not split into ", groups, " groups");
    TORCH_CHECK_VALUE(n <= INT_MAX && c <= INT_MAX, who, ": shape ", x.sizes(), " is too large");
    for (const auto& [t, name] : {std::make_pair(&weight, "weight"), std::make_pair(&bias, "bias")})
        if (*t) {
            TORCH_CHECK_VALUE((*t)->dim() == 1 && (*t)->size(0) == c, who, ": ", name, " has shape [", c, "], got ", (*t)->sizes());
            on_device(*t, x, who, name);
        }
    s.n = (int)n;
    s.c = (int)c;
    s.hw = n ? x.numel() / (n * c) : 0;
    TORCH_CHECK_VALUE(!x.numel() || erf_group_norm_workspace_bytes(s.code, s.n, s.hw, s.c, (int)groups) > 0, who, ": shape ", x.sizes(), " is too large");
    return s;
}

static Tensor gn_workspace(const Tensor& x, const GnShape& s, int64_t groups) {
    return at::empty({(int64_t)erf_group_norm_workspace_bytes(s.code, s.n, s.hw, s.c, (int)groups)}, x.options().dtype(at::kByte));
}

// (y, stats [2, N, groups]) of a contiguous channels-last x; y [N, ..., C], or as `first` [N, C, ...] in the same memory
static std::tuple<Tensor, Tensor> group_norm_fwd(const Tensor& x, const OptTensor& weight, const OptTensor& bias, int64_t groups, double eps, int64_t act,
                                                 bool first) {
    const GnShape s = gn_check(x, weight, bias, groups);
    TORCH_CHECK_VALUE(eps >= 0 && std::isfinite(eps), "group_norm_act: invalid eps ", eps);
    Tensor y = first && x.dim() > 2 ? empty_channels_last(x.movedim(-1, 1).sizes(), x.options()) : at::empty(x.sizes(), x.options());
    Tensor stats = at::empty({2, s.n, groups}, x.options().dtype(at::kFloat));
    if (x.numel() && !shape_only(x)) {
        require_gpu(x, "group_norm_act");
        const Tensor w = fp32(weight), b = fp32(bias);
        c10::DeviceGuard guard(x.device());
        const Tensor ws = gn_workspace(x, s, groups);
        float* mean = stats.data_ptr<float>();
        check_status(erf_group_norm_fwd(x.data_ptr(), y.data_ptr(), s.code, s.n, s.hw, s.c, (int)groups, (const float*)ptr(w), (const float*)ptr(b), (float)eps,
                                        (int)act, mean, mean + (int64_t)s.n * groups, ws.data_ptr(), stream_of(x)),
                     "erf_group_norm_fwd");
    }
    return {y, stats};
}

// (dx, dweight, dbias) from a contiguous channels-last dy; the parameter gradients are fp32 whatever the types
static std::tuple<Tensor, Tensor, Tensor> group_norm_bwd(const Tensor& dy, const Tensor& x, const OptTensor& weight, const OptTensor& bias, const Tensor& stats,
                                                         int64_t groups, int64_t act) {
    const GnShape s = gn_check(x, weight, bias, groups);
    TORCH_CHECK_VALUE(dy.sizes() == x.sizes() && dy.scalar_type() == x.scalar_type() && dy.is_contiguous(), "group_norm_act: dy is a contiguous ", x.dtype(),
                      " tensor of shape ", x.sizes(), ", got ", dy.dtype(), " ", dy.sizes(), " strides ", dy.strides());
    TORCH_CHECK_VALUE(stats.sizes() == at::IntArrayRef({2, s.n, groups}) && stats.scalar_type() == at::kFloat && stats.is_contiguous(),
                      "group_norm_act: stats are a contiguous fp32 tensor [2, ", s.n, ", ", groups, "], got ", stats.dtype(), " ", stats.sizes());
    on_device(dy, x, "group_norm_act", "dy");
    on_device(stats, x, "group_norm_act", "stats");
    Tensor dx = at::empty(x.sizes(), x.options()), dweight = at::empty({s.c}, stats.options()), dbias = at::empty({s.c}, stats.options());
    if (!x.numel()) {
        dweight.zero_();
        dbias.zero_();
    } else if (!shape_only(x)) {
        require_gpu(x, "group_norm_act");
        const Tensor w = fp32(weight), b = fp32(bias);
        c10::DeviceGuard guard(x.device());
        const Tensor ws = gn_workspace(x, s, groups);
        const float* mean = stats.data_ptr<float>();
        check_status(erf_group_norm_bwd(x.data_ptr(), dy.data_ptr(), dx.data_ptr(), s.code, s.n, s.hw, s.c, (int)groups, (const float*)ptr(w), (const float*)ptr(b),
                                        (int)act, mean, mean + (int64_t)s.n * groups, dweight.data_ptr<float>(), dbias.data_ptr<float>(), ws.data_ptr(),
                                        stream_of(x)),
                     "erf_group_norm_bwd");
    }
    return {dx, dweight, dbias};
}

struct GroupNormActFn : public torch::autograd::Function<GroupNormActFn> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& weight, const OptTensor& bias, int64_t groups, double eps, int64_t act) {
        const Tensor last = channels_last(x);
        auto [y, stats] = group_norm_fwd(last, weight, bias, groups, eps, act, true);
        ctx->save_for_backward({last, weight.value_or(Tensor()), bias.value_or(Tensor()), stats});
        ctx->saved_data["groups"] = groups;
        ctx->saved_data["act"] = act;
        return y;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        once_only("group_norm_act");
        const variable_list saved = ctx->get_saved_variables();
        auto given = [](const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
        auto [dx, dw, db] = group_norm_bwd(channels_last(grads[0]), saved[0], given(saved[1]), given(saved[2]), saved[3], ctx->saved_data["groups"].toInt(),
                                           ctx->saved_data["act"].toInt());
        return {channels_first(dx), saved[1].defined() ? dw.to(saved[1].scalar_type()) : Tensor(), saved[2].defined() ? db.to(saved[2].scalar_type()) : Tensor(),
                Tensor(), Tensor(), Tensor()};
    }
};

static Tensor group_norm_act(const Tensor& x, int64_t groups, const OptTensor& weight, const OptTensor& bias, double eps, const std::string& activation) {
    require_gpu(x, "group_norm_act");
    TORCH_CHECK_VALUE(x.dim() >= 2, "group_norm_act: x has shape [N, C, ...], got ", x.sizes());
    const int64_t act = activation_code(activation);
    for (const Tensor& t : {x, weight.value_or(Tensor()), bias.value_or(Tensor())}) reverse_only(t, "group_norm_act");
    if (c10::GradMode::is_enabled() && (x.requires_grad() || (weight && weight->requires_grad()) || (bias && bias->requires_grad())))
        return GroupNormActFn::apply(x, weight, bias, groups, eps, act);
    return std::get<0>(group_norm_fwd(channels_last(x), weight, bias, groups, eps, act, true));
}

// ------------------------------------------------------------------------------------------------ label log probabilities
// Logits [N, C, ...] as the C ABI takes them: rows where the classes of a position lie side by side ([N, C], or a channels-last map),
// else planes of L positions.  Other layouts are copied into planes.
struct Layout {
    Tensor z;
    int64_t n, length, sn, sc;
    int c;
    bool rows;
    std::vector<int64_t> shape;        // [N, ...]
};

static Layout class_layout(const Tensor& given) {
    const Tensor logits = given.resolve_neg();
    TORCH_CHECK_VALUE(logits.dim() >= 2 && logits.size(1) >= 1, "class_log_probs: logits have shape [N, C, ...] with at least one class, got ", logits.sizes());
    Layout q;
    q.z = logits;
    const int64_t n = logits.size(0), c = logits.size(1);
    TORCH_CHECK_VALUE(c <= (1 << 28), "class_log_probs: at most 2^28 classes, got ", c);
    q.c = (int)c;
    q.shape.push_back(n);
    int64_t length = 1;
    for (int64_t d = 2; d < logits.dim(); ++d) {
        q.shape.push_back(logits.size(d));
        length *= logits.size(d);
    }
    if (length == 1) {
        if (c > 1 && logits.stride(1) != 1) q.z = logits.contiguous();
        q.n = n; q.length = 1; q.sn = n > 1 ? q.z.stride(0) : c; q.sc = 1; q.rows = true;
        return q;
    }
    if (c > 1 && logits.stride(1) == 1 && logits.movedim(1, -1).is_contiguous()) {
        q.n = n * length; q.length = 1; q.sn = c; q.sc = 1; q.rows = true;
        return q;
    }
    int64_t dense = 1;                                       // the map's own axes, innermost last, without gaps
    bool ok = true;
    for (int64_t d = logits.dim() - 1; d >= 2; --d) {
        ok = ok && (logits.size(d) == 1 || logits.stride(d) == dense);
        dense *= logits.size(d);
    }
    if (!ok || (c > 1 && logits.stride(1) < std::max<int64_t>(length, 2))) q.z = logits.contiguous();
    q.n = n; q.length = length; q.rows = false;
    q.sn = n > 1 ? q.z.stride(0) : c * length;
    q.sc = std::max<int64_t>({c > 1 ? q.z.stride(1) : 0, length, 2});
    return q;
}

static Tensor check_target(const OptTensor& target, const Layout& q) {
    if (!target) return Tensor();
    TORCH_CHECK_TYPE(target->scalar_type() == at::kLong, "class_log_probs: targets are int64 class indices, got ", target->dtype());
    TORCH_CHECK_VALUE(target->sizes() == at::IntArrayRef(q.shape), "class_log_probs: expected targets of shape ", at::IntArrayRef(q.shape), ", got ", target->sizes());
    on_device(target, q.z, "class_log_probs", "target");
    return target->resolve_neg().contiguous();
}

// Memory of [N, k, ...] that follows the logits: k last for rows
static Tensor like_layout(const Layout& q, int64_t k, at::ScalarType type) {
    std::vector<int64_t> s = q.shape;
    s.insert(s.begin() + 1, k);
    return q.rows && s.size() > 2 ? empty_channels_last(s, q.z.options().dtype(type)) : at::empty(s, q.z.options().dtype(type));
}
// ... of a tensor [N, k, ...] given from outside
static Tensor to_layout(const Tensor& given, const Layout& q) {
    const Tensor t = given.resolve_neg();
    return q.rows && t.dim() > 2 ? t.movedim(1, -1).contiguous() : t.contiguous();
}

// (log_prob, entropy, stats [2, N, ...], top_log_probs, top_indices); stats undefined where no backward pass follows
static std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> class_log_probs_fwd(const Tensor& logits, const OptTensor& target_, int64_t top_k, int64_t ignore_index,
                                                                              bool with_stats) {
    const int code = dtype_code(logits, "class_log_probs");
    const Layout q = class_layout(logits);
    TORCH_CHECK_VALUE(top_k >= 0 && top_k <= std::min(ERF_TOP_MAX, q.c), "class_log_probs: top_k lies between 0 and min(", ERF_TOP_MAX, ", classes), got ", top_k,
                      " for ", q.c, " classes");
    const Tensor target = check_target(target_, q);
    const auto f = q.z.options().dtype(at::kFloat);
    Tensor log_prob = target.defined() ? at::empty(q.shape, f) : at::empty({0}, f), entropy = at::empty(q.shape, f), stats;
    if (with_stats) {
        std::vector<int64_t> s = q.shape;
        s.insert(s.begin(), 2);
        stats = at::empty(s, f);
    }
    Tensor top = like_layout(q, top_k, at::kFloat), index = like_layout(q, top_k, at::kLong);
    if (entropy.numel() && !shape_only(logits)) {
        require_gpu(logits, "class_log_probs");
        c10::DeviceGuard guard(logits.device());
        const size_t bytes = erf_class_log_probs_workspace_bytes(code, q.n, q.c, q.length, q.sc, (int)top_k);
        const Tensor ws = bytes ? at::empty({(int64_t)bytes}, q.z.options().dtype(at::kByte)) : Tensor();
        check_status(erf_class_log_probs_fwd(q.z.data_ptr(), code, q.n, q.c, q.length, q.sn, q.sc, (const long long*)ptr(target), ignore_index,
                                             target.defined() ? log_prob.data_ptr<float>() : nullptr, entropy.data_ptr<float>(), (float*)ptr(stats), (int)top_k,
                                             top_k ? top.data_ptr<float>() : nullptr, top_k ? (long long*)index.data_ptr() : nullptr, ptr(ws), stream_of(logits)),
                     "erf_class_log_probs_fwd");
    }
    return {log_prob, entropy, stats, top, index};
}

// d logits, laid out as the logits
static Tensor class_log_probs_bwd(const Tensor& logits, const OptTensor& target_, const Tensor& stats, const Tensor& entropy, const Tensor& top_indices,
                                  const OptTensor& g_log_prob, const OptTensor& g_entropy, const OptTensor& g_top, int64_t ignore_index) {
    const char* who = "class_log_probs";
    const int code = dtype_code(logits, who);
    const Layout q = class_layout(logits);
    const Tensor target = check_target(target_, q);
    std::vector<int64_t> two = q.shape, top_shape = q.shape;
    two.insert(two.begin(), 2);
    const int64_t k = g_top ? g_top->size(1) : 0;
    top_shape.insert(top_shape.begin() + 1, k);
    TORCH_CHECK_VALUE(stats.sizes() == at::IntArrayRef(two) && entropy.sizes() == at::IntArrayRef(q.shape) && stats.scalar_type() == at::kFloat &&
                          entropy.scalar_type() == at::kFloat && stats.is_contiguous() && entropy.is_contiguous(),
                      who, ": stats and entropy are contiguous fp32 tensors of shapes ", at::IntArrayRef(two), " and ", at::IntArrayRef(q.shape));
    TORCH_CHECK_VALUE(!g_log_prob || (target.defined() && g_log_prob->sizes() == at::IntArrayRef(q.shape)), who, ": g_log_prob has the target's shape");
    TORCH_CHECK_VALUE(!g_entropy || g_entropy->sizes() == at::IntArrayRef(q.shape), who, ": g_entropy has shape ", at::IntArrayRef(q.shape));
    TORCH_CHECK_VALUE(!g_top || (g_top->sizes() == at::IntArrayRef(top_shape) && top_indices.sizes() == g_top->sizes() && k <= ERF_TOP_MAX &&
                                 top_indices.scalar_type() == at::kLong),
                      who, ": g_top and the int64 top_indices have shape ", at::IntArrayRef(top_shape));
    for (const Tensor* t : {&stats, &entropy, &top_indices}) on_device(*t, logits, who, "a saved tensor");
    for (const OptTensor* t : {&g_log_prob, &g_entropy, &g_top}) on_device(*t, logits, who, "a gradient");
    Tensor dz = like_layout(q, q.c, logits.scalar_type());
    if (!dz.numel() || shape_only(logits)) return dz;
    require_gpu(logits, who);
    c10::DeviceGuard guard(logits.device());
    const Tensor gl = fp32(g_log_prob), gh = fp32(g_entropy), gk = k ? to_layout(g_top->to(at::kFloat), q) : Tensor(),
                 index = k ? to_layout(top_indices, q) : Tensor();
    check_status(erf_class_log_probs_bwd(q.z.data_ptr(), code, q.n, q.c, q.length, q.sn, q.sc, (const long long*)ptr(target), ignore_index, stats.data_ptr<float>(),
                                         entropy.data_ptr<float>(), (const float*)ptr(gl), (const float*)ptr(gh), (int)k, (const long long*)ptr(index),
                                         (const float*)ptr(gk), dz.data_ptr(), q.rows ? q.c : q.c * q.length, q.rows ? 1 : std::max<int64_t>(q.length, 2),
                                         stream_of(logits)),
                 "erf_class_log_probs_bwd");
    return dz;
}

struct ClassLogProbsFn : public torch::autograd::Function<ClassLogProbsFn> {
    static variable_list forward(AutogradContext* ctx, const Tensor& logits, const OptTensor& target, int64_t top_k, int64_t ignore_index) {
        auto [log_prob, entropy, stats, top, index] = class_log_probs_fwd(logits, target, top_k, ignore_index, true);
        ctx->save_for_backward({logits, target.value_or(Tensor()), stats, entropy, index});
        ctx->saved_data["ignore"] = ignore_index;
        ctx->set_materialize_grads(false);
        ctx->mark_non_differentiable({index});
        return {log_prob, entropy, top, index};
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& g) {
        once_only("class_log_probs");
        const variable_list s = ctx->get_saved_variables();
        auto given = [](const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
        const OptTensor gl = s[1].defined() ? given(g[0]) : OptTensor(), gh = given(g[1]), gk = s[4].size(1) ? given(g[2]) : OptTensor();
        if (!gl && !gh && !gk) return {Tensor(), Tensor(), Tensor(), Tensor()};
        return {class_log_probs_bwd(s[0], given(s[1]), s[2], s[3], s[4], gl, gh, gk, ctx->saved_data["ignore"].toInt()), Tensor(), Tensor(), Tensor()};
    }
};

static std::tuple<Tensor, Tensor, Tensor, Tensor> class_log_probs(const Tensor& logits, const OptTensor& target, int64_t top_k, int64_t ignore_index) {
    require_gpu(logits, "class_log_probs");
    reverse_only(logits, "class_log_probs");
    if (c10::GradMode::is_enabled() && logits.requires_grad()) {
        const variable_list r = ClassLogProbsFn::apply(logits, target, top_k, ignore_index);
        return {r[0], r[1], r[2], r[3]};
    }
    auto [log_prob, entropy, stats, top, index] = class_log_probs_fwd(logits, target, top_k, ignore_index, false);
    return {log_prob, entropy, top, index};
}

// ------------------------------------------------------------------------------------------------ AdamW's parameters
// What the device tables of an optimizer describe: which parameters they hold, which of these have a gradient, and where both lie.
// look() compares that with the present; it keeps no gradient alive.
struct ParamWatch {
    struct Entry {
        const void *param, *grad;
        bool on, copied;                        // in a table; its gradient is copied
        size_t place;                           // among those in tables
        at::ScalarType type;
        at::DimVector shape;                    // sizes, then strides
    };
    struct Move { size_t at; const void* grad; bool copied; };
    std::vector<Entry> entries;
    std::vector<Move> moves;                    // of the present look
    std::vector<Tensor> params;                 // those in tables, in the order of the groups
    std::vector<char> given;                    // which of them have a gradient
    bool changed = false;                       // whether the last look found that one came or went

    static const Tensor& tensor(PyObject* o) {
        TORCH_CHECK_TYPE(THPVariable_Check(o), "AdamW: parameters are tensors");
        return THPVariable_Unpack(o);
    }

    static void check_grad(const Tensor& p, const Tensor& g) {
        TORCH_CHECK_VALUE(g.layout() == at::kStrided && g.scalar_type() == p.scalar_type() && g.device() == p.device() && g.sizes() == p.sizes(),
                          "AdamW: a gradient of a parameter ", p.dtype(), " ", p.sizes(), " has to be a dense tensor of the same type, shape and device, got ",
                          g.dtype(), " ", g.sizes());
    }

    static bool same_shape(const Tensor& p, const Entry& e) {
        const at::IntArrayRef seen(e.shape);
        const size_t d = p.dim();
        return seen.size() == 2 * d && p.sizes() == seen.slice(0, d) && p.strides() == seen.slice(d);
    }

    // 0: all as before; 1: the same parameters, gradients elsewhere, come or gone (noted); 2: other parameters, parameters elsewhere, or
    // a gradient of one that is in no table.
    // A gradient whose strides are not its parameter's (or that holds its negative) counts as elsewhere every time: it is copied.
    // Nothing is noted before every gradient has been checked: after a refusal the next look finds the same changes.
    int look(const std::vector<py::list>& groups) {
        size_t i = 0;
        moves.clear();
        for (const py::list& group : groups)
            for (py::handle h : group) {
                const Tensor& p = tensor(h.ptr());
                const Tensor& g = p.grad();
                if (i >= entries.size()) return 2;
                const Entry& e = entries[i++];
                if (!e.on) {
                    if (g.defined() && p.numel()) return 2;
                    continue;
                }
                if (p.data_ptr() != e.param || p.scalar_type() != e.type || !same_shape(p, e)) return 2;
                if (!g.defined()) {
                    if (given[e.place]) moves.push_back({i - 1, nullptr, false});
                    continue;
                }
                const bool strided = g.layout() == at::kStrided;
                if (strided && g.data_ptr() == e.grad && g.sizes() == p.sizes() && g.strides() == p.strides() && g.scalar_type() == e.type && !e.copied && !g.is_neg()) continue;
                check_grad(p, g);
                moves.push_back({i - 1, g.data_ptr(), g.is_neg() || (g.strides() != p.strides() && !(g.is_contiguous() && p.is_contiguous()))});
            }
        if (i != entries.size()) return 2;
        changed = false;
        for (const Move& m : moves) {
            Entry& e = entries[m.at];
            e.grad = m.grad;
            e.copied = m.copied;
            changed = changed || given[e.place] != (m.grad != nullptr);
            given[e.place] = m.grad != nullptr;
        }
        return moves.empty() ? 0 : 1;
    }

    // Takes the parameters as they are: those with a gradient, and those whose places among all parameters `more` names, are in the
    // tables.  look() then reports the gradients as moved once.
    void bind(const std::vector<py::list>& groups, const std::vector<int64_t>& more) {
        entries.clear();
        params.clear();
        given.clear();
        auto next = more.begin();
        for (const py::list& group : groups)
            for (py::handle h : group) {
                const Tensor& p = tensor(h.ptr());
                const bool named = next != more.end() && *next == (int64_t)entries.size();
                if (named) ++next;
                const bool on = (p.grad().defined() || named) && p.numel();
                if (on && p.grad().defined()) check_grad(p, p.grad());
                entries.push_back({on ? p.data_ptr() : nullptr, nullptr, on, false, params.size(), p.scalar_type(), at::DimVector(p.sizes())});
                entries.back().shape.append(p.strides().begin(), p.strides().end());
                if (on) {
                    params.push_back(p);
                    given.push_back(p.grad().defined());
                }
            }
    }

    // The gradients' addresses, NULL for none, are written to the table records of one launch; which: places among the parameters in tables
    void set_grads(int64_t table, const std::vector<int>& which, const std::vector<int64_t>& copies, int64_t stream) const {
        std::vector<const void*> at, all;
        for (const Entry& e : entries)
            if (e.on) all.push_back(e.grad);
        for (size_t i = 0; i < which.size(); ++i) at.push_back(copies[i] ? (const void*)copies[i] : all.at(which[i]));
        check_status(erf_adamw_set_grads((erf_adamw_tensor*)table, at.data(), (int)at.size(), (void*)stream), "erf_adamw_set_grads");
    }

    std::vector<bool> present() const { return {given.begin(), given.end()}; }

    // Places of the gradients that need a copy in their parameter's order
    std::vector<int> copied() const {
        std::vector<int> r;
        int i = 0;
        for (const Entry& e : entries)
            if (e.on) {
                if (e.copied) r.push_back(i);
                ++i;
            }
        return r;
    }

    // The parameters with a gradient changed through their addresses
    void bump() {
        for (size_t i = 0; i < params.size(); ++i)
            if (given[i]) params[i].unsafeGetTensorImpl()->bump_version();
    }
};

// What a device table points at stays allocated as long as the table
struct TableHold { std::vector<c10::Storage> storages; };

// The table's records (CPU int64 [n, 8], grad fields 0) of these parameters with these states: (exp_avg, exp_avg_sq), or (exp_avg,
// exp_avg_sq_root, exp_avg_scale, exp_avg_sq_root_scale)
static std::tuple<Tensor, std::shared_ptr<TableHold>> adamw_table(const std::vector<Tensor>& params, const std::vector<std::vector<Tensor>>& states,
                                                                  const std::vector<int64_t>& bases) {
    const int64_t block = erf_adamw_scale_block();
    static const char* const names32[] = {"exp_avg", "exp_avg_sq"};
    static const char* const names8[] = {"exp_avg", "exp_avg_sq_root", "exp_avg_scale", "exp_avg_sq_root_scale"};
    auto hold = std::make_shared<TableHold>();
    Tensor rows = at::zeros({(int64_t)params.size(), 8}, at::kLong);
    int64_t* r = rows.data_ptr<int64_t>();
    for (size_t i = 0; i < params.size(); ++i, r += 8) {
        const Tensor& p = params[i];
        const std::vector<Tensor>& st = states.at(i);
        const bool eight = st.size() == 4;
        const at::ScalarType type = eight ? at::kFloat8_e4m3fn : at::kFloat;
        for (size_t k = 0; k < st.size(); ++k) {
            const Tensor& t = st[k];
            const char* name = eight ? names8[k] : names32[k];
            if (k < 2) {
                TORCH_CHECK_VALUE(t.defined() && t.scalar_type() == type && t.device() == p.device() && t.sizes() == p.sizes() &&
                                      (t.strides() == p.strides() || (t.is_contiguous() && p.is_contiguous())),
                                  "AdamW: state '", name, "' of a parameter of shape ", p.sizes(), ": expected a ", type, " tensor laid out as the parameter");
            } else {
                TORCH_CHECK_VALUE(t.defined() && t.scalar_type() == at::kFloat && t.device() == p.device() && t.is_contiguous() &&
                                      t.numel() == (p.numel() + block - 1) / block,
                                  "AdamW: state '", name, "' of a parameter of shape ", p.sizes(), ": expected one fp32 value per ", block, " elements");
            }
            hold->storages.push_back(t.storage());
        }
        hold->storages.push_back(p.storage());
        const int64_t row[8] = {(int64_t)p.data_ptr(), 0, (int64_t)st[0].data_ptr(), (int64_t)st[1].data_ptr(), eight ? (int64_t)st[2].data_ptr() : 0,
                                eight ? (int64_t)st[3].data_ptr() : 0, p.numel(), bases.at(i)};
        std::copy(row, row + 8, r);
    }
    return {rows, hold};
}

// Two parameters that share memory would be updated by two workgroups at once
static void adamw_no_overlap(const std::vector<Tensor>& params) {
    std::vector<std::tuple<int, const char*, const char*>> spans;
    for (const Tensor& p : params) spans.emplace_back(p.device().index(), (const char*)p.data_ptr(), (const char*)p.data_ptr() + p.numel() * p.element_size());
    std::sort(spans.begin(), spans.end());
    for (size_t i = 1; i < spans.size(); ++i)
        TORCH_CHECK_VALUE(std::get<0>(spans[i]) != std::get<0>(spans[i - 1]) || std::get<1>(spans[i]) >= std::get<2>(spans[i - 1]),
                          "AdamW: two parameters share memory; give the optimizer one of them");
}

static std::tuple<Tensor, Tensor> group_norm_act_fwd(const Tensor& x, const OptTensor& weight, const OptTensor& bias, int64_t groups, double eps,
                                                     const std::string& activation) {
    return group_norm_fwd(x.resolve_neg(), weight, bias, groups, eps, activation_code(activation), false);
}
static std::tuple<Tensor, Tensor, Tensor> group_norm_act_bwd(const Tensor& dy, const Tensor& x, const OptTensor& weight, const OptTensor& bias, const Tensor& stats,
                                                             int64_t groups, const std::string& activation) {
    return group_norm_bwd(dy.resolve_neg(), x.resolve_neg(), weight, bias, stats, groups, activation_code(activation));
}
static std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> class_log_probs_with_stats(const Tensor& logits, const OptTensor& target, int64_t top_k, int64_t ignore_index) {
    return class_log_probs_fwd(logits, target, top_k, ignore_index, true);
}
static std::tuple<Tensor, int64_t, int64_t, int64_t, int64_t, int64_t, bool> layout_of(const Tensor& logits) {
    const Layout q = class_layout(logits);
    return {q.z, q.n, q.c, q.length, q.sn, q.sc, q.rows};
}

// wrap_pybind_function: c10's errors become the Python exceptions they stand for (ValueError, TypeError, ...)
PYBIND11_MODULE(_host, m) {
    using torch::wrap_pybind_function;
    m.doc() = "Host side of the training operators in C++; used by train_ops.py, norm.py, loss.py and optim.py";
    m.def("group_norm_act", wrap_pybind_function(group_norm_act));
    m.def("group_norm_act_fwd", wrap_pybind_function(group_norm_act_fwd));
    m.def("group_norm_act_bwd", wrap_pybind_function(group_norm_act_bwd));
    m.def("class_log_probs", wrap_pybind_function(class_log_probs));
    m.def("class_log_probs_fwd", wrap_pybind_function(class_log_probs_with_stats));
    m.def("class_log_probs_bwd", wrap_pybind_function(class_log_probs_bwd));
    m.def("class_layout", wrap_pybind_function(layout_of));
    m.def("adamw_table", wrap_pybind_function(adamw_table));
    m.def("adamw_no_overlap", wrap_pybind_function(adamw_no_overlap));
    py::class_<TableHold, std::shared_ptr<TableHold>>(m, "TableHold");
    py::class_<ParamWatch>(m, "ParamWatch")
        .def(py::init<>())
        .def("look", wrap_pybind_function(&ParamWatch::look))
        .def("bind", wrap_pybind_function(&ParamWatch::bind), py::arg("groups"), py::arg("more") = std::vector<int64_t>())
        .def_readonly("changed", &ParamWatch::changed)
        .def("present", wrap_pybind_function(&ParamWatch::present))
        .def("set_grads", wrap_pybind_function(&ParamWatch::set_grads))
        .def("copied", wrap_pybind_function(&ParamWatch::copied))
        .def("bump", wrap_pybind_function(&ParamWatch::bump));
}
