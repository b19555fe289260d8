// The policy-training operators as torch sees them: argument checks, allocation, autograd and the calls of the C entries (include/plmpm_policy.h),
// whose addresses plasticinelab_amd/policy.py hands over.  No device code.  In C++ because many of these calls are shorter than what a Python
// function around them costs, and because the autograd engine's thread would have to wait for the interpreter's lock: one step of
// (1, 128) 5.6 us, with the checks in Python 10.7; forward and backward of (16, 50, 256) 93 us, 159 in Python (torch's own product and its
// backward, nothing else: 52); an update of 20 tensors 14.5 us, 48 in Python.
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <algorithm>
#include <unordered_map>

#include "../../include/plmpm.h"
#include "../../include/plmpm_policy.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

// a message of the library (plmpm_last_error) or of a missing device: plasticinelab_amd._lib.EngineError in Python
struct EngineError : std::runtime_error {
    using std::runtime_error::runtime_error;
};

struct Library {
    decltype(&plmpm_last_error) last_error = nullptr;
    decltype(&plmpm_scan_workspace) scan_workspace = nullptr;
    decltype(&plmpm_scan_forward) scan_forward = nullptr;
    decltype(&plmpm_scan_backward) scan_backward = nullptr;
    decltype(&plmpm_norm_workspace) norm_workspace = nullptr;
    decltype(&plmpm_norm_forward) norm_forward = nullptr;
    decltype(&plmpm_norm_backward) norm_backward = nullptr;
    decltype(&plmpm_adamw_workspace) adamw_workspace = nullptr;
    decltype(&plmpm_adamw_step) adamw_step = nullptr;
    decltype(&plmpm_adamw_values) adamw_values = nullptr;
    bool host = false;                  // the entries take host memory (the tests' interpreter of the device source)
} lib;

constexpr int64_t kMaxWidth = 8192, kCheckpoint = 64, kBlock = 256;
constexpr int64_t kFarRows = 1 << 23;           // elements from row to row that the norm reads in place at any width (it addresses 64 rows by 32 bits)

// an argument is not what the operator takes: ValueError in Python
#define REFUSE_IF(cond, ...) do { if (cond) throw std::invalid_argument(c10::str(__VA_ARGS__)); } while (0)

void check(int rc) { if (rc != 0) throw EngineError(lib.last_error()); }

std::string name_of(at::ScalarType t) {
    static const std::unordered_map<at::ScalarType, const char*> names = {{at::kFloat, "float32"}, {at::kBFloat16, "bfloat16"}, {at::kHalf, "float16"}, {at::kDouble, "float64"},
        {at::kChar, "int8"}, {at::kByte, "uint8"}, {at::kInt, "int32"}, {at::kLong, "int64"}, {at::kBool, "bool"}};
    const auto it = names.find(t);
    return it == names.end() ? c10::toString(t) : it->second;
}
int code_of(at::ScalarType t) { return t == at::kFloat ? PLMPM_NN_F32 : t == at::kBFloat16 ? PLMPM_NN_BF16 : t == at::kHalf ? PLMPM_NN_F16 : -1; }

// What records the operations of a program sees a call's allocations and not its kernels: the recorded program would return memory that nothing wrote to.
// (One look at the thread's dispatch keys: a recorder has one of these in there.)
void not_recorded() {
    const c10::DispatchKeySet keys = c10::impl::tls_local_dispatch_key_set().included_;
    if (!keys.has_any(c10::DispatchKeySet({c10::DispatchKey::Tracer, c10::DispatchKey::Python, c10::DispatchKey::PreDispatch}))) return;
    if (keys.has(c10::DispatchKey::Tracer)) throw EngineError("policy operators cannot be traced (torch.jit.trace): their kernels would be missing from the graph");
    using Modes = c10::impl::TorchDispatchModeTLS;
    using Key = c10::impl::TorchDispatchModeKey;
    bool found = keys.has(c10::DispatchKey::PreDispatch);
    for (const Key key : {Key::PROXY, Key::FAKE, Key::FUNCTIONAL}) found = found || Modes::get_mode(key).has_value();
    if (found) throw EngineError("policy operators cannot be traced (make_fx, fake or functional tensors): their kernels would be missing from the graph");
}
// the device that a call's kernels go to, made current, and its current stream
struct Site {
    c10::OptionalDeviceGuard guard;
    void* stream = nullptr;
    explicit Site(const Tensor& t) {
        if (!lib.last_error) throw EngineError("the library is not loaded");
        not_recorded();
        if (lib.host && t.is_cpu()) return;
        if (!t.is_cuda())
            throw EngineError("policy operators run on a ROCm device, got a tensor on " + t.device().str() + ": there is no CPU path");
        guard.reset_device(t.device());
        stream = c10::hip::getCurrentHIPStream(t.device().index()).stream();
    }
};

// Kernels read memory.  What torch has only noted beside it is applied first: a sign (x.conj().imag and gradients of complex products are such views), zeros
// that were never stored.  What is written in place has to be without.
void settle(Tensor& t) {
    if (t.is_neg()) t = t.resolve_neg();
    if (t._is_zerotensor()) t = at::zeros(t.sizes(), t.options()).add(t);
}
void settle(Maybe& t) { if (t) settle(*t); }
void settled(const Tensor& t, const char* name) {
    REFUSE_IF(t.is_neg() || t._is_zerotensor(), name, " is written in place: it cannot be a negative view or a tensor of zeros without memory");
}
// where a tensor's values lie; a null pointer would be read as a tensor that was not given
void* memory(const Tensor& t) {
    void* p = t.data_ptr();
    if (!p && t.numel()) throw EngineError("a tensor came in that holds no memory (a wrapper of one of torch's transforms)");
    return p;
}
const void* ptr(const Maybe& t) { return t ? memory(*t) : nullptr; }
template <class T = void> T* out(const Tensor& t) { return t.defined() ? (T*)memory(t) : nullptr; }
Tensor workspace(const Tensor& like, size_t bytes) { return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor(); }
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); }

void same_device(const Tensor& first, const Tensor& t, const char* name) {
    REFUSE_IF(t.device() != first.device(), name, " is on ", t.device(), ", not on ", first.device());
}
// unit stride over the last dimension (a copy if need be)
Tensor rows_of(const Tensor& t) { return t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous(); }
bool tracked(std::initializer_list<const Maybe*> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Maybe* t : ts) if (*t && (*t)->requires_grad()) return true;
    return false;
}
// A forward-mode tangent that comes with a tensor would be lost: nothing here makes one for what a kernel writes.  (There are none outside a dual level, which
// is one question a call; asking each tensor cost an update of 20 views 0.7 us.)
bool tangents_about() { return torch::autograd::ForwardADLevel::try_get_by_idx(0) && c10::AutogradState::get_tls_state().get_fw_grad_mode(); }
void no_tangents(std::initializer_list<const Maybe*> ts, const char* name) {
    if (!tangents_about()) return;
    for (const Maybe* t : ts) REFUSE_IF(*t && (*t)->_fw_grad(0).defined(), name, " has no forward-mode derivative: a tensor with a tangent came in");
}
// a tensor was changed in place: a graph that saved it has to notice (tensors of inference mode are in none)
void written(const Tensor& t) { if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version(); }
// gradients of a backward pass that was asked for its own graph: they have none, and say so when it is used
variable_list once(variable_list grads, const char* name) {
    if (!at::GradMode::is_enabled()) return grads;
    auto error = std::make_shared<torch::autograd::DelayedError>(std::string(name) + " has no second derivative", (int64_t)grads.size());
    variable_list marked;
    std::vector<size_t> at;
    for (size_t k = 0; k < grads.size(); ++k)
        if (grads[k].defined()) {
            marked.push_back(grads[k].detach().requires_grad_());
            at.push_back(k);
        }
    marked = (*error)(std::move(marked));
    for (size_t k = 0; k < at.size(); ++k) grads[at[k]] = marked[k];
    return grads;
}

// ---------------------------------------------------------------------------------------------- gated linear recurrence
plmpm_scan scan_of(const Tensor& x, const Tensor& r, const Tensor& i, const Tensor& decay, const Maybe& reset, double c) {
    plmpm_scan s{};
    s.dtype = code_of(x.scalar_type());
    s.batch = x.size(0);
    s.steps = x.size(1);
    s.width = x.size(2);
    const Tensor* in[3] = {&x, &r, &i};
    for (int k = 0; k < 3; ++k) { s.stride_b[k] = in[k]->stride(0); s.stride_t[k] = in[k]->stride(1); }
    s.c = c;
    s.x = memory(x);
    s.r = memory(r);
    s.i = memory(i);
    s.decay = out<float>(decay);
    s.reset = (const uint8_t*)ptr(reset);
    return s;
}
void run_scan(plmpm_scan& s, const Tensor& x, bool backward) {
    const Site site(x);
    size_t need = 0;
    check(lib.scan_workspace(&s, backward, &need));
    const Tensor work = workspace(x, need);
    s.workspace = out(work);
    s.workspace_bytes = need;
    check((backward ? lib.scan_backward : lib.scan_forward)(&s, site.stream));
}
// -> h, last, checkpoint (undefined unless `keep`)
std::tuple<Tensor, Tensor, Tensor> scan_forward(const Tensor& x, const Tensor& r, const Tensor& i, const Tensor& decay, const Maybe& h0, const Maybe& reset, double c, bool keep) {
    const int64_t B = x.size(0), T = x.size(1), D = x.size(2);
    const Tensor h = at::empty({B, T, D}, x.options()), last = at::empty({B, D}, decay.options());
    const Tensor checkpoint = keep ? at::empty({(T + kCheckpoint - 1) / kCheckpoint, B, D}, decay.options()) : Tensor();
    if (B && T && D) {
        plmpm_scan s = scan_of(x, r, i, decay, reset, c);
        s.h0 = (const float*)ptr(h0);
        s.h = out(h);
        s.h_last = out<float>(last);
        s.checkpoint = out<float>(checkpoint);
        run_scan(s, x, false);
    } else if (h0) last.copy_(*h0);
    else last.zero_();
    return {h, last, checkpoint};
}
struct GatedScan : torch::autograd::Function<GatedScan> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& r, const Tensor& i, const Tensor& decay, const Maybe& h0, const Maybe& reset, double c) {
        at::AutoDispatchBelowADInplaceOrView below;
        auto [h, last, checkpoint] = scan_forward(x, r, i, decay, h0, reset, c, true);
        ctx->save_for_backward({x, r, i, decay, reset ? *reset : Tensor(), checkpoint});
        ctx->saved_data["c"] = c;
        ctx->saved_data["h0"] = h0.has_value();
        ctx->set_materialize_grads(false);
        return {h, last};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &r = saved[1], &i = saved[2], &decay = saved[3], &checkpoint = saved[5];
        const Maybe arrived[2] = {maybe(grads[0]), maybe(grads[1])};
        no_tangents({&arrived[0], &arrived[1]}, "gated_scan's backward pass");
        Tensor dx, dr, di, ddecay, dh0;
        {
            at::AutoDispatchBelowADInplaceOrView below;
            const int64_t B = x.size(0), T = x.size(1), D = x.size(2);
            dx = at::empty({B, T, D}, x.options());
            dr = at::empty({B, T, D}, x.options());
            di = at::empty({B, T, D}, x.options());
            ddecay = at::empty({D}, decay.options());
            if (ctx->saved_data["h0"].toBool()) dh0 = at::empty({B, D}, decay.options());
            Tensor dh, dlast;
            for (const auto& [to, k] : {std::pair(&dh, 0), std::pair(&dlast, 1)})
                if (grads[k].defined()) {
                    settle(grads[k]);
                    *to = grads[k].contiguous();
                }
            if (B && T && D) {
                plmpm_scan s = scan_of(x, r, i, decay, maybe(saved[4]), ctx->saved_data["c"].toDouble());
                s.checkpoint = out<float>(checkpoint);
                s.dh = out(dh);
                s.dlast = out<float>(dlast);
                s.dx = out(dx);
                s.dr = out(dr);
                s.di = out(di);
                s.ddecay = out<float>(ddecay);
                s.dh0 = out<float>(dh0);
                run_scan(s, x, true);
            } else {
                ddecay.zero_();
                if (dh0.defined()) { if (dlast.defined()) dh0.copy_(dlast); else dh0.zero_(); }
            }
        }
        return once({dx, dr, di, ddecay, dh0, Tensor(), Tensor()}, "gated_scan");
    }
};

void check_scan(const Tensor& x, const Tensor& r, const Tensor& i, const Tensor& decay, double c, int64_t dims) {
    REFUSE_IF(x.dim() != dims, "x has to be a tensor of ", dims, " dimensions, got ", x.dim());
    same_device(x, r, "r");
    same_device(x, i, "i");
    same_device(x, decay, "decay");
    REFUSE_IF(code_of(x.scalar_type()) < 0, "x has to be float32, bfloat16 or float16, got ", name_of(x.scalar_type()));
    for (const Tensor* t : {&r, &i})
        REFUSE_IF(t->sizes() != x.sizes() || t->scalar_type() != x.scalar_type(), "r and i have to match x: ", x.sizes(), " ", name_of(x.scalar_type()), ", got ", t->sizes(), " ", name_of(t->scalar_type()));
    REFUSE_IF(decay.dim() != 1 || decay.size(0) != x.size(-1) || decay.scalar_type() != at::kFloat || !decay.is_contiguous(),
              "decay has to be a contiguous float32 tensor of ", x.size(-1), " values");
    REFUSE_IF(!(c > 0.0 && c < 1e30), "c has to be positive and finite, got ", c);
}

std::tuple<Tensor, Tensor> gated_scan(Tensor x, Tensor r, Tensor i, Tensor decay, Maybe h0, Maybe reset, double c) {
    check_scan(x, r, i, decay, c, 3);
    if (h0) {
        same_device(x, *h0, "h0");
        REFUSE_IF(h0->dim() != 2 || h0->size(0) != x.size(0) || h0->size(1) != x.size(2) || h0->scalar_type() != at::kFloat,
                  "h0 has to be float32 (", x.size(0), ", ", x.size(2), "), got ", h0->sizes(), " ", name_of(h0->scalar_type()));
        settle(h0);
        h0 = h0->contiguous();
    }
    if (reset) {
        same_device(x, *reset, "reset");
        REFUSE_IF(reset->dim() != 2 || reset->size(0) != x.size(0) || reset->size(1) != x.size(1) || reset->scalar_type() != at::kBool,
                  "reset has to be bool (", x.size(0), ", ", x.size(1), "), got ", reset->sizes(), " ", name_of(reset->scalar_type()));
        reset = reset->contiguous();
    }
    for (Tensor* t : {&x, &r, &i}) {
        settle(*t);
        *t = rows_of(*t);
    }
    settle(decay);
    const Maybe mx(x), mr(r), mi(i), md(decay);
    no_tangents({&mx, &mr, &mi, &md, &h0}, "gated_scan");
    if (tracked({&mx, &mr, &mi, &md, &h0})) {
        auto o = GatedScan::apply(x, r, i, decay, h0, reset, c);
        return {o[0], o[1]};
    }
    auto [h, last, none] = scan_forward(x, r, i, decay, h0, reset, c, false);
    return {h, last};
}

// behind the last element of a tensor's memory
uintptr_t end_of(const Tensor& t) {
    int64_t last = 0;
    for (int64_t k = 0; k < t.dim(); ++k) last += (t.size(k) - 1) * t.stride(k);
    return (uintptr_t)memory(t) + (uintptr_t)((last + 1) * (int64_t)t.element_size());
}

Tensor gated_scan_step(Tensor x, Tensor r, Tensor i, Tensor decay, const Tensor& state, double c) {
    check_scan(x, r, i, decay, c, 2);
    same_device(x, state, "state");
    settled(state, "state");
    REFUSE_IF(state.sizes() != x.sizes() || state.scalar_type() != at::kFloat || !state.is_contiguous(), "state has to be a contiguous float32 tensor of ", x.sizes());
    const Maybe mx(x), mr(r), mi(i), md(decay), ms(state);
    no_tangents({&mx, &mr, &mi, &md, &ms}, "gated_scan_step");
    REFUSE_IF(tracked({&mx, &mr, &mi, &md, &ms}), "gated_scan_step has no gradients: call it under torch.no_grad(), or gated_scan with one step");
    for (Tensor* t : {&x, &r, &i}) {
        settle(*t);
        *t = rows_of(*t);
    }
    settle(decay);
    // an input that lies in the state would be read after another thread moved it on, unless each element is its own
    if (x.numel()) {
        const uintptr_t from = (uintptr_t)memory(state), to = end_of(state);
        const auto meets = [&](const Tensor& t) { return (uintptr_t)memory(t) < to && end_of(t) > from; };
        for (Tensor* t : {&x, &r, &i}) if (meets(*t) && !((uintptr_t)memory(*t) == from && t->is_contiguous())) *t = t->clone(at::MemoryFormat::Contiguous);
        if (meets(decay)) decay = decay.clone();
    }
    const Tensor h = at::empty({x.size(0), x.size(1)}, x.options());
    if (h.numel()) {
        plmpm_scan s{};
        s.dtype = code_of(x.scalar_type());
        s.batch = x.size(0);
        s.steps = 1;
        s.width = x.size(1);
        s.stride_b[0] = x.stride(0);
        s.stride_b[1] = r.stride(0);
        s.stride_b[2] = i.stride(0);
        s.c = c;
        s.x = memory(x);
        s.r = memory(r);
        s.i = memory(i);
        s.decay = out<float>(decay);
        s.h0 = out<float>(state);
        s.h = out(h);
        s.h_last = out<float>(state);
        run_scan(s, x, false);
        written(state);
    }
    return h;
}

// ---------------------------------------------------------------------------------------------- norms around a block
struct NormCall {
    Tensor keep[5];                     // the rows that the pointers are of (copies, where a layout could not be read in place)
    int kept = 0;
    plmpm_norm n{};
    NormCall(const Tensor& x, const Maybe& u, const Maybe& gate, const Maybe& scale, const Maybe& post, const Maybe& pre, at::ScalarType u_type, double eps, int64_t fn) {
        n.x_dtype = code_of(x.scalar_type());
        n.u_dtype = code_of(u_type);
        const Maybe& w = pre ? pre : post ? post : scale;
        n.w_dtype = w ? code_of(w->scalar_type()) : 0;
        n.gate_fn = (int32_t)fn;
        n.width = x.size(-1);
        n.rows = x.numel() / n.width;
        n.eps = eps;
        n.x = rows(x, n.stride_x);
        if (u) n.u = rows(*u, n.stride_u);
        if (gate) n.gate = rows(*gate, n.stride_gate);
        n.scale = ptr(scale);
        n.post = ptr(post);
        n.pre = ptr(pre);
    }
    const void* rows(const Tensor& t, int64_t& stride) {
        Tensor& k = keep[kept++];
        k = rows_of(t.dim() == 2 ? t : t.reshape({-1, n.width}));
        if (k.size(0) > 1 && k.stride(0) >= kFarRows) k = k.contiguous();
        stride = k.size(0) > 1 ? k.stride(0) : n.width;
        return memory(k);
    }
};
std::tuple<Tensor, Tensor> norm_forward(const Tensor& x, const Maybe& u, const Maybe& gate, const Maybe& scale, const Maybe& post, const Maybe& pre, at::ScalarType u_type, double eps, int64_t fn) {
    const Tensor y = u ? at::empty(x.sizes(), x.options()) : Tensor(), z = pre ? at::empty(x.sizes(), x.options().dtype(u_type)) : Tensor();
    if (x.numel()) {
        const Site site(x);
        NormCall call(x, u, gate, scale, post, pre, u_type, eps, fn);
        call.n.y = out(y);
        call.n.z = out(z);
        check(lib.norm_forward(&call.n, site.stream));
    }
    return {y, z};
}
struct BlockNorm : torch::autograd::Function<BlockNorm> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Maybe& u, const Maybe& gate, const Maybe& scale, const Maybe& post, const Maybe& pre, int64_t u_type, double eps, int64_t fn) {
        at::AutoDispatchBelowADInplaceOrView below;
        auto [y, z] = norm_forward(x, u, gate, scale, post, pre, (at::ScalarType)u_type, eps, fn);
        variable_list saved{x};
        for (const Maybe* t : {&u, &gate, &scale, &post, &pre}) saved.push_back(*t ? **t : Tensor());
        ctx->save_for_backward(saved);
        ctx->saved_data["u_type"] = u_type;
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["fn"] = fn;
        ctx->set_materialize_grads(false);
        variable_list given;            // (only what there is)
        for (const Tensor* t : {&y, &z}) if (t->defined()) given.push_back(*t);
        return given;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor& x = saved[0];
        const Maybe u = maybe(saved[1]), gate = maybe(saved[2]), scale = maybe(saved[3]), post = maybe(saved[4]), pre = maybe(saved[5]);
        Tensor dy = u ? grads[0] : Tensor(), dz = pre ? grads.back() : Tensor();
        const Maybe arrived[2] = {maybe(dy), maybe(dz)};
        no_tangents({&arrived[0], &arrived[1]}, "block_norm's backward pass");
        variable_list d(9);
        if (!dy.defined() && !dz.defined()) return d;
        {
            at::AutoDispatchBelowADInplaceOrView below;
            for (Tensor* t : {&dy, &dz}) if (t->defined()) settle(*t);
            for (int k = 0; k < 6; ++k) if (saved[k].defined()) d[k] = at::empty(saved[k].sizes(), saved[k].options());
            if (x.numel()) {
                const Site site(x);
                NormCall call(x, u, gate, scale, post, pre, (at::ScalarType)ctx->saved_data["u_type"].toInt(), ctx->saved_data["eps"].toDouble(), ctx->saved_data["fn"].toInt());
                plmpm_norm& n = call.n;
                if (dy.defined()) n.dy = call.rows(dy, n.stride_dy);
                if (dz.defined()) n.dz = call.rows(dz, n.stride_dz);
                n.dx = out(d[0]);
                n.du = out(d[1]);
                n.dgate = out(d[2]);
                n.dscale = out(d[3]);
                n.dpost = out(d[4]);
                n.dpre = out(d[5]);
                size_t need = 0;
                check(lib.norm_workspace(&n, &need));
                const Tensor work = workspace(x, need);
                n.workspace = out(work);
                n.workspace_bytes = need;
                check(lib.norm_backward(&n, site.stream));
            } else
                for (int k = 3; k < 6; ++k) if (d[k].defined()) d[k].zero_();
        }
        return once(std::move(d), "block_norm");
    }
};

std::tuple<Maybe, Maybe> block_norm(const Tensor& given, Maybe u, Maybe gate, Maybe scale, Maybe post, Maybe pre, double eps, int64_t fn, std::optional<at::ScalarType> dtype) {
    Tensor x = given;
    REFUSE_IF(x.dim() < 1, "x has to be a tensor with at least one dimension");
    const std::pair<const Maybe*, const char*> others[5] = {{&u, "u"}, {&gate, "gate"}, {&scale, "scale"}, {&post, "post"}, {&pre, "pre"}};
    for (const auto& [t, name] : others) if (*t) same_device(x, **t, name);
    REFUSE_IF(code_of(x.scalar_type()) < 0, "x has to be float32, bfloat16 or float16, got ", name_of(x.scalar_type()));
    const int64_t D = x.size(-1);
    REFUSE_IF(D > kMaxWidth, "rows of ", D, " values, at most ", kMaxWidth);
    REFUSE_IF(!u && !pre, "u, pre or both are needed");
    REFUSE_IF(!(eps >= 0.0 && eps < 1e30), "eps has to be zero or above, and finite, got ", eps);
    REFUSE_IF(!u && (gate || scale || post), "gate, scale and post go with u");
    const at::ScalarType u_type = u ? u->scalar_type() : dtype ? *dtype : x.scalar_type();
    REFUSE_IF(u && dtype && *dtype != u_type, "z has u's type ", name_of(u_type), ": dtype is for calls without u");
    REFUSE_IF(u && u->sizes() != x.sizes(), "u has to have x's shape ", x.sizes(), ", got ", u->sizes());
    REFUSE_IF(code_of(u_type) < 0 || (u_type != x.scalar_type() && x.scalar_type() != at::kFloat),
              "u (or dtype) has to be x's type, or 16 bits next to a float32 x: got ", name_of(u_type), " with ", name_of(x.scalar_type()));
    REFUSE_IF(gate && (gate->sizes() != x.sizes() || gate->scalar_type() != u_type), "gate has to have x's shape ", x.sizes(), " and the type ", name_of(u_type), ", got ", gate->sizes(), " ", name_of(gate->scalar_type()));
    const Maybe* first = nullptr;
    for (int k = 2; k < 5; ++k) {
        const Maybe& w = *others[k].first;
        if (!w) continue;
        if (!first) first = &w;
        REFUSE_IF(w->dim() != 1 || w->size(0) != D || !w->is_contiguous() || w->scalar_type() != (*first)->scalar_type() || code_of(w->scalar_type()) < 0,
                  others[k].second, " has to be a contiguous tensor of ", D, " values, of one floating type with the other weights");
    }
    settle(x);
    for (Maybe* t : {&u, &gate, &scale, &post, &pre}) settle(*t);
    Tensor y, z;
    const Maybe mx(x);
    no_tangents({&mx, &u, &gate, &scale, &post, &pre}, "block_norm");
    if (tracked({&mx, &u, &gate, &scale, &post, &pre})) {
        auto o = BlockNorm::apply(x, u, gate, scale, post, pre, (int64_t)u_type, eps, fn);
        if (u) y = o[0];
        if (pre) z = o.back();
    } else
        std::tie(y, z) = norm_forward(x, u, gate, scale, post, pre, u_type, eps, fn);
    return {u ? y : given, maybe(z)};
}

// ---------------------------------------------------------------------------------------------- AdamW
float* plain(const Tensor& t, int64_t n, const Tensor& step, const char* name, size_t k) {
    REFUSE_IF(t.scalar_type() != at::kFloat || t.numel() != n || !t.is_contiguous() || t.device() != step.device(),
              name, " ", k, " has to be ", n, " contiguous float32 values on the parameters' device");
    settled(t, name);
    return out<float>(t);
}
void* codes_of(const Tensor& t, int64_t n, const Tensor& step, at::ScalarType type, const char* name, size_t k) {
    REFUSE_IF(t.scalar_type() != type || t.numel() != n || !t.is_contiguous() || t.device() != step.device(),
              name, " ", k, ": codes have to be ", n, " contiguous ", name_of(type), " values on the parameters' device");
    settled(t, name);
    return memory(t);
}
int64_t blocks_of(int64_t n) { return (n + kBlock - 1) / kBlock; }
// The memory that a call touches through its lists of tensors: what it writes it may touch through one of them only, or two updates would race.
struct Touched {
    struct Range {
        uintptr_t from;
        int64_t bytes;                  // below zero: only read
    };
    std::vector<Range> ranges;
    void reads(const void* p, int64_t bytes) { ranges.push_back({(uintptr_t)p, -bytes}); }
    void writes(const void* p, int64_t bytes) { ranges.push_back({(uintptr_t)p, bytes}); }
    bool races() {
        std::sort(ranges.begin(), ranges.end(), [](const Range& a, const Range& b) { return a.from < b.from; });
        uintptr_t read = 0, written = 0;        // where what was read or written so far ends
        for (const Range& r : ranges)
            if (r.bytes > 0) {
                if (r.from < std::max(read, written)) return true;
                written = r.from + (uintptr_t)r.bytes;
            } else {
                if (r.from < written) return true;
                read = std::max(read, r.from + (uintptr_t)-r.bytes);
            }
        return false;
    }
};

Maybe adamw_step(const std::vector<Tensor>& params, const std::vector<Maybe>& grads, const std::vector<Tensor>& first, const std::vector<Tensor>& second,
                 const std::vector<Tensor>& first_scales, const std::vector<Tensor>& second_scales, const std::vector<Maybe>& masters, const Tensor& step, int64_t bits,
                 double lr, double beta_1, double beta_2, double epsilon, double weight_decay, double max_norm, double lo, double hi) {
    const size_t count = params.size();
    REFUSE_IF(grads.size() != count || first.size() != count || second.size() != count || (!masters.empty() && masters.size() != count),
              "params, grads, first, second and masters have to be of one length");
    REFUSE_IF(step.dim() != 1 || step.size(0) != 2 || step.scalar_type() != at::kLong || !step.is_contiguous(), "step has to be an int64 tensor of two values");
    settled(step, "step");
    std::vector<plmpm_adamw_tensor> table;
    std::vector<Tensor> keep;
    std::vector<size_t> touched;
    Touched memory_of;
    const bool tangents = tangents_about();
    table.reserve(count);
    memory_of.ranges.reserve(5 * count + 1);
    memory_of.writes(memory(step), 2 * sizeof(int64_t));
    for (size_t k = 0; k < count; ++k) {
        if (!grads[k]) continue;
        const Tensor& p = params[k];
        if (tangents) {
            const Maybe mp(p);
            no_tangents({&mp, &grads[k]}, "adamw_step");
        }
        Tensor g = *grads[k];
        const int64_t n = p.numel();
        const int code = code_of(p.scalar_type());
        REFUSE_IF(code < 0 || !p.is_contiguous() || p.device() != step.device(), "parameter ", k, " has to be a contiguous float32, bfloat16 or float16 tensor on ", step.device());
        REFUSE_IF(g.scalar_type() != p.scalar_type() || g.sizes() != p.sizes() || g.device() != step.device(),
                  "gradient ", k, " has to match its parameter: ", p.sizes(), " ", name_of(p.scalar_type()), " on ", step.device());
        settled(p, "a parameter");
        settle(g);
        if (!g.is_contiguous()) g = g.contiguous();
        if (!g.is_same(*grads[k])) keep.push_back(g);
        plmpm_adamw_tensor t{};
        t.p = memory(p);
        t.g = memory(g);
        t.n = n;
        t.dtype = code;
        if (bits == 8) {
            t.m = codes_of(first[k], n, step, at::kChar, "first moment", k);
            t.v = codes_of(second[k], n, step, at::kByte, "second moment", k);
            t.m_scale = plain(first_scales[k], blocks_of(n), step, "scales of first moment", k);
            t.v_scale = plain(second_scales[k], blocks_of(n), step, "scales of second moment", k);
        } else {
            t.m = plain(first[k], n, step, "first moment", k);
            t.v = plain(second[k], n, step, "second moment", k);
        }
        if (!masters.empty() && masters[k]) {
            REFUSE_IF(code == PLMPM_NN_F32, "parameter ", k, " is float32: a master copy goes with 16 bits");
            t.master = plain(*masters[k], n, step, "master", k);
        }
        if (!n) continue;
        const int64_t size = n * (code == PLMPM_NN_F32 ? 4 : 2), moment = bits == 8 ? n : 4 * n, scales = 4 * blocks_of(n);
        memory_of.writes(t.p, size);
        if (t.g != t.p) memory_of.reads(t.g, size);               // (the parameter itself as its gradient: each element is read before it is written)
        memory_of.writes(t.m, moment);
        memory_of.writes(t.v, moment);
        if (t.m_scale) memory_of.writes(t.m_scale, scales);
        if (t.v_scale) memory_of.writes(t.v_scale, scales);
        if (t.master) memory_of.writes(t.master, 4 * n);
        table.push_back(t);
        touched.push_back(k);
    }
    REFUSE_IF(memory_of.races(), "a parameter, a moment of it, its master or step is in the list twice, or overlaps another tensor of the call: the updates would race");
    Maybe norm;
    if (max_norm > 0) norm = at::empty({}, step.options().dtype(at::kFloat));
    if (table.empty()) {
        if (norm) norm->zero_();
        return norm;
    }
    const Site site(step);
    plmpm_adamw a{};
    a.state_bits = (int32_t)bits;
    a.lr = lr;
    a.beta_1 = beta_1;
    a.beta_2 = beta_2;
    a.epsilon = epsilon;
    a.weight_decay = weight_decay;
    a.max_norm = max_norm;
    a.lo = lo;
    a.hi = hi;
    a.step = out<int64_t>(step);
    a.grad_norm = norm ? out<float>(*norm) : nullptr;
    size_t need = 0;
    check(lib.adamw_workspace(&a, table.data(), (int)table.size(), &need));
    const Tensor work = workspace(step, need);
    a.workspace = out(work);
    a.workspace_bytes = need;
    check(lib.adamw_step(&a, table.data(), (int)table.size(), site.stream));
    written(step);
    for (size_t k : touched) {
        for (const Tensor* t : {&params[k], &first[k], &second[k]}) written(*t);
        if (bits == 8) for (const Tensor* t : {&first_scales[k], &second_scales[k]}) written(*t);
        if (!masters.empty() && masters[k]) written(*masters[k]);
    }
    return norm;
}

void adamw_values(const std::vector<Tensor>& codes, const std::vector<Tensor>& scales, const std::vector<Tensor>& values) {
    const size_t count = codes.size();
    REFUSE_IF(values.size() != count, "out has to have a tensor for each moment");
    if (!count) return;
    std::vector<const void*> c;
    std::vector<const float*> s;
    std::vector<float*> o;
    std::vector<int64_t> sizes;
    std::vector<int32_t> which;
    Touched memory_of;
    for (size_t k = 0; k < count; ++k) {
        const int64_t n = codes[k].numel();
        const at::ScalarType type = codes[k].scalar_type();
        REFUSE_IF(type != at::kChar && type != at::kByte, "moment ", k, ": codes have to be int8 or uint8, got ", name_of(type));
        c.push_back(codes_of(codes[k], n, codes[0], type, "moment", k));
        s.push_back(plain(scales[k], blocks_of(n), codes[0], "scales of moment", k));
        o.push_back(plain(values[k], n, codes[0], "out", k));
        sizes.push_back(n);
        which.push_back(type == at::kByte);
        if (!n) continue;
        memory_of.reads(c.back(), n);
        memory_of.reads(s.back(), 4 * blocks_of(n));
        memory_of.writes(o.back(), 4 * n);
    }
    REFUSE_IF(memory_of.races(), "a tensor of out is in the list twice, or overlaps another tensor of the call");
    const Site site(codes[0]);
    check(lib.adamw_values(c.data(), s.data(), o.data(), sizes.data(), which.data(), (int)count, site.stream));
    for (const Tensor& t : values) written(t);
}

// the library's entries by name, the class of its errors, and whether they take host memory
void attach(const std::unordered_map<std::string, uintptr_t>& at, bool host) {
    Library l;
    const auto set = [&](auto& f, const char* name) { f = reinterpret_cast<std::remove_reference_t<decltype(f)>>(at.at(name)); };
    set(l.last_error, "plmpm_last_error");
    set(l.scan_workspace, "plmpm_scan_workspace");
    set(l.scan_forward, "plmpm_scan_forward");
    set(l.scan_backward, "plmpm_scan_backward");
    set(l.norm_workspace, "plmpm_norm_workspace");
    set(l.norm_forward, "plmpm_norm_forward");
    set(l.norm_backward, "plmpm_norm_backward");
    set(l.adamw_workspace, "plmpm_adamw_workspace");
    set(l.adamw_step, "plmpm_adamw_step");
    set(l.adamw_values, "plmpm_adamw_values");
    l.host = host;
    lib = l;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    namespace py = pybind11;
    static py::handle error = PyExc_RuntimeError;       // (attach() puts _lib.EngineError here, for the process's life)
    m.def("attach", [](const std::unordered_map<std::string, uintptr_t>& at, py::object error_class, bool host) {
        attach(at, host);
        error = error_class.release();
    });
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const EngineError& e) {
            PyErr_SetString(error.ptr(), e.what());
        } catch (const c10::Error&) {                    // (torch's own, as torch gives them: out of memory above all)
            torch::translate_exception_to_python(p);
        }
    });
    const auto unlocked = py::call_guard<py::gil_scoped_release>();
    m.def("require_device", [](const Tensor& t) { Site site(t); });
    m.def("gated_scan", &gated_scan, unlocked);
    m.def("gated_scan_step", &gated_scan_step, unlocked);
    m.def("block_norm", &block_norm, unlocked);
    m.def("adamw_step", &adamw_step, unlocked);
    m.def("adamw_values", &adamw_values, unlocked);
}
