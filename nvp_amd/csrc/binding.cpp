// The conditioning operators (nvp_amd.codes, nvp_amd.trunk, nvp_amd.quantize.linear8) as torch calls: argument checks, output and workspace allocation,
// autograd nodes, and the calls of the C ABI (include/nvp_hip.h) on the current stream of the tensors' device.  C++ rather than Python because of what small calls
// cost: a backward pass runs on autograd's own thread, and a Python backward has to take the interpreter lock there and run its few dozen lines with cold
// caches - 105 to 200 us for a forward and backward pass whose kernels take 10 to 30 us; as C++ nodes 48 us (lookup) to 86 us (residual step with all its
// gradients), some 45 of them for waking that thread (39 us in all where the engine is told to stay on the caller's).
// Host code only: no kernel lives here.  The library it calls is the one nvp_amd._lib has loaded (bind()).
#include <dlfcn.h>

#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>
#include <ATen/ATen.h>

#include <cmath>
#include <cstdint>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/nvp_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

struct Api {
    decltype(&::nvp_lookup_fwd) lookup_fwd;
    decltype(&::nvp_lookup_bwd_workspace_bytes) lookup_ws;
    decltype(&::nvp_lookup_bwd) lookup_bwd;
    decltype(&::nvp_residual_fwd) residual_fwd;
    decltype(&::nvp_residual_bwd_workspace_bytes) residual_ws;
    decltype(&::nvp_residual_bwd) residual_bwd;
    decltype(&::nvp_linear8_workspace_bytes) linear8_ws;
    decltype(&::nvp_linear8) linear8;
} api;

void bind(const std::string& path) {
    void* lib = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);      // already loaded: another handle of the same library
    TORCH_CHECK(lib, "nvp_amd: ", dlerror());
    const auto get = [&](auto& f, const char* name) {
        f = reinterpret_cast<std::decay_t<decltype(f)>>(dlsym(lib, name));
        TORCH_CHECK(f, "nvp_amd: ", path, " does not export ", name);
    };
    get(api.lookup_fwd, "nvp_lookup_fwd");
    get(api.lookup_ws, "nvp_lookup_bwd_workspace_bytes");
    get(api.lookup_bwd, "nvp_lookup_bwd");
    get(api.residual_fwd, "nvp_residual_fwd");
    get(api.residual_ws, "nvp_residual_bwd_workspace_bytes");
    get(api.residual_bwd, "nvp_residual_bwd");
    get(api.linear8_ws, "nvp_linear8_workspace_bytes");
    get(api.linear8, "nvp_linear8");
}

// ---- shared pieces -------------------------------------------------------------------------------------------------------------------------------
int type_number(at::ScalarType t) { return t == at::kFloat ? NVP_F32 : t == at::kBFloat16 ? NVP_BF16 : t == at::kHalf ? NVP_F16 : -1; }
int stream_type(const Tensor& t, const char* what) {
    const int n = type_number(t.scalar_type());
    TORCH_CHECK(n >= 0, what, ": expected float32, bfloat16 or float16, got ", t.scalar_type());
    return n;
}
void one_device(std::initializer_list<const Tensor*> ts) {
    const Tensor& first = **ts.begin();
    for (const Tensor* t : ts) {
        if (!t->defined()) continue;
        TORCH_CHECK(t->is_cuda(), "nvp_amd kernels need tensors on a HIP device (got a CPU tensor); there is no CPU path in the product - move the module/inputs with .cuda()");
        TORCH_CHECK(t->device() == first.device(), "expected every tensor on ", first.device(), ", got one on ", t->device());
    }
}
// A kernel call carries no forward-mode tangent along: its output would have none, which is the tangent zero.
void no_tangents(const char* what, std::initializer_list<const Tensor*> ts) {
    for (const Tensor* t : ts)
        TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), what, " has no forward-mode derivative: call it on tensors without a tangent (torch.autograd.forward_ad.unpack_dual)");
}
// A tracer sees the output's allocation and not the kernel: what it records would return uninitialised memory.  (A HIP graph captures the kernel itself.)
void not_recorded(const char* what) {
    typedef c10::impl::TorchDispatchModeKey Key;
    bool recorded = torch::jit::tracer::isTracing();
    for (const Key k : {Key::PROXY, Key::FAKE, Key::FUNCTIONAL}) recorded = recorded || c10::impl::TorchDispatchModeTLS::get_mode(k).has_value();
    TORCH_CHECK(!recorded, what, " cannot be recorded by torch.jit.trace, torch.fx or torch.export: call it outside the traced function");
}
void ok(int64_t rc, const char* what) {
    if (rc == 0) return;
    TORCH_CHECK(false, what, " failed: ", rc == NVP_ERR_BADARG ? std::string("bad argument") : rc == NVP_ERR_UNSUPPORTED ? std::string("unsupported configuration") : "hipError " + std::to_string(rc));
}
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
// rows side by side, values as they read (a view that negates, as the imaginary part of a conjugate, keeps its values' other sign in memory)
Tensor dense(const Tensor& t) { return t.defined() ? (t.is_neg() ? t.resolve_neg() : t).contiguous() : t; }
Tensor dense(const Maybe& t) { return t ? dense(*t) : Tensor(); }
Tensor workspace(int64_t bytes, const Tensor& like, const char* what) {
    if (bytes < 0) ok(bytes, what);
    return bytes ? at::empty({bytes}, like.options().dtype(at::kByte)) : Tensor();
}
int64_t bytes_of(const Tensor& ws) { return ws.defined() ? ws.numel() : 0; }
bool wants_grad(std::initializer_list<const Tensor*> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : ts)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}
// Gradients of a backward pass that is itself recorded (create_graph=True): the kernels cannot be differentiated a second time, and say so when it is tried.
variable_list once(variable_list grads, const char* what) {
    if (!at::GradMode::is_enabled()) return grads;
    variable_list in;
    for (Tensor& g : grads)
        if (g.defined()) {
            g = g.detach();
            g.set_requires_grad(true);
            in.push_back(g);
        }
    if (in.empty()) return grads;
    const auto err = std::make_shared<torch::autograd::DelayedError>(std::string(what) + " can be differentiated once only", (int)in.size());
    variable_list out = (*err)(std::move(in));
    size_t k = 0;
    for (Tensor& g : grads)
        if (g.defined()) g = out[k++];
    return grads;
}

// ---- lookup --------------------------------------------------------------------------------------------------------------------------------------
Tensor lookup_run(const Tensor& ids, const Tensor& table, double scale, at::ScalarType type) {
    auto shape = ids.sizes().vec();
    shape.push_back(table.size(1));
    Tensor out = at::empty(shape, table.options().dtype(type));
    ok(api.lookup_fwd(ptr(ids), ids.scalar_type() == at::kLong, ptr(table), type_number(table.scalar_type()), ptr(out), type_number(type), ids.numel(), table.size(0), table.size(1), (float)scale,
                      stream_of(table)),
       "nvp_lookup_fwd");
    return out;
}
struct Lookup : torch::autograd::Function<Lookup> {
    static Tensor forward(AutogradContext* ctx, const Tensor& ids, const Tensor& table, double scale, int64_t type) {
        ctx->save_for_backward({ids});
        ctx->saved_data["codes"] = table.size(0);
        ctx->saved_data["type"] = (int64_t)table.scalar_type();
        ctx->saved_data["scale"] = scale;
        return lookup_run(ids, table, scale, (at::ScalarType)type);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        not_recorded("the gradient of lookup");
        no_tangents("the gradient of lookup", {&grads[0]});
        Tensor ids = ctx->get_saved_variables()[0], dout = dense(grads[0]);
        const int64_t codes = ctx->saved_data["codes"].toInt(), dim = dout.size(-1), n = ids.numel();
        const auto type = (at::ScalarType)ctx->saved_data["type"].toInt();
        const c10::DeviceGuard guard(dout.device());
        Tensor ws = workspace(api.lookup_ws(n, codes, dim), dout, "nvp_lookup_bwd_workspace_bytes");
        Tensor dtable = at::empty({codes, dim}, dout.options().dtype(type));
        ok(api.lookup_bwd(ptr(ids), ids.scalar_type() == at::kLong, ptr(dout), type_number(dout.scalar_type()), ptr(dtable), type_number(type), n, codes, dim,
                          (float)ctx->saved_data["scale"].toDouble(), ptr(ws), bytes_of(ws), stream_of(dout)),
           "nvp_lookup_bwd");
        return once({Tensor(), dtable, Tensor(), Tensor()}, "lookup");
    }
};
Tensor lookup(const Tensor& ids, const Tensor& table, double scale, std::optional<at::ScalarType> dtype, bool verify) {
    TORCH_CHECK(ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt, "lookup: ids must be int64 or int32, got ", ids.scalar_type());
    TORCH_CHECK(table.dim() == 2 && table.size(0) >= 1 && table.size(1) >= 1, "lookup: the table must be [codes, dim] with at least one code, got ", table.sizes());
    stream_type(table, "lookup");
    const at::ScalarType type = dtype.value_or(table.scalar_type());
    TORCH_CHECK(type_number(type) >= 0 && (table.scalar_type() == at::kFloat || type == table.scalar_type()), "lookup: a ", table.scalar_type(), " table cannot be read as ", type);
    TORCH_CHECK(std::isfinite((float)scale), "lookup: scale must be finite in 32 bits, got ", scale);
    not_recorded("lookup");
    no_tangents("lookup", {&table});
    one_device({&table, &ids});
    const c10::DeviceGuard guard(table.device());
    if (verify && ids.numel()) {
        const int64_t most = ids.max().item().toLong();
        TORCH_CHECK_INDEX(most < table.size(0), "lookup: id ", most, " in a table of ", table.size(0), " codes");
    }
    const Tensor i = dense(ids), t = dense(table);
    return wants_grad({&t}) ? Lookup::apply(i, t, scale, (int64_t)type) : lookup_run(i, t, scale, type);
}

// ---- gated residual step --------------------------------------------------------------------------------------------------------------------------
struct Step {
    Tensor x, h, gate, post, next;
    int64_t gate_rows, act;
    double scale, eps;
    nvp_residual args() const {
        const Tensor& w = post.defined() ? post : next;
        const int64_t dim = x.size(-1);
        return {ptr(x), ptr(h), ptr(gate), ptr(post), ptr(next), x.numel() / dim, gate_rows, (int32_t)dim, type_number(x.scalar_type()), type_number(w.scalar_type()), (int32_t)act, (float)scale,
                (float)eps};
    }
};
// y and u, those that exist
variable_list residual_run(const Step& s, const Tensor& stats) {
    Tensor y = s.h.defined() ? at::empty_like(s.x) : Tensor(), u = s.next.defined() ? at::empty_like(s.x) : Tensor();
    if (s.x.numel()) {
        const nvp_residual a = s.args();
        ok(api.residual_fwd(&a, ptr(y), ptr(u), static_cast<float*>(ptr(stats)), stream_of(s.x)), "nvp_residual_fwd");
    }
    variable_list out;
    if (y.defined()) out.push_back(y);
    if (u.defined()) out.push_back(u);
    return out;
}
struct Residual : torch::autograd::Function<Residual> {
    // An absent tensor is no input of the node: the node's edges count those that are there.
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Maybe& mh, const Maybe& mgate, const Maybe& mpost, const Maybe& mnext, int64_t gate_rows, int64_t act, double scale,
                                 double eps) {
        const Tensor none, &h = mh ? *mh : none, &gate = mgate ? *mgate : none, &post = mpost ? *mpost : none, &next = mnext ? *mnext : none;
        const Step s{x, h, gate, post, next, gate_rows, act, scale, eps};
        Tensor stats = at::empty({x.numel() / x.size(-1), 2}, x.options().dtype(at::kFloat));
        ctx->save_for_backward({x, h, gate, post, next, stats});
        ctx->saved_data["rows"] = gate_rows;
        ctx->saved_data["act"] = act;
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["eps"] = eps;
        ctx->set_materialize_grads(false);
        return residual_run(s, stats);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list v = ctx->get_saved_variables();
        const Step s{v[0], v[1], v[2], v[3], v[4], ctx->saved_data["rows"].toInt(), ctx->saved_data["act"].toInt(), ctx->saved_data["scale"].toDouble(), ctx->saved_data["eps"].toDouble()};
        variable_list out(9);
        const Tensor dy = s.h.defined() ? dense(grads[0]) : Tensor(), du = s.next.defined() ? dense(grads.back()) : Tensor();
        if (!dy.defined() && !du.defined()) return out;
        not_recorded("the gradient of gated_residual");
        no_tangents("the gradient of gated_residual", {&dy, &du});
        const c10::DeviceGuard guard(s.x.device());
        const Tensor* in[5] = {&s.x, &s.h, &s.gate, &s.post, &s.next};
        const bool empty = s.x.numel() == 0;
        int edge = 0;
        for (int k = 0; k < 5; ++k)
            if (in[k]->defined() && ctx->needs_input_grad(edge++)) out[k] = empty ? at::zeros_like(*in[k]) : at::empty_like(*in[k]);
        if (!empty) {
            const nvp_residual a = s.args();
            Tensor ws = workspace(api.residual_ws(&a), s.x, "nvp_residual_bwd_workspace_bytes");
            ok(api.residual_bwd(&a, static_cast<const float*>(ptr(v[5])), ptr(dy), ptr(du), ptr(out[0]), ptr(out[1]), ptr(out[2]), ptr(out[3]), ptr(out[4]), ptr(ws), bytes_of(ws), stream_of(s.x)),
               "nvp_residual_bwd");
        }
        return once(std::move(out), "gated_residual");
    }
};
void check_rows(const Tensor& x, const char* what) {
    stream_type(x, what);
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= 8192, what, ": expected [..., D] with 1 <= D <= 8192, got ", x.sizes());
}
void check_weight(const Tensor& w, const Tensor& x, const char* what) {
    TORCH_CHECK(w.dim() == 1 && w.size(0) == x.size(-1) && (w.scalar_type() == at::kFloat || w.scalar_type() == x.scalar_type()), what, ": expected a weight [", x.size(-1), "] of float32 or ",
                x.scalar_type(), ", got ", w.scalar_type(), " ", w.sizes());
}
// How many rows of D the gate has; row r of x uses gate row r / (rows of x / rows of the gate): the gate's leading dimensions are x's up to some point and 1
// from there on (dimensions missing on the left count as 1).
int64_t gate_rows(const Tensor& x, const Tensor& gate) {
    const int64_t nx = x.dim() - 1, ng = gate.dim() - 1;
    bool fine = ng >= 0 && gate.scalar_type() == x.scalar_type() && gate.size(-1) == x.size(-1) && ng <= nx;
    int64_t rows = 1;
    if (fine) {
        int64_t k = ng;                                          // the gate's leading dimensions without the ones at their end
        while (k > 0 && gate.size(k - 1) == 1) --k;
        for (int64_t d = 0; d < k; ++d) rows *= gate.size(d);
        if (k > 0) {
            for (int64_t d = 0; d < nx - ng; ++d) fine = fine && x.size(d) == 1;      // missing on the left: 1, and so must x's be
            for (int64_t d = 0; d < k; ++d) fine = fine && gate.size(d) == x.size(d + nx - ng);
        }
    }
    TORCH_CHECK(fine, "gated_residual: a gate for x ", x.sizes(), " (", x.scalar_type(), ") has its type and its shape, or 1 in place of the last leading dimensions, got ", gate.scalar_type(), " ",
                gate.sizes());
    return rows;
}
variable_list residual(const Tensor& x, const Tensor& h, const Tensor& gate, const Tensor& post, const Tensor& next, double scale, int64_t act, double eps, const char* what) {
    TORCH_CHECK(eps >= 0 && std::isfinite((float)eps), what, ": eps must be finite in 32 bits and not negative, got ", eps);
    const int64_t grows = gate.defined() ? gate_rows(x, gate) : 1;
    not_recorded(what);
    no_tangents(what, {&x, &h, &gate, &post, &next});
    one_device({&x, &h, &gate, &post, &next});
    const c10::DeviceGuard guard(x.device());
    const Tensor xc = dense(x), hc = dense(h), gc = dense(gate), pc = dense(post), nc = dense(next);
    const auto maybe = [](const Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); };
    if (wants_grad({&xc, &hc, &gc, &pc, &nc})) return Residual::apply(xc, maybe(hc), maybe(gc), maybe(pc), maybe(nc), grows, act, scale, eps);
    return residual_run({xc, hc, gc, pc, nc, grows, act, scale, eps}, Tensor());
}
Tensor pre_norm(const Tensor& x, const Tensor& weight, double eps) {
    check_rows(x, "pre_norm");
    check_weight(weight, x, "pre_norm");
    return residual(x, Tensor(), Tensor(), Tensor(), weight, 1.0, 0, eps, "pre_norm")[0];
}
variable_list gated_residual(const Tensor& x, const Tensor& h, const Maybe& gate, const Tensor& post, const Maybe& next, double scale, int64_t act, double eps) {
    const char* what = "gated_residual";
    check_rows(x, what);
    TORCH_CHECK(h.sizes() == x.sizes() && h.scalar_type() == x.scalar_type(), "gated_residual: h must be like x (", x.scalar_type(), " ", x.sizes(), "), got ", h.scalar_type(), " ", h.sizes());
    check_weight(post, x, what);
    if (next) {
        check_weight(*next, x, what);
        TORCH_CHECK(next->scalar_type() == post.scalar_type(), "gated_residual: the two weights must be of one type, got ", post.scalar_type(), " and ", next->scalar_type());
    }
    TORCH_CHECK(std::isfinite((float)scale), "gated_residual: scale must be finite in 32 bits, got ", scale);
    return residual(x, h, gate.value_or(Tensor()), post, next.value_or(Tensor()), scale, act, eps, what);
}

// ---- 8-bit linear layer ---------------------------------------------------------------------------------------------------------------------------
Tensor linear8(const Tensor& x, const Tensor& q, const Tensor& e, const Maybe& bias) {
    TORCH_CHECK(x.dim() >= 1, "linear8 expects x [..., K]");
    const int64_t k = x.size(-1), kb = (k + 127) / 128;
    TORCH_CHECK(q.scalar_type() == at::kFloat8_e4m3fn && e.scalar_type() == at::kByte && q.dim() == 2 && e.dim() == 2, "linear8: expected a float8_e4m3fn matrix and its uint8 scales, got ",
                q.scalar_type(), " ", q.sizes(), " and ", e.scalar_type(), " ", e.sizes());
    const int64_t n = q.size(0);
    TORCH_CHECK(k >= 1 && q.size(1) == kb * 128 && e.size(0) == (n + 127) / 128 && e.size(1) == kb, "linear8: ", k, " columns in blocks of 128 x 128 need q [R, ", kb * 128, "] and e [ceil(R / 128), ", kb,
                "], got ", q.sizes(), " and ", e.sizes());
    TORCH_CHECK(n >= 1, "linear8: the weight has no rows");
    const int type = stream_type(x, "linear8");
    const Tensor b = dense(bias);
    TORCH_CHECK(!b.defined() || (b.scalar_type() == x.scalar_type() && b.dim() == 1 && b.size(0) == n), "linear8: bias must be ", x.scalar_type(), " [", n, "], got ",
                b.defined() ? b.scalar_type() : x.scalar_type(), " ", b.defined() ? b.sizes() : x.sizes());
    TORCH_CHECK_NOT_IMPLEMENTED(!wants_grad({&x, &b}), "linear8 is an inference-only path: call it under torch.no_grad() or on tensors that need no gradient");
    not_recorded("linear8");
    no_tangents("linear8", {&x, &b});
    one_device({&x, &q, &e, &b});
    const c10::DeviceGuard guard(x.device());
    const Tensor xc = dense(x), ec = e.contiguous();
    Tensor qc = q.contiguous();
    if (reinterpret_cast<uintptr_t>(qc.data_ptr()) % 16) qc = qc.clone();      // (the kernel's 16-byte loads; the allocator's addresses are aligned)
    const int64_t rows = xc.numel() / k;
    auto shape = x.sizes().vec();
    shape.back() = n;
    Tensor y = at::empty(shape, x.options().requires_grad(false));
    if (rows == 0) return y;
    const int64_t need = api.linear8_ws(rows, k, n);
    Tensor ws = workspace(need, x, "nvp_linear8_workspace_bytes");
    ok(api.linear8(ptr(xc), type, static_cast<const uint8_t*>(ptr(qc)), static_cast<const uint8_t*>(ptr(ec)), ptr(b), ptr(y), rows, k, n, ptr(ws), need, stream_of(x)), "nvp_linear8");
    return y;
}

}  // namespace

PYBIND11_MODULE(nvp_binding, m) {
    namespace py = pybind11;
    m.def("bind", &bind);
    m.def("not_recorded", &not_recorded);
    m.def("lookup", &lookup, py::call_guard<py::gil_scoped_release>());
    m.def("pre_norm", &pre_norm, py::call_guard<py::gil_scoped_release>());
    m.def("gated_residual", &gated_residual, py::call_guard<py::gil_scoped_release>());
    m.def("linear8", &linear8, py::call_guard<py::gil_scoped_release>());
}
