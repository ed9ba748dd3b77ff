// The host side of the sequence operators (sequence.py) in C++: outputs and workspaces, the launch on the current stream and
// the autograd nodes.  This bounds small calls: through ctypes and Python autograd functions a lookup of 256 tokens took 8.7 us,
// a single-token step 8.8, a lookup of 8192 with its gradient 85 and a short scan with its gradient 111 (kernels 3, 3, 30
// and 29 us); from here 3.7, 3.8, 51 and 60, of which 42 are what torch takes to run any function's gradient.
// The arguments are checked in sequence.py, those of a usual call here; the kernels and their C-ABI are in libdvae_hip.so, whose functions bind() gets.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <stdexcept>

#include "dvae_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

struct DvaeError : std::runtime_error {  // DvaeHipError in Python
    using std::runtime_error::runtime_error;
};

#define DVAE_FUNCTIONS(F)                                                                                                     \
    F(dvae_last_error) F(dvae_embed_fwd) F(dvae_embed_bwd_ws_bytes) F(dvae_embed_bwd) F(dvae_scan_state_floats) F(dvae_scan_ws_bytes) \
    F(dvae_scan_fwd) F(dvae_scan_bwd) F(dvae_scan_step)
#define F(name) decltype(&::name) p_##name = nullptr;
DVAE_FUNCTIONS(F)
#undef F

void bind(const std::map<std::string, size_t>& addresses) {
#define F(name) p_##name = reinterpret_cast<decltype(p_##name)>(addresses.at(#name));
    DVAE_FUNCTIONS(F)
#undef F
}

[[noreturn]] void fail(const char* what, long rc) {
    const char* why = p_dvae_last_error();
    throw DvaeError(std::string(what) + " failed (" + std::to_string(rc) + "): " + (why ? why : "?"));
}

int code(const Tensor& t) {
    return t.scalar_type() == at::kFloat ? DVAE_F32 : t.scalar_type() == at::kBFloat16 ? DVAE_BF16 : DVAE_F16;
}
int wide(const Tensor& t) { return t.scalar_type() == at::kLong; }
int wide(const Maybe& t) { return t && wide(*t); }
void* ptr(const Maybe& t) { return t ? t->data_ptr() : nullptr; }

// A size that the library takes in 32 bits.  Its own limits are lower, but a size cut to 32 bits would pass them.
int32_t size32(const char* what, int64_t v) {
    if (v > INT32_MAX) throw DvaeError(std::string(what) + ": " + std::to_string(v) + " are not supported");
    return (int32_t)v;
}
// a function of the library; no argument may be wider than its parameter
template <typename P, typename A> constexpr bool cut = std::is_integral_v<P> && std::is_integral_v<A> && sizeof(P) < sizeof(A);
template <typename R, typename... Ps, typename... As> R call(R (*fn)(Ps...), As... args) {
    static_assert(!(cut<Ps, As> || ...), "narrow it with size32");
    return fn(args...);
}

// calls a function of the library with the current stream of `device`, that device being the current one
template <typename Fn, typename... Args> void enqueue(const char* what, at::Device device, Fn* fn, Args... args) {
    c10::DeviceGuard guard(device);
    const int rc = call(fn, args..., (void*)c10::hip::getCurrentHIPStream(device.index()).stream());
    if (rc != 0) fail(what, rc);
}

Tensor workspace(const char* what, int64_t bytes, at::Device device) {
    if (bytes < 0) fail(what, bytes);
    return at::empty({bytes}, at::TensorOptions(at::kByte).device(device));
}

// Tensors whose elements torch holds negated (x.conj().imag) are written out first, here and below: the library reads memory.
// The rows of a [N, D] or [B, T, D] matrix whose elements lie side by side in a row: in place where the rows have one
// stride of at most 2^23 elements (the recurrence addresses a few rows with 32-bit offsets), else of a copy.
struct Rows {
    Tensor keep;
    int64_t n, d, ld;
    explicit Rows(const Tensor& given) : keep(given.resolve_neg()), d(given.size(-1)) {
        const Tensor t = keep;
        const bool flat = t.dim() == 2;
        const int64_t B = t.size(0), T = flat ? 1 : t.size(1), step = flat || T == 1 ? t.stride(0) : t.stride(1);
        n = B * T;
        ld = n > 1 ? step : d;
        const bool one = B == 1 || T <= 1 || t.stride(0) == T * step;
        if (!one || (d > 1 && t.stride(-1) != 1) || (n > 1 && ((0 < ld && ld < d) || ld > (1 << 23)))) {
            keep = t.contiguous();
            ld = d;
        }
    }
    void* p() const { return keep.data_ptr(); }
};

// Raw buffers carry no tangent: a dual tensor would give an output whose derivative is silently zero.
template <typename... Ts> void no_tangent(const char* what, const Ts&... tensors) {
    auto has = [](const Tensor& t) { return t.defined() && t._fw_grad(/* level */ 0).defined(); };
    if ((has(tensors) || ...)) throw std::invalid_argument(std::string(what) + " has no forward-mode derivative");
}

void once(const char* what, const variable_list& grads) {  // create_graph=True: the backward pass itself is not recorded
    if (at::GradMode::is_enabled()) throw std::runtime_error(std::string(what) + ": the gradient is not differentiable again");
    for (const Tensor& g : grads) no_tangent(what, g);
}

// -------------------------------------------------------------------------------------------------------------- embed

Tensor embed_forward(const Tensor& weight, const Tensor& ids, double scale) {
    const int64_t V = weight.size(0);
    const int32_t D = size32("embed: elements of a row", weight.size(1));
    at::DimVector shape(ids.sizes());
    shape.push_back(D);
    Tensor out = at::empty(shape, at::TensorOptions(weight.scalar_type()).device(weight.device()));
    enqueue("dvae_embed_fwd", weight.device(), p_dvae_embed_fwd, weight.data_ptr(), V > 1 ? weight.stride(0) : (int64_t)D, ids.data_ptr(), wide(ids),
            out.data_ptr(), ids.numel(), V, D, (float)scale, code(weight));
    return out;
}

struct Embed : torch::autograd::Function<Embed> {
    static Tensor forward(AutogradContext* ctx, const Tensor& weight, const Tensor& ids, double scale) {
        ctx->save_for_backward({ids});
        ctx->saved_data["rows"] = weight.size(0);
        ctx->saved_data["scale"] = scale;
        return embed_forward(weight, ids, scale);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once("embed", grads);
        const Tensor ids = ctx->get_saved_variables()[0];
        const int64_t n = ids.numel(), V = ctx->saved_data["rows"].toInt();
        const int32_t D = (int32_t)grads[0].size(-1);  // (as the forward pass had it)
        const Rows dout(grads[0].dim() == 2 ? grads[0] : grads[0].reshape({n, D}));
        const at::Device dev = grads[0].device();
        Tensor dw = at::empty({V, D}, at::TensorOptions(grads[0].scalar_type()).device(dev));
        Tensor ws = workspace("dvae_embed_bwd_ws_bytes", call(p_dvae_embed_bwd_ws_bytes, n, V, D), dev);
        enqueue("dvae_embed_bwd", dev, p_dvae_embed_bwd, dout.p(), dout.ld, ids.data_ptr(), wide(ids), dw.data_ptr(), ws.data_ptr(), n, V, D,
                (float)ctx->saved_data["scale"].toDouble(), code(dw));
        return {dw, Tensor(), Tensor()};
    }
};

Tensor embed(const Tensor& weight, const Tensor& ids, double scale) {
    no_tangent("embed", weight);
    const Tensor w = weight.resolve_neg();
    if (w.requires_grad() && at::GradMode::is_enabled()) return Embed::apply(w, ids, scale);
    return embed_forward(w, ids, scale);
}

// --------------------------------------------------------------------------------------------------------- recurrence

// h, last and, if `keep`, the states that the backward pass reads
std::tuple<Tensor, Tensor, Tensor> scan_forward(const Tensor& gate, const Tensor& x, const Maybe& offsets, const Maybe& h0, int64_t seqs, bool keep) {
    const int32_t D = size32("gated_scan: channels", x.size(-1));
    const Rows g(gate), y(x);
    const at::Device dev = x.device();
    const at::TensorOptions f32 = at::TensorOptions(at::kFloat).device(dev);
    Tensor h = at::empty(x.sizes(), at::TensorOptions(x.scalar_type()).device(dev)), last = at::empty({seqs, D}, f32), states;
    if (keep) {
        const int64_t floats = call(p_dvae_scan_state_floats, g.n, D);
        if (floats < 0) fail("dvae_scan_state_floats", floats);
        states = at::empty({floats}, f32);
    }
    Tensor ws = workspace("dvae_scan_ws_bytes", call(p_dvae_scan_ws_bytes, g.n, D), dev);
    enqueue("dvae_scan_fwd", dev, p_dvae_scan_fwd, g.p(), g.ld, y.p(), y.ld, ptr(offsets), wide(offsets), (const float*)ptr(h0), h.data_ptr(),
            (float*)last.data_ptr(), keep ? (float*)states.data_ptr() : nullptr, ws.data_ptr(), g.n, seqs, D, code(x));
    return {h, last, states};
}

struct Scan : torch::autograd::Function<Scan> {
    static variable_list forward(AutogradContext* ctx, const Tensor& gate, const Tensor& x, const Maybe& offsets, const Maybe& h0, int64_t seqs) {
        auto [h, last, states] = scan_forward(gate, x, offsets, h0, seqs, true);
        ctx->save_for_backward({gate, x, offsets.value_or(Tensor()), h0.value_or(Tensor()), states});
        ctx->saved_data["seqs"] = seqs;
        ctx->set_materialize_grads(false);
        return {h, last};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once("gated_scan", grads);
        const variable_list saved = ctx->get_saved_variables();
        auto maybe = [](const Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); };
        const Tensor &gate = saved[0], &x = saved[1], &states = saved[4];
        const Maybe offsets = maybe(saved[2]), h0 = maybe(saved[3]);
        const int64_t seqs = ctx->saved_data["seqs"].toInt();
        const int32_t D = (int32_t)x.size(-1);  // (as the forward pass had it)
        const Rows g(gate), y(x);
        const at::Device dev = x.device();
        std::optional<Rows> dh;
        if (grads[0].defined()) dh.emplace(grads[0]);
        const Maybe dlast = grads[1].defined() ? Maybe(grads[1].resolve_neg().contiguous()) : Maybe();
        const at::TensorOptions like = at::TensorOptions(x.scalar_type()).device(dev);
        Tensor dgate = at::empty(gate.sizes(), like), dx = at::empty(x.sizes(), like), dh0;
        // (the edges are those of the tensors that were given: gate, x, offsets if any, h0)
        if (h0 && ctx->needs_input_grad(offsets ? 3 : 2)) dh0 = at::empty({seqs, D}, like.dtype(at::kFloat));
        Tensor ws = workspace("dvae_scan_ws_bytes", call(p_dvae_scan_ws_bytes, g.n, D), dev);
        enqueue("dvae_scan_bwd", dev, p_dvae_scan_bwd, g.p(), g.ld, y.p(), y.ld, ptr(offsets), wide(offsets), (const float*)ptr(h0),
                (const float*)states.data_ptr(), dh ? dh->p() : nullptr, dh ? dh->ld : (int64_t)0, (const float*)ptr(dlast), dgate.data_ptr(),
                dx.data_ptr(), dh0.defined() ? (float*)dh0.data_ptr() : nullptr, ws.data_ptr(), g.n, seqs, D, code(x));
        return {dgate, dx, Tensor(), dh0, Tensor()};
    }
};

std::tuple<Tensor, Tensor> scan(const Tensor& gate, const Tensor& x, const Maybe& offsets, const Maybe& first, int64_t seqs) {
    no_tangent("gated_scan", gate, x, first.value_or(Tensor()));
    const Maybe h0 = first ? Maybe(first->resolve_neg()) : first;
    if (at::GradMode::is_enabled() && (gate.requires_grad() || x.requires_grad() || (h0 && h0->requires_grad()))) {
        variable_list out = Scan::apply(gate, x, offsets, h0, seqs);
        return {out[0], out[1]};
    }
    auto [h, last, states] = scan_forward(gate, x, offsets, h0, seqs, false);
    return {h, last};
}

// whether two matrices may share memory: by the addresses between their first and last elements, and columns beside each other
// in rows of one stride are told apart
bool may_overlap(const Tensor& a, const Tensor& b) {
    auto span = [](const Tensor& t) {
        int64_t last = 0;
        for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
        const char* from = (const char*)t.data_ptr();
        return std::make_pair(from, from + (last + 1) * t.element_size());
    };
    if (a.numel() == 0 || b.numel() == 0) return false;
    const auto [a0, a1] = span(a);
    const auto [b0, b1] = span(b);
    if (a0 >= b1 || b0 >= a1) return false;
    const int64_t ld = a.stride(0) * a.element_size();
    if (ld <= 0 || a.element_size() != b.element_size() || a.stride(0) != b.stride(0) || (a.size(1) > 1 && a.stride(1) != 1) ||
        (b.size(1) > 1 && b.stride(1) != 1))
        return true;
    const int64_t apart = ((b0 - a0) % ld + ld) % ld;  // where a row of b begins in a's rows
    return apart < a.size(1) * a.element_size() || apart + b.size(1) * b.element_size() > ld;
}

Tensor step(const Tensor& gate, const Tensor& x, const Tensor& state, const Maybe& slots) {
    no_tangent("gated_step", gate, x, state);
    const int32_t B = size32("gated_step: rows", x.size(0)), D = size32("gated_step: channels", x.size(1));
    // rows that lie in the pool itself are read before any state is written
    const Rows g(may_overlap(gate, state) ? gate.clone() : gate), y(may_overlap(x, state) ? x.clone() : x);
    const int64_t P = state.size(0);
    Tensor h = at::empty(x.sizes(), at::TensorOptions(x.scalar_type()).device(x.device()));
    enqueue("dvae_scan_step", x.device(), p_dvae_scan_step, g.p(), g.ld, y.p(), y.ld, (float*)state.data_ptr(), P > 1 ? state.stride(0) : (int64_t)D, P,
            ptr(slots), wide(slots), h.data_ptr(), B, D, code(x));
    if (!state.is_inference()) torch::autograd::impl::bump_version(state);  // as by an in-place operation
    return h;
}

// ------------------------------------------------------------------------------------- what the checks would let pass as it is

// The usual call, whose arguments sequence.py would find in order and change nothing of, is recognised here; nothing (None) is
// returned for any other, which sequence.py then checks one by one: it refuses it, or brings it in order first.
const Tensor* tensor(py::handle h) { return THPVariable_Check(h.ptr()) ? &THPVariable_Unpack(h.ptr()) : nullptr; }
bool matrix(const Tensor* t, int64_t dims) {
    return t && t->dim() == dims && t->is_cuda() &&
           (t->scalar_type() == at::kFloat || t->scalar_type() == at::kBFloat16 || t->scalar_type() == at::kHalf);
}
bool alike(const Tensor& a, const Tensor& b) { return a.scalar_type() == b.scalar_type() && a.device() == b.device() && a.sizes() == b.sizes(); }
bool index(const Tensor* t, at::Device device) {
    return t && (t->scalar_type() == at::kInt || t->scalar_type() == at::kLong) && t->device() == device && t->is_contiguous() && !t->is_neg();
}
bool rows_side_by_side(const Tensor& t) { return (t.size(1) == 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1)); }

py::object usual_embed(py::handle weight, py::handle ids, double scale) {
    const Tensor *w = tensor(weight), *t = tensor(ids);
    if (!matrix(w, 2) || w->numel() == 0 || !rows_side_by_side(*w) || !index(t, w->device())) return py::none();
    Tensor out;
    {
        py::gil_scoped_release without_gil;
        out = embed(*w, *t, scale);
    }
    return py::cast(out);
}

py::object usual_scan(py::handle gate, py::handle x, py::handle offsets, py::handle h0) {
    const Tensor *g = tensor(gate), *y = tensor(x);
    Maybe off, first;
    const int64_t dims = offsets.is_none() ? 3 : 2;
    if (!matrix(g, dims) || !matrix(y, dims) || !alike(*g, *y) || y->size(-1) == 0) return py::none();
    if (dims == 2) {
        const Tensor* o = tensor(offsets);
        if (!index(o, y->device()) || o->dim() != 1 || o->numel() < 1) return py::none();
        off = *o;
    }
    const int64_t seqs = dims == 2 ? off->numel() - 1 : y->size(0);
    if (!h0.is_none()) {
        const Tensor* h = tensor(h0);
        if (!h || h->scalar_type() != at::kFloat || h->device() != y->device() || h->dim() != 2 || h->size(0) != seqs ||
            h->size(1) != y->size(-1) || !h->is_contiguous())
            return py::none();
        first = *h;
    }
    std::tuple<Tensor, Tensor> out;
    {
        py::gil_scoped_release without_gil;
        out = scan(*g, *y, off, first, seqs);
    }
    return py::cast(out);
}

py::object usual_step(py::handle gate, py::handle x, py::handle state, py::handle slots) {
    const Tensor *g = tensor(gate), *y = tensor(x), *s = tensor(state);
    Maybe which;
    if (!matrix(g, 2) || !matrix(y, 2) || !alike(*g, *y) || y->size(1) == 0 || !s || s->dim() != 2 || s->scalar_type() != at::kFloat ||
        s->device() != y->device() || s->size(1) != y->size(1) || !rows_side_by_side(*s) || s->is_neg())
        return py::none();
    if (at::GradMode::is_enabled() && (g->requires_grad() || y->requires_grad() || s->requires_grad())) return py::none();
    if (slots.is_none()) {
        if (y->size(0) > s->size(0)) return py::none();
    } else {
        const Tensor* i = tensor(slots);
        if (!index(i, y->device()) || i->dim() != 1 || i->size(0) != y->size(0)) return py::none();
        which = *i;
    }
    Tensor out;
    {
        py::gil_scoped_release without_gil;
        out = step(*g, *y, *s, which);
    }
    return py::cast(out);
}

}  // namespace

PYBIND11_MODULE(_dvae_sequence, m) {
    static PyObject* error = nullptr;
    m.def("bind", [](const std::map<std::string, size_t>& addresses, py::object cls) {
        bind(addresses);
        error = cls.release().ptr();
    });
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const DvaeError& e) {
            PyErr_SetString(error ? error : PyExc_RuntimeError, e.what());
        }
    });
#define F(name) #name,
    m.attr("functions") = std::vector<std::string>{DVAE_FUNCTIONS(F)};
#undef F
    m.def("embed", &embed, py::call_guard<py::gil_scoped_release>());
    m.def("scan", &scan, py::call_guard<py::gil_scoped_release>());
    m.def("step", &step, py::call_guard<py::gil_scoped_release>());
    m.def("usual_embed", &usual_embed);
    m.def("usual_scan", &usual_scan);
    m.def("usual_step", &usual_step);
}
