// The operator's host path on PyTorch tensors: stage calls, autograd nodes and the argument fast path.
//
// Why native: with Python autograd functions around ctypes calls, a second-order step over a small layer
// (forward, first gradients kept in the graph, second gradients; five kernels) cost 390 us of host time
// whatever its size, on a GPU that needs a fraction of that; the nodes below run without the interpreter.
//
// PyTorch supplies device memory, streams and the autograd engine; all arithmetic is in libbob_sm100.so,
// whose entry points flashbob_b200/_native.py hands over as addresses (one library per process, wherever
// it was loaded from).  The autograd protocol is the reference's (reference: src/bob/sdpa.py:239-368):
//   * SdpaNode::apply runs only the first backward when grad mode is off, otherwise it also records a
//     SecondOrderNode over (q, k, v, dO), whose apply is the second backward;
//   * undefined incoming gradients stay undefined and switch off the products they would feed.
#include "../../include/bob_sm100.h"

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <array>
#include <cmath>
#include <cstring>
#include <optional>

namespace {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

// ---- the library ------------------------------------------------------------------------------------
struct Library {
    decltype(&bob_sm100_fwd) fwd = nullptr;
    decltype(&bob_sm100_bwd1) bwd1 = nullptr;
    decltype(&bob_sm100_bwd2) bwd2 = nullptr;
    decltype(&bob_sm100_workspace_bytes) workspace_bytes = nullptr;
    decltype(&bob_sm100_read_status) read_status = nullptr;
    decltype(&bob_sm100_last_status) last_status = nullptr;
    decltype(&bob_sm100_error_string) error_string = nullptr;
    decltype(&bob_sm100_rotate) rotate = nullptr;
    decltype(&bob_sm100_cache_append) cache_append = nullptr;
    decltype(&bob_sm100_cache_read) cache_read = nullptr;
    decltype(&bob_sm100_paged_workspace_bytes) paged_workspace_bytes = nullptr;
    decltype(&bob_sm100_paged_fwd) paged_fwd = nullptr;
};
Library lib;
PyObject* error_class = nullptr;           // BobSm100Error

[[noreturn]] void fail(const std::string& what, int rc) {
    // the Python exception class is kept, also from the autograd engine's threads
    pybind11::gil_scoped_acquire gil;
    PyErr_SetString(error_class, (what + " failed with code " + std::to_string(rc) + ": " + lib.error_string(rc)).c_str());
    python_error e;
    e.persist();
    throw e;
}

struct Mask {
    bool causal = false;
    int window = 0;
    int64_t q_offset = 0, k_offset = 0;
    std::optional<double> scale;           // none: 1 / sqrt(D)
    bool check_status = false;             // wait for the stream after each stage and read its status word
};

// In-place addressing needs unit stride along the head dim, batch / head / row strides that are positive
// multiples of 8 elements (16 bytes) and a 16-byte aligned base; anything else is made contiguous.
Tensor tma_ready(const Tensor& t) {
    bool ok = t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0;
    for (int i = 0; i < 3; ++i) ok = ok && t.stride(i) % 8 == 0 && (t.stride(i) > 0 || t.size(i) == 1);
    return ok ? t : t.contiguous();
}

void set_strides(int64_t (&field)[3], const Tensor& t) {
    for (int i = 0; i < 3; ++i) field[i] = t.stride(i);
}

bob_sm100_geom geometry(const Tensor& q, const Tensor& k, const Mask& m) {
    bob_sm100_geom g = {};
    g.B = static_cast<int32_t>(q.size(0)); g.Hq = static_cast<int32_t>(q.size(1)); g.Hkv = static_cast<int32_t>(k.size(1));
    g.Nq = static_cast<int32_t>(q.size(2)); g.Nk = static_cast<int32_t>(k.size(2)); g.D = static_cast<int32_t>(q.size(3));
    g.dtype = q.scalar_type() == at::kBFloat16 ? BOB_SM100_BF16 : BOB_SM100_FP16;
    g.is_causal = m.causal;
    g.window = m.window;
    g.device = q.device().index();
    g.flags = BOB_SM100_SPLIT_KEYS;        // (every workspace below is sized for its own call)
    g.q_offset = m.q_offset;
    g.k_offset = m.k_offset;
    g.scale = static_cast<float>(m.scale ? *m.scale : 1.0 / std::sqrt(static_cast<double>(g.D)));
    return g;
}

Tensor empty(at::IntArrayRef size, at::ScalarType type, const Tensor& like) {
    return at::detail::empty_cuda(size, type, like.device(), std::nullopt);
}
Tensor workspace(int stage, const bob_sm100_geom& g, const Tensor& like) {
    return empty({static_cast<int64_t>(lib.workspace_bytes(stage, &g))}, at::kByte, like);
}
void* ptr(const Tensor& t) { return t.defined() ? const_cast<void*>(t.const_data_ptr()) : nullptr; }
float* fptr(const Tensor& t) { return static_cast<float*>(ptr(t)); }
void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// Raises if a kernel on this device gave up on a bounded wait: by default a non-blocking look at the
// device's host-visible status word (a time-out of an earlier call surfaces here), with `check_status` the
// call's own status word after waiting for the stream.
void finish(int rc, const char* what, const Mask& m, const Tensor& ws) {
    if (rc) fail(what, rc);
    if (m.check_status && (rc = lib.read_status(ptr(ws), stream_of(ws)))) fail(std::string(what) + " (device status)", rc);
    if ((rc = lib.last_status(ws.device().index())))
        fail("an earlier libbob_sm100 kernel on cuda:" + std::to_string(ws.device().index()) + " (seen after " + what +
             "; its results are undefined)", rc);
}

// ---- the three stages -------------------------------------------------------------------------------
struct Forward { Tensor out, lse; };
Forward run_forward(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Mask& m) {
    const Tensor q = tma_ready(q_), k = tma_ready(k_), v = tma_ready(v_);
    bob_sm100_geom g = geometry(q, k, m);
    set_strides(g.q_strides, q); set_strides(g.k_strides, k); set_strides(g.v_strides, v);
    Forward r{empty(q.sizes(), q.scalar_type(), q), empty(q.sizes().slice(0, 3), at::kFloat, q)};
    const Tensor ws = workspace(BOB_SM100_STAGE_FWD, g, q);
    const int rc = lib.fwd(&g, ptr(q), ptr(k), ptr(v), ptr(r.out), fptr(r.lse), ptr(ws), stream_of(q));
    finish(rc, "bob_sm100_fwd", m, ws);
    return r;
}

struct First { Tensor dQ, dK, dV, delta, pk; };
First run_first(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& out_, const Tensor& lse_,
                const Tensor& dO_, const Mask& m, bool for_second_order) {
    const Tensor q = tma_ready(q_), k = tma_ready(k_), v = tma_ready(v_), out = tma_ready(out_), dO = tma_ready(dO_);
    const Tensor lse = lse_.contiguous();
    bob_sm100_geom g = geometry(q, k, m);
    set_strides(g.q_strides, q); set_strides(g.k_strides, k); set_strides(g.v_strides, v);
    set_strides(g.out_strides, out); set_strides(g.do_strides, dO);
    First r{empty(q.sizes(), q.scalar_type(), q), empty(k.sizes(), q.scalar_type(), q), empty(k.sizes(), q.scalar_type(), q),
            empty(q.sizes().slice(0, 3), at::kFloat, q), for_second_order ? empty(q.sizes(), at::kFloat, q) : Tensor()};
    const Tensor ws = workspace(BOB_SM100_STAGE_BWD1, g, q);
    const int rc = lib.bwd1(&g, ptr(q), ptr(k), ptr(v), ptr(out), fptr(lse), ptr(dO), ptr(r.dQ), ptr(r.dK), ptr(r.dV),
                            fptr(r.delta), fptr(r.pk), ptr(ws), stream_of(q));
    finish(rc, "bob_sm100_bwd1", m, ws);
    return r;
}

struct Second { Tensor Qbar, Kbar, Vbar, dObar; };
Second run_second(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& out_, const Tensor& lse_,
                  const Tensor& delta_, const Tensor& pk_, const Tensor& dO_, const Tensor& dQ_, const Tensor& uQ_,
                  const Tensor& uK_, const Tensor& uV_, const Mask& m) {
    const Tensor q = tma_ready(q_), k = tma_ready(k_), v = tma_ready(v_), out = tma_ready(out_), dO = tma_ready(dO_), dQ = tma_ready(dQ_);
    auto tangent = [&](const Tensor& t) { return t.defined() ? tma_ready(t.scalar_type() == q.scalar_type() ? t : t.to(q.scalar_type())) : t; };
    const Tensor uQ = tangent(uQ_), uK = tangent(uK_), uV = tangent(uV_);
    const Tensor lse = lse_.contiguous(), delta = delta_.contiguous(), pk = pk_.contiguous();
    bob_sm100_geom g = geometry(q, k, m);
    set_strides(g.q_strides, q); set_strides(g.k_strides, k); set_strides(g.v_strides, v);
    set_strides(g.out_strides, out); set_strides(g.do_strides, dO); set_strides(g.dq_strides, dQ);
    if (uQ.defined()) set_strides(g.uq_strides, uQ);
    if (uK.defined()) set_strides(g.uk_strides, uK);
    if (uV.defined()) set_strides(g.uv_strides, uV);
    Second r{empty(q.sizes(), q.scalar_type(), q), empty(k.sizes(), q.scalar_type(), q), empty(k.sizes(), q.scalar_type(), q),
             empty(q.sizes(), q.scalar_type(), q)};
    const Tensor ws = workspace(BOB_SM100_STAGE_BWD2, g, q);
    const int rc = lib.bwd2(&g, ptr(q), ptr(k), ptr(v), ptr(out), fptr(lse), fptr(delta), fptr(pk), ptr(dO), ptr(dQ), ptr(uQ),
                            ptr(uK), ptr(uV), ptr(r.Qbar), ptr(r.Kbar), ptr(r.Vbar), ptr(r.dObar), ptr(ws), stream_of(q));
    finish(rc, "bob_sm100_bwd2", m, ws);
    return r;
}

// ---- autograd nodes ---------------------------------------------------------------------------------
// The nodes call the library below PyTorch's dispatcher; copies of awkwardly strided inputs must not be
// recorded on the tape either.
struct Untracked {
    at::AutoGradMode grad_off{false};
    at::AutoDispatchBelowADInplaceOrView below;
};

// deleteNode frees a graph node by node; a plain destructor would free a node's predecessors inside its own, one
// stack frame deeper for each of a chain of calls.
template <class N> std::shared_ptr<N> make_node() { return std::shared_ptr<N>(new N(), torch::autograd::deleteNode); }

// First backward as a differentiable function of (q, k, v, dO): its gradient is the second backward.
struct SecondOrderNode : Node {
    Mask mask;
    SavedVariable q, k, v, dO, out, lse, dQ, delta, pk;
    std::string name() const override { return "BoBSecondOrderBackward"; }
    variable_list apply(variable_list&& u) override {
        std::lock_guard<std::mutex> lock(mutex_);
        if (!u[0].defined() && !u[1].defined() && !u[2].defined()) return variable_list(4);
        const Tensor q_ = q.unpack(), k_ = k.unpack(), v_ = v.unpack(), dO_ = dO.unpack(), out_ = out.unpack(), lse_ = lse.unpack(),
                     dQ_ = dQ.unpack(shared_from_this()), delta_ = delta.unpack(), pk_ = pk.unpack();
        Untracked untracked;
        const c10::cuda::CUDAGuard device(q_.device());
        Second r = run_second(q_, k_, v_, out_, lse_, delta_, pk_, dO_, dQ_, u[0], u[1], u[2], mask);
        return {r.Qbar, r.Kbar, r.Vbar, r.dObar};
    }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        for (SavedVariable* s : {&q, &k, &v, &dO, &out, &lse, &dQ, &delta, &pk}) s->reset_data();
    }
};

// Attention forward whose gradient is itself differentiable once more.
struct SdpaNode : Node {
    Mask mask;
    SavedVariable q, k, v, out, lse;
    std::string name() const override { return "SDPAWithBoBBackward"; }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        const Tensor& dO = grads[0];
        if (!dO.defined()) return variable_list(3);
        const Tensor q_ = q.unpack(), k_ = k.unpack(), v_ = v.unpack(), out_ = out.unpack(shared_from_this()), lse_ = lse.unpack();
        const bool record = torch::autograd::compute_requires_grad(q_, k_, v_, dO);
        // a graph that is kept would hold a derivative from which the tangent's term is missing
        TORCH_CHECK_NOT_IMPLEMENTED(!record || !dO._fw_grad(0).defined(), "forward-mode AD is unsupported; differentiate with "
                                    "reverse mode (torch.autograd.grad twice) instead");
        First r;
        {
            Untracked untracked;
            const c10::cuda::CUDAGuard device(q_.device());
            r = run_first(q_, k_, v_, out_, lse_, dO, mask, record);
        }
        if (record) {
            auto node = make_node<SecondOrderNode>();
            node->set_next_edges(torch::autograd::collect_next_edges(q_, k_, v_, dO));
            node->mask = mask;
            node->q = SavedVariable(q_, false); node->k = SavedVariable(k_, false); node->v = SavedVariable(v_, false);
            node->dO = SavedVariable(dO, false); node->out = SavedVariable(out_.detach(), false); node->lse = SavedVariable(lse_, false);
            node->delta = SavedVariable(r.delta, false); node->pk = SavedVariable(r.pk, false);
            for (const Tensor& t : {r.dQ, r.dK, r.dV}) torch::autograd::set_history(t, node);
            node->dQ = SavedVariable(r.dQ, true);
        }
        return {r.dQ, r.dK, r.dV};
    }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        for (SavedVariable* s : {&q, &k, &v, &out, &lse}) s->reset_data();
    }
};

Tensor sdpa(const Tensor& q, const Tensor& k, const Tensor& v, const Mask& m) {
    const bool record = torch::autograd::compute_requires_grad(q, k, v);
    Forward r;
    {
        Untracked untracked;
        const c10::cuda::CUDAGuard device(q.device());
        r = run_forward(q, k, v, m);
    }
    if (record) {
        auto node = make_node<SdpaNode>();
        node->set_next_edges(torch::autograd::collect_next_edges(q, k, v));
        node->mask = m;
        node->q = SavedVariable(q, false); node->k = SavedVariable(k, false); node->v = SavedVariable(v, false);
        node->lse = SavedVariable(r.lse, false);
        torch::autograd::set_history(r.out, node);
        node->out = SavedVariable(r.out, true);
    }
    return r.out;
}

// ---- rotary positions -------------------------------------------------------------------------------
// The kernels for positions and the paged cache read any layout with unit stride along the head dim, strides that are
// multiples of 8 elements (zero for an expanded tensor) and a 16-byte aligned base.  Anything else is copied: contiguous()
// would give back a tensor that is contiguous but starts elsewhere, or has an odd stride along a dimension of one entry.
Tensor tokens_ready(const Tensor& t) {
    bool ok = t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0;
    for (int i = 0; i < 3; ++i) ok = ok && t.stride(i) % 8 == 0 && t.stride(i) >= 0;
    return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

int32_t dtype_of(const Tensor& t) { return t.scalar_type() == at::kBFloat16 ? BOB_SM100_BF16 : BOB_SM100_FP16; }

// As finish(), for calls whose kernels report to the device's word only.
void finish_reported(int rc, const char* what, int device, bool check_status) {
    if (rc) fail(what, rc);
    if (check_status) c10::cuda::getCurrentCUDAStream(device).synchronize();
    if ((rc = lib.last_status(device))) {
        // a call's kernels, and their threads, report one after another: what is still to come is part of this error
        if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) {
            c10::cuda::getCurrentCUDAStream(device).synchronize();
            lib.last_status(device);
        }
        fail((check_status ? std::string(what) + " (device status)" : "an earlier libbob_sm100 kernel on cuda:" + std::to_string(device) +
              " (seen after " + what + "; its results are undefined)"), rc);
    }
}

struct Rotation {
    bob_sm100_rotary rotary = {};
    int64_t first = 0;
    bool inverse = false, check_status = false;
};

// x[0] and x[1] [B, H, N, D], of which one may be undefined, turned to their positions (undefined: first + row).
std::array<Tensor, 2> run_rotate(const std::array<Tensor, 2>& x, const Tensor& positions, const Rotation& r) {
    bob_sm100_rotate_args a = {};
    std::array<Tensor, 2> in, out;
    int n = 0, device = 0;
    for (int i = 0; i < 2; ++i) {
        if (!x[i].defined()) continue;
        in[i] = tokens_ready(x[i]);
        out[i] = empty(in[i].sizes(), in[i].scalar_type(), in[i]);
        a.B = static_cast<int32_t>(in[i].size(0)); a.N = static_cast<int32_t>(in[i].size(2)); a.D = static_cast<int32_t>(in[i].size(3));
        a.dtype = dtype_of(in[i]);
        a.device = device = in[i].device().index();
        a.heads[n] = static_cast<int32_t>(in[i].size(1));
        a.in[n] = ptr(in[i]);
        a.out[n] = ptr(out[i]);
        set_strides(a.in_strides[n++], in[i]);
    }
    if (positions.defined()) {                   // [N] or [B, N]
        a.positions = ptr(positions);
        a.position_bits = positions.scalar_type() == at::kLong ? 64 : 32;
        a.position_strides[0] = positions.dim() == 2 && positions.size(0) > 1 ? positions.stride(0) : 0;
        a.position_strides[1] = positions.stride(-1);
    }
    a.first = r.first;
    a.inverse = r.inverse;
    a.rotary = r.rotary;
    const int rc = lib.rotate(&a, c10::cuda::getCurrentCUDAStream(device).stream());
    finish_reported(rc, "bob_sm100_rotate", device, r.check_status);
    return out;
}

std::array<Tensor, 2> rotate(const std::array<Tensor, 2>& x, const Tensor& positions, const Rotation& r);

// The gradient of a rotation is the rotation back, recorded like any other: differentiable any number of times.
struct RotateNode : Node {
    Rotation rotation;
    SavedVariable positions;
    bool has[2] = {false, false};
    std::string name() const override { return "RotaryBackward"; }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        std::array<Tensor, 2> u;
        for (int i = 0, n = 0; i < 2; ++i)
            if (has[i]) u[i] = grads[n++];
        if (!u[0].defined() && !u[1].defined()) return variable_list(2);
        for (const Tensor& t : u)
            TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(), "forward-mode AD is unsupported; differentiate with "
                                        "reverse mode (torch.autograd.grad twice) instead");
        Rotation back = rotation;
        back.inverse = !back.inverse;
        std::array<Tensor, 2> g = rotate(u, positions.unpack(), back);
        return {g[0], g[1]};
    }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        positions.reset_data();
    }
};

std::array<Tensor, 2> rotate(const std::array<Tensor, 2>& x, const Tensor& positions, const Rotation& r) {
    std::array<Tensor, 2> y;
    {
        Untracked untracked;
        const c10::cuda::CUDAGuard device((x[0].defined() ? x[0] : x[1]).device());
        y = run_rotate(x, positions, r);
    }
    if (torch::autograd::compute_requires_grad(x[0], x[1])) {
        auto node = make_node<RotateNode>();
        node->set_next_edges(torch::autograd::collect_next_edges(x[0], x[1]));
        node->rotation = r;
        node->positions = SavedVariable(positions, false);
        for (int i = 0; i < 2; ++i) {
            node->has[i] = y[i].defined();
            if (y[i].defined()) torch::autograd::set_history(y[i], node);
        }
    }
    return y;
}

// ---- paged cache ------------------------------------------------------------------------------------
struct Cache {
    Tensor data[2], scales[2];
    bob_sm100_cache c = {};
};
struct Sequences {
    Tensor table, lengths, counts;
    bob_sm100_sequences s = {};
};

void run_append(const Tensor& k_, const Tensor& v_, Cache& cache, const Sequences& seq, const bob_sm100_rotary& rotary, bool check_status) {
    const Tensor k = tokens_ready(k_), v = tokens_ready(v_);
    int64_t ks[3], vs[3];
    set_strides(ks, k);
    set_strides(vs, v);
    const int rc = lib.cache_append(&cache.c, &seq.s, &rotary, static_cast<int>(k.size(2)), ptr(k), ks, ptr(v), vs, stream_of(k));
    for (const Tensor& t : {cache.data[0], cache.data[1], cache.scales[0], cache.scales[1]})
        if (t.defined() && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();      // what autograd has saved of them is stale
    finish_reported(rc, "bob_sm100_cache_append", cache.c.device, check_status);
}

std::array<Tensor, 2> run_read(const Cache& cache, const Sequences& seq, int64_t n, at::ScalarType type, bool check_status) {
    const std::array<int64_t, 4> size{seq.s.B, cache.c.heads, n, cache.c.D};
    std::array<Tensor, 2> out{empty(size, type, cache.data[0]), empty(size, type, cache.data[0])};
    const int rc = lib.cache_read(&cache.c, &seq.s, static_cast<int>(n), ptr(out[0]), ptr(out[1]), stream_of(out[0]));
    finish_reported(rc, "bob_sm100_cache_read", cache.c.device, check_status);
    return out;
}

Tensor run_paged(const Tensor& q_, const Cache& cache, const Sequences& seq, const bob_sm100_rotary& rotary, bool causal, int64_t window,
                 std::optional<double> scale, bool check_status) {
    const Tensor q = tokens_ready(q_);
    const Tensor out = empty(q.sizes(), q.scalar_type(), q);
    bob_sm100_paged_args a = {};
    a.cache = cache.c;
    a.seq = seq.s;
    a.rotary = rotary;
    a.Hq = static_cast<int32_t>(q.size(1)); a.N = static_cast<int32_t>(q.size(2));
    a.is_causal = causal;
    a.window = static_cast<int32_t>(window);
    a.q = ptr(q);
    set_strides(a.q_strides, q);
    a.out = ptr(out);
    a.scale = static_cast<float>(scale ? *scale : 1.0 / std::sqrt(static_cast<double>(q.size(3))));
    const Tensor ws = empty({static_cast<int64_t>(lib.paged_workspace_bytes(&a))}, at::kByte, q);
    const int rc = lib.paged_fwd(&a, ptr(ws), stream_of(q));
    finish_reported(rc, "bob_sm100_paged_fwd", cache.c.device, check_status);
    return out;
}

// ---- Python entry points ----------------------------------------------------------------------------
bool is_int(PyObject* o) { return PyLong_CheckExact(o); }       // a bool is a subclass: not exact

// The argument checks of sdpa_bob in their common, valid form.  Anything else - a CPU tensor, an int-like
// that is no int, a grouped call with a window, an invalid shape, a call that torch.jit.trace records - is left
// to the Python side, which raises or resolves it; its checks are the one statement of what is allowed.
bool common_call(const Tensor& q, const Tensor& k, const Tensor& v, PyObject* causal, PyObject* scale, PyObject* window,
                 PyObject* q_offset, PyObject* k_offset, Mask& m) {
    if (torch::jit::tracer::isTracing()) return false;
    const auto type = q.scalar_type();
    if (!q.is_cuda() || q.dim() != 4 || k.dim() != 4 || v.dim() != 4 || (type != at::kHalf && type != at::kBFloat16)) return false;
    if (k.scalar_type() != type || v.scalar_type() != type || k.device() != q.device() || v.device() != q.device()) return false;
    if (k.sizes() != v.sizes() || q.numel() <= 0 || k.numel() <= 0) return false;
    const int64_t n_q = q.size(2), n_k = k.size(2), D = q.size(3), group = q.size(1) / k.size(1);
    if (k.size(0) != q.size(0) || k.size(3) != D || group * k.size(1) != q.size(1) || (D != 32 && D != 64 && D != 128)) return false;
    if (n_q > INT32_MAX || n_k > INT32_MAX || q.size(0) > INT32_MAX || q.size(1) > INT32_MAX) return false;
    for (const Tensor* t : {&q, &k, &v})
        if (t->_fw_grad(0).defined()) return false;
    if (!PyBool_Check(causal) || !is_int(window) || !is_int(k_offset) || !(q_offset == Py_None || is_int(q_offset))) return false;
    m.causal = causal == Py_True;
    auto count = [](PyObject* o, int64_t& x) {
        int overflow = 0;
        x = PyLong_AsLongLongAndOverflow(o, &overflow);
        return !overflow && x >= 0 && x < (int64_t(1) << 40);
    };
    int64_t w = 0;
    if (!count(window, w) || !count(k_offset, m.k_offset)) return false;
    if (w > 0 && !m.causal) return false;
    if (q_offset != Py_None) {
        if (!count(q_offset, m.q_offset)) return false;
    } else {                               // a causal rectangle defaults to right alignment
        m.q_offset = m.k_offset + (m.causal && n_k > n_q ? n_k - n_q : 0);
    }
    const bool rectangular = n_q != n_k || m.q_offset != m.k_offset;
    // a window that already covers every causal key is no window
    if (m.causal && w > 0 && w >= (rectangular ? m.q_offset - m.k_offset + n_q : n_q)) w = 0;
    if (w > INT32_MAX) return false;
    m.window = static_cast<int>(w);
    if (group > 1 && (rectangular || w > 0 || type != at::kBFloat16 || group > 32)) return false;
    if (scale != Py_None) {
        if (!PyFloat_CheckExact(scale)) return false;
        const float s = static_cast<float>(PyFloat_AS_DOUBLE(scale));
        if (!(s > 0) || !std::isfinite(s)) return false;
        m.scale = PyFloat_AS_DOUBLE(scale);
    }
    return true;
}

const Tensor& tensor_arg(PyObject* o) {
    if (!THPVariable_Check(o)) throw torch::TypeError("expected a torch.Tensor");
    return THPVariable_Unpack(o);
}
Tensor optional_tensor_arg(PyObject* o) { return o == Py_None ? Tensor() : tensor_arg(o); }

int64_t int_arg(PyObject* o) {
    const int64_t x = PyLong_AsLongLong(o);
    if (x == -1 && PyErr_Occurred()) throw python_error();
    return x;
}

// (is_causal, window_size, q_offset, k_offset, scale or None, check_status), all checked by the caller
Mask mask_args(PyObject* const* a) {
    Mask m;
    m.causal = PyObject_IsTrue(a[0]);
    m.window = static_cast<int>(int_arg(a[1]));
    m.q_offset = int_arg(a[2]);
    m.k_offset = int_arg(a[3]);
    if (a[4] != Py_None) {
        m.scale = PyFloat_AsDouble(a[4]);
        if (PyErr_Occurred()) throw python_error();
    }
    m.check_status = PyObject_IsTrue(a[5]);
    return m;
}

template <class F> auto without_gil(F f) {
    pybind11::gil_scoped_release released;
    return f();
}

void want(Py_ssize_t got, Py_ssize_t n) {
    if (got != n) throw torch::TypeError("expected " + std::to_string(n) + " arguments, got " + std::to_string(got));
}

PyObject* tuple_of(std::initializer_list<Tensor> ts) {
    PyObject* r = PyTuple_New(static_cast<Py_ssize_t>(ts.size()));
    Py_ssize_t i = 0;
    for (const Tensor& t : ts) PyTuple_SET_ITEM(r, i++, THPVariable_Wrap(t));     // None for an undefined tensor
    return r;
}

// try_sdpa(q, k, v, is_causal, scale, window_size, q_offset, k_offset, check_status) -> out, or None when
// the call is not in the common form
PyObject* py_try_sdpa(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    want(n, 9);
    if (!THPVariable_Check(a[0]) || !THPVariable_Check(a[1]) || !THPVariable_Check(a[2])) Py_RETURN_NONE;
    const Tensor &q = THPVariable_Unpack(a[0]), &k = THPVariable_Unpack(a[1]), &v = THPVariable_Unpack(a[2]);
    Mask m;
    if (!common_call(q, k, v, a[3], a[4], a[5], a[6], a[7], m)) Py_RETURN_NONE;
    m.check_status = PyObject_IsTrue(a[8]);
    return THPVariable_Wrap(without_gil([&] { return sdpa(q, k, v, m); }));
    END_HANDLE_TH_ERRORS
}

// sdpa(q, k, v, <mask>) -> out; arguments checked and resolved by the caller
PyObject* py_sdpa(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    want(n, 9);
    const Tensor &q = tensor_arg(a[0]), &k = tensor_arg(a[1]), &v = tensor_arg(a[2]);
    const Mask m = mask_args(a + 3);
    return THPVariable_Wrap(without_gil([&] { return sdpa(q, k, v, m); }));
    END_HANDLE_TH_ERRORS
}

// forward(q, k, v, <mask>) -> (out, lse)
PyObject* py_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    want(n, 9);
    Untracked untracked;
    const Tensor &q = tensor_arg(a[0]), &k = tensor_arg(a[1]), &v = tensor_arg(a[2]);
    const Mask m = mask_args(a + 3);
    const c10::cuda::CUDAGuard device(q.device());
    Forward r = without_gil([&] { return run_forward(q, k, v, m); });
    return tuple_of({r.out, r.lse});
    END_HANDLE_TH_ERRORS
}

// first_backward(q, k, v, out, lse, dO, <mask>, for_second_order) -> (dQ, dK, dV, delta, pk)
PyObject* py_first(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    want(n, 13);
    Untracked untracked;
    const Tensor &q = tensor_arg(a[0]), &k = tensor_arg(a[1]), &v = tensor_arg(a[2]), &out = tensor_arg(a[3]), &lse = tensor_arg(a[4]),
                 &dO = tensor_arg(a[5]);
    const Mask m = mask_args(a + 6);
    const bool for_second_order = PyObject_IsTrue(a[12]);
    const c10::cuda::CUDAGuard device(q.device());
    First r = without_gil([&] { return run_first(q, k, v, out, lse, dO, m, for_second_order); });
    return tuple_of({r.dQ, r.dK, r.dV, r.delta, r.pk});
    END_HANDLE_TH_ERRORS
}

// second_backward(q, k, v, out, lse, delta, pk, dO, dQ, uQ, uK, uV, <mask>) -> (Qbar, Kbar, Vbar, dObar)
PyObject* py_second(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    want(n, 18);
    Untracked untracked;
    const Tensor &q = tensor_arg(a[0]), &k = tensor_arg(a[1]), &v = tensor_arg(a[2]), &out = tensor_arg(a[3]), &lse = tensor_arg(a[4]),
                 &delta = tensor_arg(a[5]), &pk = tensor_arg(a[6]), &dO = tensor_arg(a[7]), &dQ = tensor_arg(a[8]);
    const Tensor uQ = optional_tensor_arg(a[9]), uK = optional_tensor_arg(a[10]), uV = optional_tensor_arg(a[11]);
    const Mask m = mask_args(a + 12);
    const c10::cuda::CUDAGuard device(q.device());
    Second r = without_gil([&] { return run_second(q, k, v, out, lse, delta, pk, dO, dQ, uQ, uK, uV, m); });
    return tuple_of({r.Qbar, r.Kbar, r.Vbar, r.dObar});
    END_HANDLE_TH_ERRORS
}

// The bytes of a bob_sm100_rotary; None: no rotation.
bob_sm100_rotary rotary_arg(PyObject* o) {
    bob_sm100_rotary r = {};
    if (o == Py_None) return r;
    char* data = nullptr;
    Py_ssize_t size = 0;
    if (PyBytes_AsStringAndSize(o, &data, &size)) throw python_error();
    if (size != static_cast<Py_ssize_t>(sizeof(r))) throw torch::TypeError("a rotation is " + std::to_string(sizeof(r)) + " bytes");
    std::memcpy(&r, data, sizeof(r));
    return r;
}

// (keys, values, key scales or None, value scales or None, 16-bit type of the rows), checked by the caller
Cache cache_args(PyObject* const* a) {
    Cache r;
    bob_sm100_cache& c = r.c;
    for (int i = 0; i < 2; ++i) {
        const Tensor& t = r.data[i] = tensor_arg(a[i]);
        const int64_t size = t.element_size();
        c.data[i] = ptr(t);
        for (int k = 0; k < 3; ++k) c.strides[i][k] = t.stride(k) * size;
        r.scales[i] = optional_tensor_arg(a[2 + i]);
        c.scales[i] = ptr(r.scales[i]);
        if (r.scales[i].defined())
            for (int k = 0; k < 3; ++k) c.scale_strides[i][k] = r.scales[i].stride(k) * 4;
    }
    const Tensor& k = r.data[0];
    c.bits = r.scales[0].defined() ? 4 : 16;
    c.pages = static_cast<int32_t>(k.size(0)); c.heads = static_cast<int32_t>(k.size(1)); c.page_size = static_cast<int32_t>(k.size(2));
    c.D = static_cast<int32_t>(k.size(3)) * (c.bits == 4 ? 2 : 1);
    c.dtype = PyObject_IsTrue(a[4]) ? BOB_SM100_BF16 : BOB_SM100_FP16;
    c.device = k.device().index();
    return r;
}

// (page table, lengths, counts or None), checked by the caller
Sequences sequence_args(PyObject* const* a) {
    Sequences r;
    r.table = tensor_arg(a[0]);
    if (r.table.stride(1) != 1) r.table = r.table.contiguous();
    r.lengths = tensor_arg(a[1]).contiguous();
    r.counts = optional_tensor_arg(a[2]);
    if (r.counts.defined()) r.counts = r.counts.contiguous();
    r.s.B = static_cast<int32_t>(r.table.size(0)); r.s.max_pages = static_cast<int32_t>(r.table.size(1));
    r.s.table = static_cast<const int32_t*>(ptr(r.table));
    r.s.table_stride = r.table.stride(0);
    r.s.lengths = static_cast<const int32_t*>(ptr(r.lengths));
    r.s.counts = static_cast<const int32_t*>(ptr(r.counts));
    return r;
}

// The argument checks of the operations on positions and the paged cache in their common, valid form, as common_call has
// them for the operator: what is not plainly valid is left to the Python side, whose checks say what is allowed.
bool common_heads(const Tensor& t) {
    const auto type = t.scalar_type();
    if (!t.is_cuda() || t.dim() != 4 || (type != at::kHalf && type != at::kBFloat16) || t.numel() <= 0 || t._fw_grad(0).defined()) return false;
    const int64_t D = t.size(3);
    return (D == 32 || D == 64 || D == 128) && t.size(0) <= INT32_MAX && t.size(1) <= INT32_MAX && t.size(2) <= (1 << 28);
}
bool common_rotary(PyObject* packed, PyObject* head_dim, int64_t D) {
    return packed == Py_None || (PyBytes_CheckExact(packed) && is_int(head_dim) && PyLong_AsLongLong(head_dim) == D);
}
bool common_rows(const Tensor& t, const Tensor& cache_k, PyObject* scales, PyObject* bf16) {
    return common_heads(t) && t.device() == cache_k.device() && t.scalar_type() == (bf16 == Py_True ? at::kBFloat16 : at::kHalf) &&
           t.size(3) == cache_k.size(3) * (scales == Py_None ? 1 : 2) && !(t.requires_grad() && at::GradMode::is_enabled());
}
bool common_sequences(PyObject* const* a, const Tensor& cache_k, int64_t B) {
    for (int i = 0; i < 3; ++i) {
        if (i == 2 && a[i] == Py_None) continue;
        if (!THPVariable_Check(a[i])) return false;
        const Tensor& t = THPVariable_Unpack(a[i]);
        if (t.scalar_type() != at::kInt || t.dim() != (i ? 1 : 2) || t.numel() <= 0 || t.device() != cache_k.device() || t.size(0) != B) return false;
    }
    return THPVariable_Unpack(a[0]).size(1) * cache_k.size(2) <= (1 << 28);
}

// try_rotate(q, k or None, rotary, its head_dim, positions or None, offset, check_status) -> (q, k), or None
PyObject* py_try_rotate(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    want(n, 7);
    if (torch::jit::tracer::isTracing()) Py_RETURN_NONE;
    std::array<Tensor, 2> x;
    for (int i = 0; i < 2; ++i) {
        if (i == 1 && a[i] == Py_None) continue;
        if (!THPVariable_Check(a[i])) Py_RETURN_NONE;
        x[i] = THPVariable_Unpack(a[i]);
        if (!common_heads(x[i])) Py_RETURN_NONE;
    }
    const Tensor& q = x[0];
    if (x[1].defined() && (x[1].device() != q.device() || x[1].scalar_type() != q.scalar_type() || x[1].size(0) != q.size(0) ||
                           x[1].size(2) != q.size(2) || x[1].size(3) != q.size(3))) Py_RETURN_NONE;
    if (a[2] == Py_None || !common_rotary(a[2], a[3], q.size(3)) || !is_int(a[5])) Py_RETURN_NONE;
    Rotation r;
    int overflow = 0;
    r.first = PyLong_AsLongLongAndOverflow(a[5], &overflow);
    if (overflow || r.first < 0 || r.first >= (int64_t(1) << 62)) Py_RETURN_NONE;
    Tensor positions;
    if (a[4] != Py_None) {
        if (!THPVariable_Check(a[4]) || r.first) Py_RETURN_NONE;
        positions = THPVariable_Unpack(a[4]);
        const auto type = positions.scalar_type();
        const int64_t dim = positions.dim();
        if ((type != at::kLong && type != at::kInt) || positions.device() != q.device() || dim < 1 || dim > 2 || positions.size(-1) != q.size(2) ||
            (dim == 2 && positions.size(0) != q.size(0))) Py_RETURN_NONE;
    }
    r.rotary = rotary_arg(a[2]);
    r.check_status = a[6] == Py_True;
    const std::array<Tensor, 2> y = without_gil([&] { return rotate(x, positions, r); });
    return tuple_of({y[0], y[1]});
    END_HANDLE_TH_ERRORS
}

// try_append(k, v, <cache>, <sequences>, rotary or None, its head_dim, check_status) -> whether it was done
PyObject* py_try_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    want(n, 13);
    if (torch::jit::tracer::isTracing() || !THPVariable_Check(a[0]) || !THPVariable_Check(a[1])) Py_RETURN_FALSE;
    const Tensor &k = THPVariable_Unpack(a[0]), &v = THPVariable_Unpack(a[1]), &ck = THPVariable_Unpack(a[2]);
    if (!common_rows(k, ck, a[4], a[6]) || !common_rows(v, ck, a[4], a[6]) || k.sizes() != v.sizes() || k.size(1) != ck.size(1) ||
        !common_sequences(a + 7, ck, k.size(0)) || !common_rotary(a[10], a[11], k.size(3))) Py_RETURN_FALSE;
    Untracked untracked;
    const c10::cuda::CUDAGuard device(k.device());
    Cache cache = cache_args(a + 2);
    const Sequences seq = sequence_args(a + 7);
    const bob_sm100_rotary rotary = rotary_arg(a[10]);
    const bool check = a[12] == Py_True;
    without_gil([&] { run_append(k, v, cache, seq, rotary, check); return 0; });
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// try_paged(q, <cache>, <sequences>, rotary or None, its head_dim, is_causal, scale, window_size, check_status) -> out, or None
PyObject* py_try_paged(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    want(n, 15);
    if (torch::jit::tracer::isTracing() || !THPVariable_Check(a[0])) Py_RETURN_NONE;
    const Tensor &q = THPVariable_Unpack(a[0]), &ck = THPVariable_Unpack(a[1]);
    if (!common_rows(q, ck, a[3], a[5])) Py_RETURN_NONE;
    const int64_t group = q.size(1) / ck.size(1);
    if (group * ck.size(1) != q.size(1) || group < 1 || group > 32 || !common_sequences(a + 6, ck, q.size(0)) || !common_rotary(a[9], a[10], q.size(3)))
        Py_RETURN_NONE;
    if (!PyBool_Check(a[11]) || !is_int(a[13])) Py_RETURN_NONE;
    const bool causal = a[11] == Py_True;
    int overflow = 0;
    const int64_t window = PyLong_AsLongLongAndOverflow(a[13], &overflow);
    if (overflow || window < 0 || window > (1 << 28) || (!causal && (window > 0 || a[9] != Py_None))) Py_RETURN_NONE;
    std::optional<double> scale;
    if (a[12] != Py_None) {
        if (!PyFloat_CheckExact(a[12])) Py_RETURN_NONE;
        const float s = static_cast<float>(PyFloat_AS_DOUBLE(a[12]));
        if (!(s > 0) || !std::isfinite(s)) Py_RETURN_NONE;
        scale = PyFloat_AS_DOUBLE(a[12]);
    }
    Untracked untracked;
    const c10::cuda::CUDAGuard device(q.device());
    const Cache cache = cache_args(a + 1);
    const Sequences seq = sequence_args(a + 6);
    const bob_sm100_rotary rotary = rotary_arg(a[9]);
    const bool check = a[14] == Py_True;
    return THPVariable_Wrap(without_gil([&] { return run_paged(q, cache, seq, rotary, causal, window, scale, check); }));
    END_HANDLE_TH_ERRORS
}

// rotate(q, k or None, rotary, positions or None, first, check_status) -> (q, k)
PyObject* py_rotate(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    want(n, 6);
    const std::array<Tensor, 2> x{tensor_arg(a[0]), optional_tensor_arg(a[1])};
    Rotation r;
    r.rotary = rotary_arg(a[2]);
    const Tensor positions = optional_tensor_arg(a[3]);
    r.first = int_arg(a[4]);
    r.check_status = PyObject_IsTrue(a[5]);
    const std::array<Tensor, 2> y = without_gil([&] { return rotate(x, positions, r); });
    return tuple_of({y[0], y[1]});
    END_HANDLE_TH_ERRORS
}

// cache_append(k, v, <cache>, <sequences>, rotary or None, check_status)
PyObject* py_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    want(n, 12);
    Untracked untracked;
    const Tensor &k = tensor_arg(a[0]), &v = tensor_arg(a[1]);
    const c10::cuda::CUDAGuard device(k.device());
    Cache cache = cache_args(a + 2);
    const Sequences seq = sequence_args(a + 7);
    const bob_sm100_rotary rotary = rotary_arg(a[10]);
    const bool check = PyObject_IsTrue(a[11]);
    without_gil([&] { run_append(k, v, cache, seq, rotary, check); return 0; });
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// cache_read(<cache>, <sequences>, n, check_status) -> (k, v)
PyObject* py_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    want(n, 10);
    Untracked untracked;
    const c10::cuda::CUDAGuard device(tensor_arg(a[0]).device());
    const Cache cache = cache_args(a);
    const Sequences seq = sequence_args(a + 5);
    const int64_t rows = int_arg(a[8]);
    const bool check = PyObject_IsTrue(a[9]);
    const std::array<Tensor, 2> r =
        without_gil([&] { return run_read(cache, seq, rows, cache.c.dtype == BOB_SM100_BF16 ? at::kBFloat16 : at::kHalf, check); });
    return tuple_of({r[0], r[1]});
    END_HANDLE_TH_ERRORS
}

// paged(q, <cache>, <sequences>, rotary or None, is_causal, window_size, scale or None, check_status) -> out
PyObject* py_paged(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    want(n, 14);
    Untracked untracked;
    const Tensor& q = tensor_arg(a[0]);
    const c10::cuda::CUDAGuard device(q.device());
    const Cache cache = cache_args(a + 1);
    const Sequences seq = sequence_args(a + 6);
    const bob_sm100_rotary rotary = rotary_arg(a[9]);
    const bool causal = PyObject_IsTrue(a[10]), check = PyObject_IsTrue(a[13]);
    const int64_t window = int_arg(a[11]);
    std::optional<double> scale;
    if (a[12] != Py_None) {
        scale = PyFloat_AsDouble(a[12]);
        if (PyErr_Occurred()) throw python_error();
    }
    return THPVariable_Wrap(without_gil([&] { return run_paged(q, cache, seq, rotary, causal, window, scale, check); }));
    END_HANDLE_TH_ERRORS
}

// bind(error class, addresses of fwd, bwd1, bwd2, workspace_bytes, read_status, last_status, error_string, rotate,
// cache_append, cache_read, paged_workspace_bytes, paged_fwd)
PyObject* py_bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    want(n, 13);
    auto address = [&](int i) { return reinterpret_cast<void*>(int_arg(a[i])); };
    Py_INCREF(a[0]);
    error_class = a[0];
    lib.fwd = reinterpret_cast<decltype(lib.fwd)>(address(1));
    lib.bwd1 = reinterpret_cast<decltype(lib.bwd1)>(address(2));
    lib.bwd2 = reinterpret_cast<decltype(lib.bwd2)>(address(3));
    lib.workspace_bytes = reinterpret_cast<decltype(lib.workspace_bytes)>(address(4));
    lib.read_status = reinterpret_cast<decltype(lib.read_status)>(address(5));
    lib.last_status = reinterpret_cast<decltype(lib.last_status)>(address(6));
    lib.error_string = reinterpret_cast<decltype(lib.error_string)>(address(7));
    lib.rotate = reinterpret_cast<decltype(lib.rotate)>(address(8));
    lib.cache_append = reinterpret_cast<decltype(lib.cache_append)>(address(9));
    lib.cache_read = reinterpret_cast<decltype(lib.cache_read)>(address(10));
    lib.paged_workspace_bytes = reinterpret_cast<decltype(lib.paged_workspace_bytes)>(address(11));
    lib.paged_fwd = reinterpret_cast<decltype(lib.paged_fwd)>(address(12));
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

#define BOB_METHOD(name, fn) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(fn)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {
    BOB_METHOD("try_sdpa", py_try_sdpa), BOB_METHOD("sdpa", py_sdpa), BOB_METHOD("forward", py_forward),
    BOB_METHOD("first_backward", py_first), BOB_METHOD("second_backward", py_second), BOB_METHOD("bind", py_bind),
    BOB_METHOD("rotate", py_rotate), BOB_METHOD("cache_append", py_append), BOB_METHOD("cache_read", py_read), BOB_METHOD("paged", py_paged),
    BOB_METHOD("try_rotate", py_try_rotate), BOB_METHOD("try_append", py_try_append), BOB_METHOD("try_paged", py_try_paged),
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "bob_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_bob_torch() { return PyModule_Create(&module_def); }
