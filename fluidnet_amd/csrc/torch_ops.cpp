// What the operators on torch tensors do on the host, as a Python extension module (fluidnet_amd/engine/_torch_ops.so): the checks, the autograd
// node of the norms around a residual block, and the address tables of lists of tensors.  The kernels and their C ABI are libfluidnet_hip.
//
// Why native: a training pass of these operators takes 15 to 50 us on the GPU.  With the node in Python its backward ran on autograd's thread behind
// the interpreter lock and cost 100 us; a list of 60 parameters cost 70 us in Python loops.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>

#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>

#include <string>
#include <unordered_set>
#include <vector>

#include "../../include/fluidnet_hip.h"

namespace {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::variable_list;

// The entry points used here, of the library that engine.runtime has loaded, and its FluidNetHipError; set by bind()
struct Library {
    decltype(&fnet_block_norm_fwd) block_norm_fwd;
    decltype(&fnet_block_norm_bwd) block_norm_bwd;
    decltype(&fnet_block_norm_workspace) block_norm_workspace;
    decltype(&fnet_strerror) strerror;
    decltype(&fnet_last_hip_error) last_hip_error;
} g_lib;
PyObject* g_hip_error = nullptr;

struct HipFailure : std::runtime_error {
    using std::runtime_error::runtime_error;
};
void check_rc(int rc, const char* what) {
    if (rc == FNET_OK) return;
    std::string s = std::string(what) + ": " + g_lib.strerror(rc);
    if (rc == FNET_E_HIP) s += " hipError=" + std::to_string(g_lib.last_hip_error());
    throw HipFailure(s);
}

int code_of(at::ScalarType t) {
    return t == at::kFloat ? FNET_F32 : t == at::kBFloat16 ? FNET_BF16 : t == at::kHalf ? FNET_F16 : -1;
}
std::string name_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return "torch.float32";
        case at::kBFloat16: return "torch.bfloat16";
        case at::kHalf: return "torch.float16";
        case at::kDouble: return "torch.float64";
        default: return c10::toString(t);
    }
}
std::string shape_of(const Tensor& t) {
    std::string s = "(";
    for (int64_t d = 0; d < t.dim(); ++d) s += (d ? ", " : "") + std::to_string(t.size(d));
    return s + (t.dim() == 1 ? ",)" : ")");
}

hipStream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.get_device()).stream(); }

// ---- norms around a residual block
enum { X, BRANCH, GATE, SCALE, POST_W, POST_B, PRE_W, PRE_B, INPUTS };

struct Spec {
    FnetBlockNorm a;                          // all but addresses and row strides
    bool pre;
};

void check_param(const char* name, const Tensor& t, const Tensor& x, int& seen) {
    if (!t.defined()) return;
    const int64_t C = x.size(-1);
    TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == C && t.device() == x.device(), name, " must have shape (", C, ",) on ", x.device(), " (got ",
                      shape_of(t), " on ", t.device(), ")");
    TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat || t.scalar_type() == x.scalar_type(), name, " must be float32 or ", name_of(x.scalar_type()), " (got ",
                      name_of(t.scalar_type()), ")");
    const int code = code_of(t.scalar_type());
    TORCH_CHECK_VALUE(seen < 0 || seen == code, "weights, biases and scale must all have one type");
    seen = code;
}

int gate_kind(const Tensor& gate, const Tensor& x) {
    const auto g = gate.sizes(), s = x.sizes();
    const size_t n = s.size();
    if (g.size() == 1 && g[0] == s[n - 1] && n > 1) return FNET_GATE_CHANNEL;
    if (g == s) return FNET_GATE_ELEMENT;
    if (g.size() == n) {
        const auto ones = [&](size_t from) {
            for (size_t d = from; d + 1 < n; ++d)
                if (g[d] != 1) return false;
            return true;
        };
        if (g.slice(0, n - 1) == s.slice(0, n - 1) && g[n - 1] == 1) return FNET_GATE_TOKEN;
        if (g[n - 1] == s[n - 1]) {
            if (n > 2 && g[0] == s[0] && ones(1)) return FNET_GATE_SAMPLE;
            if (ones(0)) return FNET_GATE_CHANNEL;
        }
    }
    TORCH_CHECK_VALUE(false, "gate of shape ", shape_of(gate), " for x of shape ", shape_of(x), ": expected x's shape, [..., 1], [B, 1, .., C] or [C]");
}

Spec make_spec(const Tensor (&in)[INPUTS], int kind, bool post, bool pre, int act, double residual_scale, double eps) {
    const Tensor &x = in[X], &branch = in[BRANCH], &gate = in[GATE];
    Spec s{};
    FnetBlockNorm& a = s.a;
    a.dtype = code_of(x.scalar_type());
    TORCH_CHECK_VALUE(a.dtype >= 0, "x must be float32, bfloat16 or float16 (got ", name_of(x.scalar_type()), ")");
    TORCH_CHECK_VALUE(x.dim() > 0 && x.size(-1) >= 1 && x.size(-1) <= FNET_BLOCK_NORM_MAX_WIDTH, "the last axis must have 1 to ", FNET_BLOCK_NORM_MAX_WIDTH,
                      " elements (got shape ", shape_of(x), ")");
    TORCH_CHECK_VALUE(eps >= 0, "eps must not be negative (got ", eps, ")");
    a.width = (int32_t)x.size(-1);
    a.rows = a.tokens = x.numel() / a.width;
    TORCH_CHECK_VALUE(a.rows < (1ll << 31), "at most 2^31 - 1 rows");
    if (!branch.defined()) {
        TORCH_CHECK_VALUE(!gate.defined() && !in[SCALE].defined(), "a gate or scale needs a branch");
        post = false;
    } else {
        TORCH_CHECK_VALUE(branch.sizes() == x.sizes() && branch.scalar_type() == x.scalar_type() && branch.device() == x.device(), "branch must be like x: ",
                          shape_of(x), " ", name_of(x.scalar_type()), " on ", x.device(), " (got ", shape_of(branch), " ", name_of(branch.scalar_type()),
                          " on ", branch.device(), ")");
    }
    TORCH_CHECK_VALUE(post || (!in[POST_W].defined() && !in[POST_B].defined()), "post_weight / post_bias need post=True");
    TORCH_CHECK_VALUE(pre || (!in[PRE_W].defined() && !in[PRE_B].defined()), "pre_weight / pre_bias need pre=True");
    int seen = -1;
    check_param("scale", in[SCALE], x, seen);
    check_param("post_weight", in[POST_W], x, seen);
    check_param("post_bias", in[POST_B], x, seen);
    check_param("pre_weight", in[PRE_W], x, seen);
    check_param("pre_bias", in[PRE_B], x, seen);
    a.param_dtype = seen < 0 ? FNET_F32 : seen;
    if (gate.defined()) {
        TORCH_CHECK_VALUE(gate.device() == x.device() && (gate.scalar_type() == at::kFloat || gate.scalar_type() == x.scalar_type()), "gate must be float32 or ",
                          name_of(x.scalar_type()), " on ", x.device(), " (got ", name_of(gate.scalar_type()), " on ", gate.device(), ")");
        a.gate_kind = gate_kind(gate, x);
        a.gate_dtype = code_of(gate.scalar_type());
        if (a.gate_kind == FNET_GATE_SAMPLE && a.rows) {
            a.tokens = a.rows / x.size(0);
            if (a.tokens == 1) a.gate_kind = FNET_GATE_ELEMENT;      // a row of values per row
        }
    }
    a.kind = kind;
    a.post = post;
    a.gate_act = act;
    a.residual_scale = (float)residual_scale;
    a.eps = (float)eps;
    s.pre = pre;
    TORCH_CHECK(x.is_cuda(), "fluidnet_amd block norms run on MI355X only (got a CPU tensor); there is no CPU fallback");
    for (const Tensor& t : in)
        TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(), "fluidnet_amd block norms have no forward-mode derivative");
    return s;
}

// The distance of the rows; the tensor is copied if its last axis is not dense or its rows are not evenly spaced.
int64_t rows_of(Tensor& t) {
    const auto size = t.sizes(), stride = t.strides();
    const int64_t n = t.dim(), C = size[n - 1];
    if (t.is_neg()) t = t.resolve_neg();
    if (t.is_contiguous()) return C;
    if (stride[n - 1] == 1 || C == 1) {
        int64_t step = -1, count = 1;                 // distance of neighbouring rows; rows in the axes looked at so far
        bool even = true;
        for (int64_t d = n - 2; d >= 0 && even; --d) {
            if (size[d] == 1) continue;
            if (step < 0) step = stride[d];
            else even = stride[d] == step * count;
            count *= size[d];
        }
        if (even) return step < 0 ? C : step;
    }
    t = t.contiguous();
    return C;
}
uint64_t address(const Tensor& t) { return t.defined() ? (uint64_t)t.data_ptr() : 0; }
uint64_t dense_address(Tensor& t) {
    if (!t.defined()) return 0;
    if (t.is_neg()) t = t.resolve_neg();
    t = t.contiguous();
    return (uint64_t)t.data_ptr();
}

// What both directions read, as the kernels take it; `in` is left as the tensors that the addresses belong to
void put_operands(FnetBlockNorm& a, Tensor (&in)[INPUTS]) {
    a.x_stride = rows_of(in[X]);
    a.x = address(in[X]);
    if (in[BRANCH].defined()) {
        a.branch_stride = rows_of(in[BRANCH]);
        a.branch = address(in[BRANCH]);
        if (in[GATE].defined()) {
            Tensor& g = in[GATE];
            if (g.is_neg()) g = g.resolve_neg();
            if (a.gate_kind == FNET_GATE_ELEMENT || a.gate_kind == FNET_GATE_TOKEN) {
                a.gate_stride = rows_of(g);
            } else if (a.gate_kind == FNET_GATE_SAMPLE && g.stride(-1) == 1) {
                a.gate_stride = g.stride(0);
            } else {
                g = g.contiguous();
                a.gate_stride = a.width;
            }
            a.gate = address(g);
        }
    }
    a.scale = dense_address(in[SCALE]);
    a.post_weight = dense_address(in[POST_W]);
    a.post_bias = dense_address(in[POST_B]);
    a.pre_weight = dense_address(in[PRE_W]);
    a.pre_bias = dense_address(in[PRE_B]);
}

Tensor like(const Tensor& t, bool zero = false) {
    return zero ? at::zeros_like(t, t.options(), at::MemoryFormat::Contiguous) : at::empty_like(t, t.options(), at::MemoryFormat::Contiguous);
}

struct Outputs { Tensor y, h, stats; };
Outputs run_forward(const Spec& s, const Tensor (&given)[INPUTS], bool keep) {
    at::AutoDispatchBelowADInplaceOrView below;
    Outputs out;
    Tensor in[INPUTS];
    for (int i = 0; i < INPUTS; ++i) in[i] = given[i];
    FnetBlockNorm a = s.a;
    c10::DeviceGuard guard(in[X].device());
    if (in[BRANCH].defined()) out.y = like(in[X]);
    if (s.pre) out.h = like(in[X]);
    if (keep && (a.post || s.pre)) out.stats = at::empty({4, a.rows}, in[X].options().dtype(at::kFloat));
    if (a.rows == 0 || (!out.y.defined() && !out.h.defined())) return out;
    put_operands(a, in);
    a.y = address(out.y);
    a.h = address(out.h);
    a.stats = address(out.stats);
    check_rc(g_lib.block_norm_fwd(&a, stream_of(in[X])), "fnet_block_norm_fwd");
    return out;
}

// the nodes of leaves in the graph below `node`
std::unordered_set<Node*> leaves_below(Node* node) {
    std::unordered_set<Node*> seen{node}, leaves;
    std::vector<Node*> todo{node};
    while (!todo.empty()) {
        Node* n = todo.back();
        todo.pop_back();
        for (const auto& e : n->next_edges()) {
            Node* below = e.function.get();
            if (!below || !seen.insert(below).second) continue;
            todo.push_back(below);
            if (dynamic_cast<torch::autograd::AccumulateGrad*>(below)) leaves.insert(below);
        }
    }
    return leaves;
}
// While a graph is captured: refuses if a leaf's gradient would be ordered after the default stream, where its node was made.  A leaf's node
// lives as long as any graph (of whatever operation) or anyone else holds it.
void check_capture(Node* node) {
    const auto* info = torch::autograd::get_current_graph_task_exec_info();
    for (Node* leaf : leaves_below(node)) {
        if (info && !info->empty()) {
            const auto it = info->find(leaf);
            if (it == info->end() || !it->second.should_execute()) continue;
        }
        const auto made_on = leaf->stream();
        TORCH_CHECK(!made_on || made_on->id() != 0, "outputs of an earlier call from the same leaves, made on the default stream, are alive: drop them "
                                                    "before capturing a backward pass");
    }
}

struct BlockNormBackward : public Node {
    Spec spec;
    bool has_y = false;
    torch::autograd::SavedVariable saved[INPUTS], stats;

    std::string name() const override { return "BlockNormBackward"; }
    // mutex_ guards what is saved, as in torch's own nodes: a backward pass on one thread may release it while another one reads it
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        for (auto& v : saved) v.reset_data();
        stats.reset_data();
    }
    variable_list apply(variable_list&& grads) override {
        variable_list out = gradients(grads);
        if (!at::GradMode::is_enabled()) return out;
        // create_graph: the gradients are functions of the operands whose derivative is not there, so whoever asks for it is told
        for (Tensor& t : out)
            if (t.defined()) t = t.detach().set_requires_grad(true);
        torch::autograd::DelayedError error("trying to differentiate twice a function that was marked with @once_differentiable", (int64_t)out.size());
        return error.apply(std::move(out));
    }

    variable_list gradients(const variable_list& grads) {
        variable_list out(INPUTS);
        Tensor dy = has_y ? grads[0] : Tensor(), dh = spec.pre ? grads[has_y ? 1 : 0] : Tensor();
        if (!dy.defined() && !dh.defined()) return out;
        Tensor in[INPUTS], st;
        {
            std::lock_guard<std::mutex> lock(mutex_);
            for (int i = 0; i < INPUTS; ++i) in[i] = saved[i].unpack();
            st = stats.unpack();
        }
        at::AutoDispatchBelowADInplaceOrView below;
        FnetBlockNorm a = spec.a;
        c10::DeviceGuard guard(in[X].device());
        const hipStream_t stream = stream_of(in[X]);
        hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
        if (stream && hipStreamIsCapturing(stream, &capture) == hipSuccess && capture != hipStreamCaptureStatusNone) check_capture(this);
        const bool none = a.rows == 0, with_h = dh.defined();
        bool sums = false;
        for (int i = 0; i < INPUTS; ++i) {
            if (!in[i].defined() || !task_should_compute_output(i)) continue;
            // without a gradient of h, the gradient of x is that of y, and the second norm's are zero
            if (i == X && !with_h) out[X] = dy;
            else out[i] = like(in[i], none || (!with_h && i >= PRE_W));
            sums = sums || i >= GATE;
        }
        if (none || !(with_h || out[BRANCH].defined() || sums)) return out;
        put_operands(a, in);
        a.stats = address(st);
        if (dy.defined()) {
            a.dy_stride = rows_of(dy);
            a.dy = address(dy);
        }
        if (with_h) {
            a.dh_stride = rows_of(dh);
            a.dh = address(dh);
            a.dx = address(out[X]);
            a.dpre_weight = address(out[PRE_W]);
            a.dpre_bias = address(out[PRE_B]);
        }
        a.dbranch = address(out[BRANCH]);
        a.dgate = address(out[GATE]);
        a.dscale = address(out[SCALE]);
        a.dpost_weight = address(out[POST_W]);
        a.dpost_bias = address(out[POST_B]);
        Tensor workspace;                             // partial sums of what is summed over rows
        if (sums) {
            check_rc(g_lib.block_norm_workspace(&a, &a.workspace_bytes), "fnet_block_norm_workspace");
            if (a.workspace_bytes) workspace = at::empty({a.workspace_bytes}, in[X].options().dtype(at::kByte));
            a.workspace = address(workspace);
        }
        check_rc(g_lib.block_norm_bwd(&a, stream), "fnet_block_norm_bwd");
        return out;
    }
};

struct Released {                             // the interpreter lock, while nothing of Python is touched
    PyThreadState* state = PyEval_SaveThread();
    ~Released() { PyEval_RestoreThread(state); }
};

Outputs block_norm(const Tensor (&in)[INPUTS], int kind, bool post, bool pre, int act, double residual_scale, double eps) {
    const Spec s = make_spec(in, kind, post, pre, act, residual_scale, eps);
    bool wanted = false;
    if (at::GradMode::is_enabled())
        for (const Tensor& t : in) wanted = wanted || (t.defined() && t.requires_grad());
    Outputs out = run_forward(s, in, wanted);
    if (!wanted) return out;
    auto node = std::shared_ptr<BlockNormBackward>(new BlockNormBackward(), torch::autograd::deleteNode);
    node->spec = s;
    node->has_y = out.y.defined();
    node->set_next_edges(torch::autograd::collect_next_edges(in[0], in[1], in[2], in[3], in[4], in[5], in[6], in[7]));
    for (int i = 0; i < INPUTS; ++i)
        if (in[i].defined()) node->saved[i] = torch::autograd::SavedVariable(in[i], false);
    if (out.stats.defined()) node->stats = torch::autograd::SavedVariable(out.stats, false);
    if (out.y.defined()) torch::autograd::set_history(out.y, node);
    if (out.h.defined()) torch::autograd::set_history(out.h, node);
    return out;
}

#define FNET_PY_BEGIN HANDLE_TH_ERRORS try {
#define FNET_PY_END                                                         \
    } catch (const HipFailure& e) {                                          \
        PyErr_SetString(g_hip_error, e.what());                              \
        return nullptr;                                                      \
    }                                                                        \
    END_HANDLE_TH_ERRORS

PyObject* wrap(const Tensor& t) {
    if (t.defined()) return THPVariable_Wrap(t);
    Py_RETURN_NONE;
}

// block_norm(x, branch, gate, scale, post_weight, post_bias, pre_weight, pre_bias, kind, post, pre, gate_act, residual_scale, eps) -> (y, h)
PyObject* py_block_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
    FNET_PY_BEGIN
    static const char* const names[INPUTS] = {"x", "branch", "gate", "scale", "post_weight", "post_bias", "pre_weight", "pre_bias"};
    TORCH_CHECK_TYPE(n == INPUTS + 6, "block_norm takes ", INPUTS + 6, " arguments (got ", n, ")");
    Tensor in[INPUTS];
    for (int i = 0; i < INPUTS; ++i) {
        if (i != X && args[i] == Py_None) continue;
        TORCH_CHECK_TYPE(THPVariable_Check(args[i]), names[i], " must be a tensor (got ", Py_TYPE(args[i])->tp_name, ")");
        in[i] = THPVariable_Unpack(args[i]);
    }
    const long kind = PyLong_AsLong(args[8]), act = PyLong_AsLong(args[11]);
    const int post = PyObject_IsTrue(args[9]), pre = PyObject_IsTrue(args[10]);
    const double scale = PyFloat_AsDouble(args[12]), eps = PyFloat_AsDouble(args[13]);
    if (PyErr_Occurred()) return nullptr;
    Outputs out;
    {
        Released gil;
        out = block_norm(in, (int)kind, post, pre, (int)act, scale, eps);
    }
    PyObject *y = wrap(out.y), *h = wrap(out.h), *both = y && h ? PyTuple_Pack(2, y, h) : nullptr;
    Py_XDECREF(y);
    Py_XDECREF(h);
    return both;
    FNET_PY_END
}

// ---- lists of tensors
struct List {                                 // of the items of a list or tuple, for as long as the call lasts
    PyObject* fast;
    explicit List(PyObject* o) : fast(PySequence_Fast(o, "expected a list of tensors")) {
        if (!fast) throw python_error();
    }
    ~List() { Py_XDECREF(fast); }
    List(const List&) = delete;
    Py_ssize_t size() const { return PySequence_Fast_GET_SIZE(fast); }
    bool none(Py_ssize_t k) const { return PySequence_Fast_GET_ITEM(fast, k) == Py_None; }
    const Tensor& operator[](Py_ssize_t k) const {
        PyObject* o = PySequence_Fast_GET_ITEM(fast, k);
        TORCH_CHECK_TYPE(THPVariable_Check(o), "expected a tensor (got ", Py_TYPE(o)->tp_name, ")");
        return THPVariable_Unpack(o);
    }
};
template <typename T>
PyObject* to_bytes(const std::vector<T>& v) { return PyBytes_FromStringAndSize((const char*)v.data(), (Py_ssize_t)(v.size() * sizeof(T))); }

// tensor_table(tensors) -> (all contiguous, addresses, element counts, types), or None unless all are fp32, bf16 or fp16 on one GPU
PyObject* py_tensor_table(PyObject*, PyObject* arg) {
    FNET_PY_BEGIN
    const List list(arg);
    const Py_ssize_t n = list.size();
    std::vector<uint64_t> ptr(n);
    std::vector<int64_t> numel(n);
    std::vector<int32_t> type(n);
    bool contiguous = true;
    for (Py_ssize_t k = 0; k < n; ++k) {
        const Tensor& t = list[k];
        type[k] = code_of(t.scalar_type());
        if (type[k] < 0 || !t.is_cuda() || t.is_neg() || t.device() != list[0].device()) Py_RETURN_NONE;
        contiguous = contiguous && t.is_contiguous();
        ptr[k] = (uint64_t)t.data_ptr();
        numel[k] = t.numel();
    }
    return Py_BuildValue("(NNNN)", PyBool_FromLong(contiguous), to_bytes(ptr), to_bytes(numel), to_bytes(type));
    FNET_PY_END
}

// addresses(tensors): of dense tensors; 0 for None
PyObject* py_addresses(PyObject*, PyObject* arg) {
    FNET_PY_BEGIN
    const List list(arg);
    std::vector<uint64_t> ptr(list.size());
    for (Py_ssize_t k = 0; k < list.size(); ++k) ptr[k] = list.none(k) ? 0 : (uint64_t)list[k].data_ptr();
    return to_bytes(ptr);
    FNET_PY_END
}

// marks(tensors): address and version of each, as bytes to compare
PyObject* py_marks(PyObject*, PyObject* arg) {
    FNET_PY_BEGIN
    const List list(arg);
    std::vector<uint64_t> mark(2 * list.size());
    for (Py_ssize_t k = 0; k < list.size(); ++k) {
        mark[2 * k] = (uint64_t)list[k].data_ptr();
        mark[2 * k + 1] = (uint64_t)list[k]._version();
    }
    return to_bytes(mark);
    FNET_PY_END
}

// adam_fits(params, grads, exp_avgs, exp_avg_sqs, masters): whether every parameter, its gradient (of its type), moments and, unless it is fp32,
// master (all fp32) are contiguous, of one shape and on the first gradient's device
PyObject* py_adam_fits(PyObject*, PyObject* const* args, Py_ssize_t n) {
    FNET_PY_BEGIN
    TORCH_CHECK_TYPE(n == 5, "adam_fits takes 5 lists");
    const List params(args[0]), grads(args[1]), m(args[2]), v(args[3]), masters(args[4]);
    const auto fits = [&](const Tensor& t, const Tensor& g, at::ScalarType type) {
        return t.scalar_type() == type && t.device() == g.device() && t.sizes() == g.sizes() && t.is_contiguous() && !t.is_neg();
    };
    bool ok = true;
    for (Py_ssize_t k = 0; k < grads.size() && ok; ++k) {
        const Tensor& g = grads[k];
        ok = g.is_contiguous() && g.device() == grads[0].device() && fits(params[k], g, g.scalar_type()) && fits(m[k], g, at::kFloat) &&
             fits(v[k], g, at::kFloat) && (g.scalar_type() == at::kFloat || (!masters.none(k) && fits(masters[k], g, at::kFloat)));
    }
    return PyBool_FromLong(ok);
    FNET_PY_END
}

// written(params, exp_avgs, exp_avg_sqs, masters, clock): tells autograd of an Adam step in place.  Masters of fp32 parameters are not written.
PyObject* py_written(PyObject*, PyObject* const* args, Py_ssize_t n) {
    FNET_PY_BEGIN
    TORCH_CHECK_TYPE(n == 5 && THPVariable_Check(args[4]), "written takes 4 lists and a tensor");
    const auto bump = [](const Tensor& t) {
        if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    };
    const List params(args[0]), m(args[1]), v(args[2]), masters(args[3]);
    for (Py_ssize_t k = 0; k < params.size(); ++k) {
        bump(params[k]);
        bump(m[k]);
        bump(v[k]);
        if (params[k].scalar_type() != at::kFloat) bump(masters[k]);
    }
    bump(THPVariable_Unpack(args[4]));
    Py_RETURN_NONE;
    FNET_PY_END
}

// bind(error class, addresses of the entry points in Library's order); before anything else
PyObject* py_bind(PyObject*, PyObject* args) {
    PyObject* cls;
    unsigned long long at[5];
    if (!PyArg_ParseTuple(args, "OKKKKK", &cls, at, at + 1, at + 2, at + 3, at + 4)) return nullptr;
    g_lib = Library{(decltype(g_lib.block_norm_fwd))at[0], (decltype(g_lib.block_norm_bwd))at[1], (decltype(g_lib.block_norm_workspace))at[2],
                    (decltype(g_lib.strerror))at[3], (decltype(g_lib.last_hip_error))at[4]};
    Py_INCREF(cls);
    Py_XDECREF(g_hip_error);
    g_hip_error = cls;
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"block_norm", (PyCFunction)(void (*)(void))py_block_norm, METH_FASTCALL, nullptr},
    {"tensor_table", py_tensor_table, METH_O, nullptr},
    {"addresses", py_addresses, METH_O, nullptr},
    {"marks", py_marks, METH_O, nullptr},
    {"adam_fits", (PyCFunction)(void (*)(void))py_adam_fits, METH_FASTCALL, nullptr},
    {"written", (PyCFunction)(void (*)(void))py_written, METH_FASTCALL, nullptr},
    {"bind", py_bind, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_ops", "Host side of the operators on torch tensors", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_ops() { return PyModule_Create(&module); }
