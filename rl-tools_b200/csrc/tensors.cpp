// The operators of residual networks on torch tensors: checks of the operands, outputs and workspaces from torch's allocator, the current stream, one C call. Compiled,
// because a small call is host time: the same steps in Python with ctypes cost 10 to 40 us a call, of which the kernel needs 3 to 5. The Python wrappers (residual.py) hold the
// names and defaults; the kernels are reached through the addresses of the C entry points that `bind` is given.
#include <Python.h>
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include "../../include/b200rl.h"
#include <string>
#include <type_traits>

namespace {

PyObject *g_refusal = nullptr, *g_status = nullptr;      // exceptions: what is wrong with the arguments; the status of a C entry point

#define ENTRY(name) decltype(&b200rl_##name) name = nullptr
struct Entries {
    ENTRY(dense_residual_forward_workspace_bytes); ENTRY(dense_residual_forward); ENTRY(dense_residual_backward_activation);
    ENTRY(dense_residual_backward_input_workspace_bytes); ENTRY(dense_residual_backward_input);
    ENTRY(dense_residual_backward_weights_workspace_bytes); ENTRY(dense_residual_backward_weights);
    ENTRY(norm_residual_forward); ENTRY(norm_residual_backward_scratch_bytes); ENTRY(norm_residual_backward); ENTRY(dropout);
} E;

struct Refusal { std::string what; };
struct Status { int status; };
// text by std::to_string, not by streams: torch's libraries export parts of libstdc++'s stream classes whose locales nobody has set up
std::string text(const char* s){ return s; }
std::string text(const std::string& s){ return s; }
template <typename I, typename = std::enable_if_t<std::is_integral<I>::value>> std::string text(I i){ return std::to_string(i); }
template <typename... A> [[noreturn]] void refuse(const A&... a){ std::string s; ((s += text(a)), ...); throw Refusal{s}; }
void check(int status){ if(status) throw Status{status}; }

struct Matrix { void* p; int ld; };
const at::Tensor* tensor(const char* call, const char* name, PyObject* o){
    if(o == Py_None) return nullptr;
    if(!THPVariable_Check(o)) refuse(call, ": ", name, " has to be a tensor");
    return &THPVariable_Unpack(o);
}
const char* type_name(at::ScalarType t){ return t == at::kFloat ? "float32" : t == at::kBFloat16 ? "bfloat16" : t == at::kHalf ? "float16" : c10::toString(t); }

std::string shape(const at::Tensor& t){
    std::string s = "[";
    for(int64_t i = 0; i < t.dim(); i++) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + "]";
}

// The operands of one call: each is checked against the type, the shape and the current device and gives its address and pitch.
struct Operands {
    const char* call;
    at::ScalarType dtype;
    int type;
    int device = -1;                                     // the first tensor's; -2: on no GPU, -3: two devices
    int other = -1;
    Operands(const char* call, const at::Tensor& first, bool fp32) : call(call), dtype(first.scalar_type()) {
        type = dtype == at::kFloat && fp32 ? B200RL_TYPE_FLOAT32 : dtype == at::kBFloat16 ? B200RL_TYPE_BFLOAT16 : dtype == at::kHalf ? B200RL_TYPE_FLOAT16 : -1;
        if(type < 0) refuse(call, ": no kernel for matrices of ", type_name(dtype));
    }
    void seen(const at::Tensor& t){
        const int d = t.is_cuda() ? (int)t.get_device() : -2;
        if(device == -1) device = d;
        else if(d != device && device >= 0){ other = d; device = d == -2 ? -2 : -3; }
    }
    Matrix matrix(const char* name, const at::Tensor* t, int64_t rows, int64_t cols){
        if(!t) return {nullptr, 0};
        if(t->scalar_type() != dtype || t->dim() != 2 || t->size(0) != rows || t->size(1) != cols)
            refuse(call, ": ", name, " is a ", shape(*t), " ", type_name(t->scalar_type()), ", not a [", rows, ", ", cols, "] ", type_name(dtype));
        if(cols > 1 && t->stride(1) != 1) refuse(call, ": the elements of ", name, "'s rows do not follow one another");
        const int64_t ld = rows > 1 ? t->stride(0) : cols;
        if(ld < cols) refuse(call, ": the rows of ", name, " overlap");
        if(rows > INT_MAX || ld > INT_MAX) refuse(call, ": ", name, " has more than 2^31 - 1 rows, or elements from one row to the next");
        seen(*t);
        return {t->data_ptr(), (int)ld};
    }
    float* vector(const char* name, const at::Tensor* t, int64_t n){
        if(!t) return nullptr;
        if(t->scalar_type() != at::kFloat || t->dim() != 1 || t->size(0) != n || (n > 1 && t->stride(0) != 1)) refuse(call, ": ", name, " is not ", n, " float32 values in a row");
        seen(*t);
        return static_cast<float*>(t->data_ptr());
    }
    // all on the current device (looked at last: types and shapes are refused on machines without one too); returns the current stream
    void* here(){
        if(device == -2) refuse(call, ": takes CUDA tensors");
        const int current = c10::cuda::current_device();
        if(device != current) refuse(call, ": a tensor lies on cuda:", device == -3 ? other : device, ", the current device is cuda:", current);
        return c10::cuda::getCurrentCUDAStream(current).stream();
    }
};

// an uninitialised tensor beside `like`; straight from the CUDA allocator where that is on a GPU (the dispatcher's way there takes as long again)
at::Tensor empty(at::IntArrayRef shape, const at::Tensor& like, at::ScalarType type){
    if(like.is_cuda()) return at::detail::empty_cuda(shape, type, like.device(), c10::nullopt);
    return at::empty(shape, like.options().dtype(type));
}
at::Tensor workspace(size_t bytes, const at::Tensor& like, void** p){
    if(bytes == 0){ *p = nullptr; return {}; }
    at::Tensor t = empty({(int64_t)bytes}, like, at::kByte);
    *p = t.data_ptr();
    return t;
}
// the tensor that was given, or a new one; `made` keeps what is new alive and hands it out
struct Output {
    at::Tensor made;
    PyObject* given = nullptr;
    const at::Tensor* get() const { return given ? &THPVariable_Unpack(given) : made.defined() ? &made : nullptr; }
    PyObject* hand() const { return given ? (Py_INCREF(given), given) : made.defined() ? THPVariable_Wrap(made) : (Py_INCREF(Py_None), Py_None); }
};
Output output(const char* call, const char* name, PyObject* given, bool wanted, at::IntArrayRef shape, const at::Tensor& like, at::ScalarType type, bool zero = false){
    Output o;
    if(given != Py_None){ tensor(call, name, given); o.given = given; }
    else if(wanted) o.made = zero ? at::zeros(shape, like.options().dtype(type)) : empty(shape, like, type);
    return o;
}
void is_matrix(const char* call, const char* name, const at::Tensor* t){
    if(!t || t->dim() != 2) refuse(call, ": ", name, " has to be a matrix");
    if(t->size(0) > INT_MAX || t->size(1) > INT_MAX) refuse(call, ": ", name, " has more than 2^31 - 1 rows or columns");
}
int activation(const char* call, PyObject* o){
    const long a = PyLong_Check(o) ? PyLong_AsLong(o) : -1;
    if(a < B200RL_ACT_IDENTITY || a > B200RL_ACT_SILU) refuse(call, ": no such activation");
    return (int)a;
}
int norm(const char* call, PyObject* o){
    const long a = PyLong_Check(o) ? PyLong_AsLong(o) : -1;
    if(a < B200RL_NORM_NONE || a > B200RL_NORM_RMS) refuse(call, ": no such norm");
    return (int)a;
}
double number(const char* call, const char* name, PyObject* o){
    const double v = PyFloat_AsDouble(o);
    if(v == -1.0 && PyErr_Occurred()){ PyErr_Clear(); refuse(call, ": ", name, " is not a number"); }
    return v;
}
long long integer(const char* call, const char* name, PyObject* o){
    const long long v = PyLong_Check(o) ? PyLong_AsLongLong(o) : (PyErr_SetString(PyExc_TypeError, ""), -1);
    if(v == -1 && PyErr_Occurred()){ PyErr_Clear(); refuse(call, ": ", name, " is not a whole number"); }
    return v;
}
unsigned long long word(const char* call, const char* name, PyObject* o){       // modulo 2^64
    if(!PyLong_Check(o)) refuse(call, ": ", name, " is not a whole number");
    return PyLong_AsUnsignedLongLongMask(o);
}

// (W, x, act, bias, residual, scale, want_pre, y, pre) -> (pre, y)
PyObject* dense_residual_forward(PyObject* const* a){
    const char* call = "dense_residual_forward";
    const at::Tensor *W = tensor(call, "W", a[0]), *x = tensor(call, "x", a[1]);
    is_matrix(call, "x", x); is_matrix(call, "W", W);
    const int64_t B = x->size(0), I = x->size(1), O = W->size(0);
    if(I < 1 || O < 1) refuse(call, ": a layer has at least one input and one output");
    Operands o(call, *x, false);
    const int act = activation(call, a[2]);
    const Matrix mx = o.matrix("x", x, B, I), mw = o.matrix("W", W, O, I), mr = o.matrix("residual", tensor(call, "residual", a[4]), B, O);
    const float* bias = o.vector("bias", tensor(call, "bias", a[3]), O);
    const Output y = output(call, "y", a[7], true, {B, O}, *x, o.dtype), pre = output(call, "pre", a[8], a[6] == Py_True, {B, O}, *x, o.dtype);
    const Matrix my = o.matrix("y", y.get(), B, O), mp = o.matrix("pre", pre.get(), B, O);
    const float scale = (float)number(call, "scale", a[5]);
    void *stream = o.here(), *ws;
    const size_t n = E.dense_residual_forward_workspace_bytes(mw.p, mw.ld, mx.p, mx.ld, (int)B, (int)I, (int)O);
    const at::Tensor keep = workspace(n, *x, &ws);
    check(E.dense_residual_forward(o.type, mw.p, mw.ld, bias, mx.p, mx.ld, mr.p, mr.ld, scale, mp.p, mp.ld, my.p, my.ld, (int)B, (int)I, (int)O, act, ws, n, stream));
    return Py_BuildValue("NN", pre.hand(), y.hand());
}

// (pre, d_y, act, scale, d_pre) -> d_pre
PyObject* dense_residual_backward_activation(PyObject* const* a){
    const char* call = "dense_residual_backward_activation";
    const at::Tensor *pre = tensor(call, "pre", a[0]), *d_y = tensor(call, "d_y", a[1]);
    is_matrix(call, "d_y", d_y);
    const int64_t B = d_y->size(0), O = d_y->size(1);
    Operands o(call, *d_y, false);
    const int act = activation(call, a[2]);
    if(O < 1 || (!pre && act != B200RL_ACT_IDENTITY)) refuse(call, ": the slope needs the pre-activations, and rows at least one element");
    const Output out = output(call, "d_pre", a[4], true, {B, O}, *d_y, o.dtype);
    const Matrix md = o.matrix("d_y", d_y, B, O), mp = o.matrix("pre", pre, B, O), mo = o.matrix("d_pre", out.get(), B, O);
    const float scale = (float)number(call, "scale", a[3]);
    void* stream = o.here();
    check(E.dense_residual_backward_activation(o.type, mp.p, mp.ld, md.p, md.ld, scale, mo.p, mo.ld, (int)B, (int)O, act, stream));
    return out.hand();
}

// (W, x, d_pre, d_W, d_bias, add, pre_in, act_in, d_in, want_d_in, want_grads) -> (d_W, d_bias, d_in)
PyObject* dense_residual_backward(PyObject* const* a){
    const char* call = "dense_residual_backward";
    const at::Tensor *W = tensor(call, "W", a[0]), *x = tensor(call, "x", a[1]), *d = tensor(call, "d_pre", a[2]), *pre = tensor(call, "pre_in", a[6]);
    is_matrix(call, "d_pre", d); is_matrix(call, "W", W);
    const int64_t B = d->size(0), O = d->size(1), I = W->size(1);
    if(I < 1 || O < 1) refuse(call, ": a layer has at least one input and one output");
    const bool want_d_in = a[9] == Py_True, want_grads = a[10] == Py_True;
    Operands o(call, *d, false);
    const int act = activation(call, a[7]);
    const Matrix md = o.matrix("d_pre", d, B, O), mw = o.matrix("W", W, O, I);
    Matrix mx{}, ma{}, mp{}, mi{};
    Output d_W, d_bias, d_in;
    float *g_W = nullptr, *g_b = nullptr;
    bool given = false;
    if(want_grads){
        if(!x) refuse(call, ": the weights' gradient needs x");
        mx = o.matrix("x", x, B, I);
        given = a[3] != Py_None || a[4] != Py_None;
        d_W = output(call, "d_W", a[3], true, {O, I}, *d, at::kFloat, given);
        d_bias = output(call, "d_bias", a[4], true, {O}, *d, at::kFloat, given);
        const at::Tensor& t = *d_W.get();
        if(t.scalar_type() != at::kFloat || t.dim() != 2 || t.size(0) != O || t.size(1) != I || !t.is_contiguous()) refuse(call, ": d_W is not a dense [", O, ", ", I, "] float32 matrix");
        o.seen(t);
        g_W = static_cast<float*>(t.data_ptr());
        g_b = o.vector("d_bias", d_bias.get(), O);
    }
    if(want_d_in){
        if(act != B200RL_ACT_IDENTITY && !pre) refuse(call, ": the slope needs the pre-activations");
        ma = o.matrix("add", tensor(call, "add", a[5]), B, I);
        mp = o.matrix("pre_in", pre, B, I);
        d_in = output(call, "d_in", a[8], true, {B, I}, *d, o.dtype);
        mi = o.matrix("d_in", d_in.get(), B, I);
    }
    else if(a[8] != Py_None) d_in.given = a[8];
    void *stream = o.here(), *ws;
    // the weights first: d_in may lie over what only it reads, never over x or d_pre
    if(want_grads){
        const size_t n = E.dense_residual_backward_weights_workspace_bytes(mx.p, mx.ld, md.p, md.ld, g_W, (int)B, (int)I, (int)O);
        const at::Tensor keep = workspace(n, *d, &ws);
        check(E.dense_residual_backward_weights(o.type, mx.p, mx.ld, md.p, md.ld, g_W, g_b, given, (int)B, (int)I, (int)O, ws, n, stream));
    }
    if(want_d_in){
        const size_t n = E.dense_residual_backward_input_workspace_bytes(mw.p, mw.ld, md.p, md.ld, (int)B, (int)I, (int)O);
        const at::Tensor keep = workspace(n, *d, &ws);
        check(E.dense_residual_backward_input(o.type, mw.p, mw.ld, md.p, md.ld, ma.p, ma.ld, mp.p, mp.ld, act, mi.p, mi.ld, (int)B, (int)I, (int)O, ws, n, stream));
    }
    return Py_BuildValue("NNN", d_W.hand(), d_bias.hand(), d_in.hand());
}

int64_t gate_count(const char* call, const at::Tensor* gate, long long gate_rows, int64_t rows){
    if(!gate) return 0;
    if(rows == 0) return gate->dim() == 2 ? gate->size(0) : 0;      // no row looks at it
    if(gate_rows < 1 || gate_rows > INT_MAX) refuse(call, ": a gate row serves at least one row");
    return (rows - 1) / gate_rows + 1;
}
void check_dim(const char* call, int64_t D){
    if(D < 1 || D > B200RL_NORM_MAX_DIM) refuse(call, ": rows have 1 to ", B200RL_NORM_MAX_DIM, " elements, not ", D);
}

// (branch, residual, post, post_weight, post_bias, gate, gate_rows, scale, pre, pre_weight, pre_bias, epsilon, out, normed) -> (out, normed)
PyObject* norm_residual_forward(PyObject* const* a){
    const char* call = "norm_residual_forward";
    const at::Tensor *branch = tensor(call, "branch", a[0]), *residual = tensor(call, "residual", a[1]), *gate = tensor(call, "gate", a[5]), *first = branch ? branch : residual;
    if(!first) refuse(call, ": neither branch nor residual");
    is_matrix(call, branch ? "branch" : "residual", first);
    const int64_t R = first->size(0), D = first->size(1);
    Operands o(call, *first, true);
    const int post = norm(call, a[2]), pre = norm(call, a[8]);
    check_dim(call, D);
    if(!branch && (post || gate)) refuse(call, ": a norm or a gate of a branch that is not there");
    if((!post && (a[3] != Py_None || a[4] != Py_None)) || (!pre && (a[9] != Py_None || a[10] != Py_None || a[13] != Py_None)))
        refuse(call, ": a weight, bias or output of a norm that is not there");
    const long long gate_rows = integer(call, "gate_rows", a[6]);
    const Matrix mb = o.matrix("branch", branch, R, D), mr = o.matrix("residual", residual, R, D), mg = o.matrix("gate", gate, gate_count(call, gate, gate_rows, R), D);
    const float *pw = o.vector("post_weight", tensor(call, "post_weight", a[3]), D), *pb = o.vector("post_bias", tensor(call, "post_bias", a[4]), D);
    const float *nw = o.vector("pre_weight", tensor(call, "pre_weight", a[9]), D), *nb = o.vector("pre_bias", tensor(call, "pre_bias", a[10]), D);
    const Output out = output(call, "out", a[12], true, {R, D}, *first, o.dtype), normed = output(call, "normed", a[13], pre != 0, {R, D}, *first, o.dtype);
    const Matrix mo = o.matrix("out", out.get(), R, D), mn = o.matrix("normed", normed.get(), R, D);
    const float scale = (float)number(call, "scale", a[7]), epsilon = (float)number(call, "epsilon", a[11]);
    void* stream = o.here();
    if(R) check(E.norm_residual_forward(o.type, post, pw, pb, mb.p, mb.ld, mg.p, mg.ld, (int)gate_rows, scale, mr.p, mr.ld, mo.p, mo.ld, pre, nw, nb, mn.p, mn.ld, (int)R, (int)D, epsilon,
                                        stream));
    return Py_BuildValue("NN", out.hand(), normed.hand());
}

// (branch, out, d_out, d_normed, post, post_weight, post_bias, gate, gate_rows, scale, pre, pre_weight, pre_bias, epsilon, d_branch, d_residual, d_gate, d_post_weight, d_post_bias,
// d_pre_weight, d_pre_bias) -> dict
PyObject* norm_residual_backward(PyObject* const* a){
    const char* call = "norm_residual_backward";
    const at::Tensor *branch = tensor(call, "branch", a[0]), *out = tensor(call, "out", a[1]), *d_out = tensor(call, "d_out", a[2]), *d_normed = tensor(call, "d_normed", a[3]);
    const at::Tensor *gate = tensor(call, "gate", a[7]), *first = d_normed ? d_normed : d_out;
    if(!first) refuse(call, ": neither d_out nor d_normed");
    is_matrix(call, d_normed ? "d_normed" : "d_out", first);
    const int64_t R = first->size(0), D = first->size(1);
    Operands o(call, *first, true);
    const int post = norm(call, a[4]), pre = norm(call, a[10]);
    check_dim(call, D);
    if(!branch && (post || gate)) refuse(call, ": a norm or a gate of a branch that is not there");
    if((pre != 0) != (d_normed != nullptr) || (pre && !out)) refuse(call, ": d_normed and out go with the norm behind the sum");
    if((!post && (a[5] != Py_None || a[6] != Py_None)) || (!pre && (a[11] != Py_None || a[12] != Py_None))) refuse(call, ": a weight or bias of a norm that is not there");
    if((!branch && a[14] != Py_None) || (!gate && a[16] != Py_None)) refuse(call, ": the gradient of an operand that is not there");
    const long long gate_rows = integer(call, "gate_rows", a[8]);
    const int64_t G = gate_count(call, gate, gate_rows, R);
    const Matrix mb = o.matrix("branch", branch, R, D), mo = o.matrix("out", out, R, D), mdo = o.matrix("d_out", d_out, R, D), mdn = o.matrix("d_normed", d_normed, R, D);
    const Matrix mg = o.matrix("gate", gate, G, D);
    // the parameters that are there have gradients: accumulated onto when given
    static const char* const parameter[4] = {"post_weight", "post_bias", "pre_weight", "pre_bias"};
    static const char* const gradient[4] = {"d_post_weight", "d_post_bias", "d_pre_weight", "d_pre_bias"};
    PyObject* const params[4] = {a[5], a[6], a[11], a[12]};
    const float* p[4];
    bool given = false;
    for(int i = 0; i < 4; i++){
        p[i] = o.vector(parameter[i], tensor(call, parameter[i], params[i]), D);
        if(a[17 + i] != Py_None){
            if(!p[i] && params[i] == Py_None) refuse(call, ": ", gradient[i], " of a parameter that is not there");
            given = true;
        }
    }
    const Output d_branch = output(call, "d_branch", a[14], branch != nullptr, {R, D}, *first, o.dtype), d_residual = output(call, "d_residual", a[15], true, {R, D}, *first, o.dtype);
    const Output d_gate = output(call, "d_gate", a[16], gate != nullptr, {G, D}, *first, o.dtype);
    const Matrix mdb = o.matrix("d_branch", d_branch.get(), R, D), mdr = o.matrix("d_residual", d_residual.get(), R, D), mdg = o.matrix("d_gate", d_gate.get(), G, D);
    Output d_param[4];
    float* g[4];
    for(int i = 0; i < 4; i++){
        d_param[i] = output(call, gradient[i], a[17 + i], params[i] != Py_None, {D}, *first, at::kFloat, given);
        g[i] = o.vector(gradient[i], d_param[i].get(), D);
    }
    const float scale = (float)number(call, "scale", a[9]), epsilon = (float)number(call, "epsilon", a[13]);
    void *stream = o.here(), *ws;
    const size_t n = E.norm_residual_backward_scratch_bytes((int)R, (int)D);
    const at::Tensor keep = workspace(n, *first, &ws);
    if(R == 0 && d_gate.get()) d_gate.get()->zero_();               // sums over no rows; the C call takes a gate of an empty batch to have none
    check(E.norm_residual_backward(o.type, post, p[0], p[1], mb.p, mb.ld, mg.p, mg.ld, (int)gate_rows, scale, mo.p, mo.ld, pre, p[2], mdo.p, mdo.ld, mdn.p, mdn.ld, mdb.p, mdb.ld, mdr.p,
                                   mdr.ld, mdg.p, mdg.ld, g[0], g[1], g[2], g[3], given, (int)R, (int)D, epsilon, ws, n, stream));
    return Py_BuildValue("{sNsNsNsNsNsNsN}", "d_branch", d_branch.hand(), "d_residual", d_residual.hand(), "d_gate", d_gate.hand(), gradient[0], d_param[0].hand(), gradient[1],
                         d_param[1].hand(), gradient[2], d_param[2].hand(), gradient[3], d_param[3].hand());
}

// (x, p, seed, stream_id, call_index, call_counter, residual, y) -> y
PyObject* dropout(PyObject* const* a){
    const char* call = "dropout";
    const at::Tensor *x = tensor(call, "x", a[0]), *counter = tensor(call, "call_counter", a[5]);
    is_matrix(call, "x", x);
    const int64_t R = x->size(0), D = x->size(1);
    Operands o(call, *x, true);
    const double p = number(call, "p", a[1]);
    const long long stream_id = integer(call, "stream_id", a[3]);
    if(D < 1 || !(p >= 0.0 && p <= 1.0) || stream_id < 0 || stream_id >= 65536) refuse(call, ": rows of at least one element, 0 <= p <= 1, 0 <= stream_id < 65536");
    const unsigned long long seed = word(call, "seed", a[2]), index = word(call, "call_index", a[4]);
    const Output y = output(call, "y", a[7], true, {R, D}, *x, o.dtype);
    const Matrix mx = o.matrix("x", x, R, D), mr = o.matrix("residual", tensor(call, "residual", a[6]), R, D), my = o.matrix("y", y.get(), R, D);
    if(counter){
        if(counter->scalar_type() != at::kLong || counter->numel() != 1) refuse(call, ": call_counter is one int64 value");
        o.seen(*counter);
    }
    void* stream = o.here();
    check(E.dropout(o.type, mx.p, mx.ld, mr.p, mr.ld, my.p, my.ld, (int)R, (int)D, (float)p, seed, (unsigned)stream_id, index,
                    counter ? static_cast<const unsigned long long*>(counter->data_ptr()) : nullptr, stream));
    return y.hand();
}

// nothing leaves a call but a result or a Python exception
template <PyObject* (*F)(PyObject* const*), int N> PyObject* guarded(PyObject*, PyObject* const* args, Py_ssize_t n){
    if(n != N){ PyErr_Format(PyExc_TypeError, "%d arguments, got %zd", N, n); return nullptr; }
    if(!E.dropout){ PyErr_SetString(PyExc_RuntimeError, "the C entry points are not bound"); return nullptr; }
    try { return F(args); }
    catch(const Refusal& r){ PyErr_SetString(g_refusal, r.what.c_str()); }
    catch(const Status& s){ PyErr_SetObject(g_status, PyLong_FromLong(s.status)); }
    catch(...){ torch::translate_exception_to_python(std::current_exception()); }       // torch's own: out of memory stays torch.OutOfMemoryError
    return nullptr;
}

// addresses of the C entry points, in the order of `Entries`
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n){
    constexpr Py_ssize_t count = sizeof(Entries) / sizeof(void*);
    if(n != count){ PyErr_Format(PyExc_TypeError, "%zd addresses, got %zd", count, n); return nullptr; }
    void* p[count];
    for(Py_ssize_t i = 0; i < n; i++){
        p[i] = PyLong_AsVoidPtr(args[i]);
        if(!p[i]){ if(!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "an address of 0"); return nullptr; }
    }
    memcpy(static_cast<void*>(&E), p, sizeof(E));
    Py_RETURN_NONE;
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f))
PyMethodDef methods[] = {
    {"bind", FAST(bind), METH_FASTCALL, nullptr},
    {"dense_residual_forward", FAST((guarded<dense_residual_forward, 9>)), METH_FASTCALL, nullptr},
    {"dense_residual_backward_activation", FAST((guarded<dense_residual_backward_activation, 5>)), METH_FASTCALL, nullptr},
    {"dense_residual_backward", FAST((guarded<dense_residual_backward, 11>)), METH_FASTCALL, nullptr},
    {"norm_residual_forward", FAST((guarded<norm_residual_forward, 14>)), METH_FASTCALL, nullptr},
    {"norm_residual_backward", FAST((guarded<norm_residual_backward, 21>)), METH_FASTCALL, nullptr},
    {"dropout", FAST((guarded<dropout, 8>)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensors", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensors(){
    PyObject* m = PyModule_Create(&module);
    if(!m) return nullptr;
    if(!g_refusal) g_refusal = PyErr_NewException("b200rl.Refusal", nullptr, nullptr);
    if(!g_status) g_status = PyErr_NewException("b200rl.Status", nullptr, nullptr);
    if(!g_refusal || !g_status || PyModule_AddObjectRef(m, "Refusal", g_refusal) < 0 || PyModule_AddObjectRef(m, "Status", g_status) < 0){ Py_DECREF(m); return nullptr; }
    return m;
}
