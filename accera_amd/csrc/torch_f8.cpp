// The 8-bit feed-forward operators on torch tensors: argument checks, allocation of results and the call of the C entry point
// (include/accera_mi355x_f8.h) in one step from Python.  The smallest calls are bound by the host: quantising 8 x 4096 took 8.0 us a call with
// the same steps in Python, of which the launch is 2.9.
//
// Functions take their arguments by position (accera_amd/f8.py gives them names); a stream is None, for the device's current one, or a raw hipStream_t.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/StreamGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/accera_mi355x_f8.h"

namespace {

using at::Tensor;

constexpr at::ScalarType F8 = at::kFloat8_e4m3fn;
int64_t blocks_of(int64_t n) { return (n + ACC950_F8_BLOCK - 1) / ACC950_F8_BLOCK; }
void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

std::string name_of(at::ScalarType t)
{
    switch (t) {
    case at::kFloat: return "torch.float32";
    case at::kDouble: return "torch.float64";
    case at::kHalf: return "torch.float16";
    case at::kBFloat16: return "torch.bfloat16";
    case at::kFloat8_e4m3fn: return "torch.float8_e4m3fn";
    case at::kByte: return "torch.uint8";
    case at::kInt: return "torch.int32";
    case at::kLong: return "torch.int64";
    default: return c10::toString(t);
    }
}

std::string shape_of(at::IntArrayRef s)
{
    std::string text = "(";
    for (size_t i = 0; i < s.size(); ++i) text += (i ? ", " : "") + std::to_string(s[i]);
    return text + (s.size() == 1 ? ",)" : ")");
}

#define REFUSE_IF(condition, ...) TORCH_CHECK_VALUE(!(condition), __VA_ARGS__)

int64_t float_type(const Tensor& t, const char* name)
{
    switch (t.scalar_type()) {
    case at::kFloat: return ACC950_F32;
    case at::kHalf: return ACC950_F16;
    case at::kBFloat16: return ACC950_BF16;
    default: TORCH_CHECK_VALUE(false, name, " must be fp32, fp16 or bf16, not ", name_of(t.scalar_type()));
    }
}

void fits(const Tensor& t, at::IntArrayRef shape, at::ScalarType type, const char* name)
{
    REFUSE_IF(t.scalar_type() != type || t.sizes() != shape, name, " must be ", name_of(type), " of shape ", shape_of(shape), ", not ", name_of(t.scalar_type()), " of ",
              shape_of(t.sizes()));
}

void is_matrix(const Tensor& t, const char* name) { REFUSE_IF(t.dim() != 2, name, " must be 2-D"); }
void rows_contiguous(const Tensor& t, const char* name) { REFUSE_IF(t.size(1) > 1 && t.stride(1) != 1, name, " must be contiguous along its last axis"); }
void contiguous(const Tensor& t, const char* name) { REFUSE_IF(!t.is_contiguous(), name, " must be contiguous"); }

// ---- arguments from Python

const Tensor& tensor(PyObject* o, const char* name)
{
    TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a tensor");
    return THPVariable_Unpack(o);
}
Tensor maybe_tensor(PyObject* o, const char* name) { return o == Py_None ? Tensor() : tensor(o, name); }
int64_t integer(PyObject* o)
{
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
}
double real(PyObject* o)
{
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return v;
}
bool flag(PyObject* o)
{
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw python_error();
    return v != 0;
}

// The one GPU of a call's tensors and the stream that the call goes to, both made current for the call.
// What it allocates is memory of that stream: of a given one too, for a block that was freed a moment ago on the caller's current stream may have work
// pending there, which the given stream does not wait for.  Scratch memory is done with when the stream is, and nothing else uses it.  A result that the caller
// may also use on the stream that was current (having made it wait) is noted as used there, so that it is not handed on before that one is done either.
struct Place {
    c10::OptionalDeviceGuard device_guard;
    c10::OptionalStreamGuard stream_guard;
    c10::Device device;
    std::optional<c10::Stream> current; // the caller's, where another one was given
    void* stream;
    Place(PyObject* given, const Tensor& first, std::initializer_list<const Tensor*> others) : device(first.device()), stream(nullptr)
    {
        REFUSE_IF(!first.is_cuda(), "tensors must live on the GPU (there is no CPU path)");
        for (const Tensor* t : others) REFUSE_IF(t->defined() && t->device() != device, "tensors must live on one GPU");
        device_guard.reset_device(device);
        // (torch on ROCm calls the GPU a CUDA device, in its streams too)
        const auto now = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(device.index());
        stream = now.stream();
        if (given == Py_None) return;
        void* const other = PyLong_AsVoidPtr(given);
        if (!other && PyErr_Occurred()) throw python_error();
        if (other == stream) return;
        stream = other;
        current = now.unwrap();
        stream_guard.reset_stream(other ? c10::hip::getStreamFromExternalMasqueradingAsCUDA((hipStream_t)other, device.index()).unwrap()
                                        : c10::hip::getDefaultHIPStreamMasqueradingAsCUDA(device.index()).unwrap());
    }
    Tensor scratch(at::IntArrayRef shape, at::ScalarType type) const { return at::empty(shape, at::TensorOptions().dtype(type).device(device)); }
    Tensor result(Tensor t) const
    {
        if (current) t.record_stream(*current);
        return t;
    }
    Tensor result(at::IntArrayRef shape, at::ScalarType type) const { return result(scratch(shape, type)); }
};

// an entry point's status as the exception that the rest of the package raises
void check(int rc)
{
    if (rc == ACC950_OK) return;
    PyObject* module = PyImport_ImportModule("accera_amd._lib");
    PyObject* done = module ? PyObject_CallMethod(module, "check", "i", rc) : nullptr;
    Py_XDECREF(module);
    if (done) { // (it raises)
        Py_DECREF(done);
        PyErr_SetString(PyExc_RuntimeError, "an entry point failed");
    }
    throw python_error();
}

PyObject* wrap(const Tensor& t) { return THPVariable_Wrap(t); }
PyObject* pair(const Tensor& a, const Tensor& b)
{
    PyObject *x = wrap(a), *y = wrap(b);
    PyObject* both = x && y ? PyTuple_Pack(2, x, y) : nullptr;
    Py_XDECREF(x);
    Py_XDECREF(y);
    return both;
}

// ---- operators

// (x, out, scale, group_rows, transpose, activation, power_of_two, stream) -> (q, scale)
PyObject* quantize(PyObject* const* a)
{
    const Tensor& x = tensor(a[0], "x");
    Tensor q = maybe_tensor(a[1], "out"), scale = maybe_tensor(a[2], "scale");
    acc950_f8_quantize_call c{};
    c.group_rows = integer(a[3]);
    c.transpose = flag(a[4]);
    c.activation = integer(a[5]);
    c.power_of_two = flag(a[6]);
    is_matrix(x, "x");
    REFUSE_IF(c.group_rows != 1 && c.group_rows != ACC950_F8_BLOCK, "group_rows must be 1 or 128");
    c.in_type = float_type(x, "x");
    c.rows = x.size(0);
    c.cols = x.size(1);
    if (c.activation == ACC950_ACT_SILU_MUL) {
        REFUSE_IF(c.cols % 2, "silu_mul takes an even number of columns: gate and up");
        c.cols /= 2;
    }
    const Place place(a[7], x, {&q, &scale});
    const int64_t rows = c.transpose ? c.cols : c.rows, cols = c.transpose ? c.rows : c.cols;
    const int64_t groups = (rows + c.group_rows - 1) / c.group_rows, blocks = blocks_of(cols);
    if (!q.defined()) {
        const int64_t pitch = (cols + 15) / 16 * 16; // (rows that the product can fetch 16 bytes at a time)
        q = place.result({rows, pitch}, F8);
        if (pitch != cols) q = q.narrow(1, 0, cols);
    } else {
        fits(q, {rows, cols}, F8, "out");
        rows_contiguous(q, "out");
    }
    if (!scale.defined()) {
        const int64_t strides[2] = {c.group_rows == 1 ? 1 : blocks, c.group_rows == 1 ? groups : 1};
        scale = place.result(at::empty_strided({groups, blocks}, strides, at::TensorOptions().dtype(at::kFloat).device(place.device)));
    } else fits(scale, {groups, blocks}, at::kFloat, "scale");
    c.x = data(x); c.x_row_stride = x.stride(0); c.x_col_stride = x.stride(1);
    c.q = data(q); c.q_row_stride = q.stride(0);
    c.scale = data(scale); c.s_row_stride = scale.stride(0); c.s_block_stride = scale.stride(1);
    c.stream = place.stream;
    check(acc950_f8_quantize(&c));
    return pair(q, scale);
}

// (A, a_scale, B, b_scale, C, epilogue, variant, k_slices, stream)
PyObject* gemm(PyObject* const* a)
{
    const Tensor &A = tensor(a[0], "A"), &a_scale = tensor(a[1], "a_scale"), &B = tensor(a[2], "B"), &b_scale = tensor(a[3], "b_scale"), &C = tensor(a[4], "C");
    is_matrix(A, "A"); is_matrix(B, "B"); is_matrix(C, "C");
    acc950_f8_gemm_call c{};
    c.M = A.size(0); c.K = A.size(1); c.N = B.size(1);
    REFUSE_IF(B.size(0) != c.K || C.size(0) != c.M || C.size(1) != c.N, "shape mismatch: A ", shape_of(A.sizes()), ", B ", shape_of(B.sizes()), ", C ", shape_of(C.sizes()));
    REFUSE_IF(A.scalar_type() != F8 || B.scalar_type() != F8, "unsupported dtypes ", name_of(A.scalar_type()), ", ", name_of(B.scalar_type()), ": gemm_f8 takes ", name_of(F8));
    c.out_type = float_type(C, "C");
    const int64_t blocks = blocks_of(c.K);
    fits(a_scale, {c.M, blocks}, at::kFloat, "a_scale");
    c.group_cols = b_scale.dim() == 2 && b_scale.size(0) == blocks && b_scale.size(1) == c.N ? 1 : ACC950_F8_BLOCK;
    fits(b_scale, {blocks, c.group_cols == 1 ? c.N : blocks_of(c.N)}, at::kFloat, "b_scale");
    c.epilogue = integer(a[5]);
    c.variant = integer(a[6]);
    c.k_slices = integer(a[7]);
    const Place place(a[8], A, {&a_scale, &B, &b_scale, &C});
    c.A = data(A); c.a_row_stride = A.stride(0); c.a_col_stride = A.stride(1);
    c.a_scale = data(a_scale); c.as_row_stride = a_scale.stride(0); c.as_block_stride = a_scale.stride(1);
    c.B = data(B); c.b_row_stride = B.stride(0); c.b_col_stride = B.stride(1);
    c.b_scale = data(b_scale); c.bs_block_stride = b_scale.stride(0); c.bs_col_stride = b_scale.stride(1);
    c.C = data(C); c.c_row_stride = C.stride(0); c.c_col_stride = C.stride(1);
    c.workspace_bytes = std::max<int64_t>(acc950_f8_gemm_workspace(&c), 0); // (negative: the call refuses and says why)
    Tensor workspace;
    if (c.workspace_bytes) workspace = place.scratch({c.workspace_bytes}, at::kByte);
    c.workspace = data(workspace);
    c.stream = place.stream;
    check(acc950_f8_gemm(&c));
    Py_RETURN_NONE;
}

// (logits, top_k, score, bias, groups, top_groups or None, group_score, renormalise, scale, stream) -> (ids, weights)
PyObject* route(PyObject* const* a)
{
    const Tensor& logits = tensor(a[0], "logits");
    const Tensor bias = maybe_tensor(a[3], "bias");
    is_matrix(logits, "logits");
    acc950_route_call c{};
    c.in_type = float_type(logits, "logits");
    c.tokens = logits.size(0); c.experts = logits.size(1);
    c.top_k = integer(a[1]);
    c.score = integer(a[2]);
    c.groups = integer(a[4]);
    c.top_groups = a[5] == Py_None ? c.groups : integer(a[5]);
    c.group_score = integer(a[6]);
    c.renormalise = flag(a[7]);
    c.route_scale = real(a[8]);
    rows_contiguous(logits, "logits");
    REFUSE_IF(c.top_k < 0, "top_k must not be negative");
    if (bias.defined()) {
        fits(bias, {c.experts}, at::kFloat, "bias");
        contiguous(bias, "bias");
    }
    const Place place(a[9], logits, {&bias});
    if (c.top_k > c.experts) check(acc950_route(&c)); // (refused, before memory is taken for it)
    const Tensor ids = place.result({c.tokens, c.top_k}, at::kInt), weights = place.result({c.tokens, c.top_k}, at::kFloat);
    c.logits = data(logits); c.l_row_stride = logits.stride(0);
    c.bias = data(bias); c.ids = data(ids); c.weights = data(weights);
    c.stream = place.stream;
    check(acc950_route(&c));
    return pair(ids, weights);
}

// (logits, ids, dweights, score, renormalise, scale, out, stream) -> out
PyObject* route_backward(PyObject* const* a)
{
    const Tensor &logits = tensor(a[0], "logits"), &ids = tensor(a[1], "ids"), &dweights = tensor(a[2], "dweights");
    Tensor out = maybe_tensor(a[6], "out");
    is_matrix(logits, "logits");
    acc950_route_backward_call c{};
    c.in_type = float_type(logits, "logits");
    c.tokens = logits.size(0); c.experts = logits.size(1);
    rows_contiguous(logits, "logits");
    c.top_k = ids.dim() ? ids.size(-1) : 0;
    fits(ids, {c.tokens, c.top_k}, at::kInt, "ids");
    fits(dweights, {c.tokens, c.top_k}, at::kFloat, "dweights");
    REFUSE_IF(!ids.is_contiguous() || !dweights.is_contiguous(), "ids and dweights must be contiguous");
    c.score = integer(a[3]);
    c.renormalise = flag(a[4]);
    c.route_scale = real(a[5]);
    const Place place(a[7], logits, {&ids, &dweights, &out});
    if (!out.defined()) out = place.result({c.tokens, c.experts}, logits.scalar_type());
    else {
        fits(out, {c.tokens, c.experts}, logits.scalar_type(), "out");
        rows_contiguous(out, "out");
    }
    c.logits = data(logits); c.l_row_stride = logits.stride(0);
    c.ids = data(ids); c.dweights = data(dweights);
    c.dlogits = data(out); c.grad_row_stride = out.stride(0);
    c.stream = place.stream;
    check(acc950_route_backward(&c));
    return wrap(out);
}

// A plan in one tensor: order (pairs), position (pairs), offsets (experts + 1), scratch memory.
// (ids, experts, stream) -> that
PyObject* plan(PyObject* const* a)
{
    const Tensor& ids = tensor(a[0], "ids");
    is_matrix(ids, "ids");
    REFUSE_IF(ids.scalar_type() != at::kInt || !ids.is_contiguous(), "ids must be contiguous int32");
    acc950_expert_plan_call c{};
    c.tokens = ids.size(0); c.top_k = ids.size(1);
    c.experts = integer(a[1]);
    const Place place(a[2], ids, {});
    const int64_t pairs = c.tokens * c.top_k, need = acc950_expert_plan_workspace(c.tokens, c.top_k, c.experts);
    if (need < 0) check(acc950_expert_plan(&c)); // (refused, before memory is taken for it)
    const Tensor all = place.result({2 * pairs + c.experts + 1 + need / 4}, at::kInt);
    int* at = (int*)data(all);
    c.ids = data(ids); c.order = at; c.position = at + pairs; c.offsets = at + 2 * pairs;
    c.workspace = at + 2 * pairs + c.experts + 1;
    c.stream = place.stream;
    check(acc950_expert_plan_within(&c, need));
    return wrap(all);
}

// (A, a_scale, B, b_scale, plan's tensor, tokens, top_k, experts, C, gather, row_weights, variant, stream)
PyObject* expert_gemm(PyObject* const* a)
{
    const Tensor &A = tensor(a[0], "A"), &a_scale = tensor(a[1], "a_scale"), &B = tensor(a[2], "B"), &b_scale = tensor(a[3], "b_scale"), &all = tensor(a[4], "plan"), &C = tensor(a[8], "C");
    const Tensor row_weights = maybe_tensor(a[10], "row_weights");
    const int64_t tokens = integer(a[5]), top_k = integer(a[6]), pairs = tokens * top_k, planned = integer(a[7]);
    const bool gather = flag(a[9]);
    REFUSE_IF(A.dim() != 2 || B.dim() != 3 || C.dim() != 2, "A and C must be 2-D, B 3-D");
    acc950_f8_expert_gemm_call c{};
    c.rows = pairs; c.top_k = top_k; c.experts = B.size(0); c.K = B.size(1); c.N = B.size(2); c.gather = gather;
    REFUSE_IF(A.scalar_type() != F8 || B.scalar_type() != F8, "unsupported dtypes ", name_of(A.scalar_type()), ", ", name_of(B.scalar_type()), ": expert_gemm_f8 takes ", name_of(F8));
    REFUSE_IF(c.experts != planned || A.size(0) != (gather ? tokens : pairs) || A.size(1) != c.K || C.size(0) != pairs || C.size(1) != c.N, "shape mismatch: A ", shape_of(A.sizes()),
              ", B ", shape_of(B.sizes()), ", C ", shape_of(C.sizes()), " for ", tokens, " tokens of ", planned, " experts, ", top_k, " each");
    c.out_type = float_type(C, "C");
    fits(a_scale, {A.size(0), blocks_of(c.K)}, at::kFloat, "a_scale");
    fits(b_scale, {c.experts, blocks_of(c.K), blocks_of(c.N)}, at::kFloat, "b_scale");
    REFUSE_IF((c.K > 1 && (A.stride(1) != 1 || B.stride(1) != 1)) || (c.N > 1 && C.stride(1) != 1), "A and B must be contiguous along K, C along its last axis");
    if (row_weights.defined()) {
        fits(row_weights, {tokens, top_k}, at::kFloat, "row_weights");
        contiguous(row_weights, "row_weights");
    }
    c.variant = integer(a[11]);
    const Place place(a[12], A, {&a_scale, &B, &b_scale, &C, &all, &row_weights});
    const int* at = (const int*)data(all);
    c.order = at; c.offsets = at + 2 * pairs;
    c.A = data(A); c.a_row_stride = A.stride(0);
    c.a_scale = data(a_scale); c.as_row_stride = a_scale.stride(0); c.as_block_stride = a_scale.stride(1);
    c.B = data(B); c.b_expert_stride = B.stride(0); c.b_col_stride = B.stride(2);
    c.b_scale = data(b_scale); c.bs_expert_stride = b_scale.stride(0); c.bs_block_stride = b_scale.stride(1); c.bs_col_stride = b_scale.stride(2);
    c.row_weights = data(row_weights);
    c.C = data(C); c.c_row_stride = C.stride(0);
    c.stream = place.stream;
    check(acc950_f8_expert_gemm(&c));
    Py_RETURN_NONE;
}

// (x, plan's tensor, tokens, top_k, weights, out, stream) -> out
PyObject* combine(PyObject* const* a)
{
    const Tensor &x = tensor(a[0], "x"), &all = tensor(a[1], "plan");
    const Tensor weights = maybe_tensor(a[4], "weights");
    Tensor out = maybe_tensor(a[5], "out");
    acc950_expert_combine_call c{};
    c.tokens = integer(a[2]); c.top_k = integer(a[3]);
    const int64_t pairs = c.tokens * c.top_k;
    c.type = float_type(x, "x");
    REFUSE_IF(x.dim() != 2 || x.size(0) != pairs, "x must have ", pairs, " rows");
    c.cols = x.size(1);
    if (weights.defined()) {
        fits(weights, {c.tokens, c.top_k}, at::kFloat, "weights");
        contiguous(weights, "weights");
    }
    const Place place(a[6], x, {&all, &weights, &out});
    if (!out.defined()) out = place.result({c.tokens, c.cols}, x.scalar_type());
    else fits(out, {c.tokens, c.cols}, x.scalar_type(), "out");
    REFUSE_IF(c.cols > 1 && (x.stride(1) != 1 || out.stride(1) != 1), "x and out must be contiguous along their last axis");
    c.x = data(x); c.x_row_stride = x.stride(0);
    c.position = (const int*)data(all) + pairs;
    c.weights = data(weights);
    c.y = data(out); c.y_row_stride = out.stride(0);
    c.stream = place.stream;
    check(acc950_expert_combine(&c));
    return wrap(out);
}

// (x, ids, weights, w13, w13_scale, w2, w2_scale, out, workspace, stream) -> out
PyObject* expert_ffn(PyObject* const* a)
{
    const Tensor &x = tensor(a[0], "x"), &ids = tensor(a[1], "ids"), &weights = tensor(a[2], "weights"), &w13 = tensor(a[3], "w13"), &w13_scale = tensor(a[4], "w13_scale"),
                 &w2 = tensor(a[5], "w2"), &w2_scale = tensor(a[6], "w2_scale");
    Tensor out = maybe_tensor(a[7], "out"), workspace = maybe_tensor(a[8], "workspace");
    is_matrix(x, "x");
    REFUSE_IF(w13.dim() != 4 || ids.dim() != 2, "w13 must be 4-D, ids 2-D");
    acc950_f8_expert_ffn_call c{};
    c.type = float_type(x, "x");
    c.tokens = x.size(0); c.hidden = x.size(1); c.experts = w13.size(0); c.inner = w13.size(2); c.top_k = ids.size(1);
    fits(w13, {c.experts, 2, c.inner, c.hidden}, F8, "w13");
    fits(w2, {c.experts, c.hidden, c.inner}, F8, "w2");
    fits(w13_scale, {c.experts, 2, blocks_of(c.inner), blocks_of(c.hidden)}, at::kFloat, "w13_scale");
    fits(w2_scale, {c.experts, blocks_of(c.hidden), blocks_of(c.inner)}, at::kFloat, "w2_scale");
    fits(ids, {c.tokens, c.top_k}, at::kInt, "ids");
    fits(weights, {c.tokens, c.top_k}, at::kFloat, "weights");
    REFUSE_IF(!w13.is_contiguous() || !w2.is_contiguous() || !w13_scale.is_contiguous() || !w2_scale.is_contiguous() || !ids.is_contiguous() || !weights.is_contiguous(),
              "weights, their scales, ids and routing weights must be contiguous");
    const Place place(a[9], x, {&ids, &weights, &w13, &w13_scale, &w2, &w2_scale, &out, &workspace});
    if (!out.defined()) out = place.result({c.tokens, c.hidden}, x.scalar_type());
    else fits(out, {c.tokens, c.hidden}, x.scalar_type(), "out");
    REFUSE_IF(c.hidden > 1 && (x.stride(1) != 1 || out.stride(1) != 1), "x and out must be contiguous along their last axis");
    const int64_t need = acc950_f8_expert_ffn_workspace(c.tokens, c.hidden, c.inner, c.experts, c.top_k);
    if (!workspace.defined()) workspace = place.scratch({std::max<int64_t>(need, 1)}, at::kByte);
    else REFUSE_IF(workspace.scalar_type() != at::kByte || !workspace.is_contiguous() || workspace.numel() < need, "workspace must be a contiguous uint8 tensor of at least ", need,
                   " elements");
    c.x = data(x); c.x_row_stride = x.stride(0);
    c.ids = data(ids); c.weights = data(weights);
    c.w13 = data(w13); c.w13_scale = data(w13_scale); c.w2 = data(w2); c.w2_scale = data(w2_scale);
    c.y = data(out); c.y_row_stride = out.stride(0);
    c.workspace = data(workspace);
    c.stream = place.stream;
    check(acc950_f8_expert_ffn_within(&c, workspace.numel()));
    return wrap(out);
}

template <PyObject* (*RUN)(PyObject* const*), int COUNT>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t count)
{
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(count == COUNT, "takes ", COUNT, " arguments, not ", count);
    return RUN(args);
    END_HANDLE_TH_ERRORS
}

#define ENTRY(name, count) {#name, (PyCFunction)(void (*)(void))entry<name, count>, METH_FASTCALL, nullptr}
PyMethodDef entries[] = {ENTRY(quantize, 8),    ENTRY(gemm, 9),    ENTRY(route, 10),      ENTRY(route_backward, 8), ENTRY(plan, 3),
                         ENTRY(expert_gemm, 13), ENTRY(combine, 7), ENTRY(expert_ffn, 10), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_torch_f8", nullptr, -1, entries, nullptr, nullptr, nullptr, nullptr};

} // namespace

PyMODINIT_FUNC PyInit__torch_f8() { return PyModule_Create(&module_def); }
