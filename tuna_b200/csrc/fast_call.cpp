// The argument checks and the launch of `ops.matmul` and of the operators of mx.py and fp8.py in one native call.  In Python they take
// 8 us of host time, more than the kernel of a small layer (4096x4096 at 1 token 6.8 us), so a decode step's small GEMMs waited
// for the host.
//
// matmul(x, q, s, c, o, m, n, k) answers True when the GEMM was launched and False when anything is not as the
// common case has it - a wrong type, device, layout or size, no workspace yet, one too small.  Nothing has been launched
// then, and ops.py takes the call through its own checks, which raise what is wrong.  Any other status of the
// library is the answer itself: a call of several launches may have made some of them, and is not made again.
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/cuda/CUDAFunctions.h>
#include "../../include/tuna_b200.h"

namespace {

using MatmulFn = int (*)(const void *q, const void *x, const void *code, const void *absmax, void *o, int m, int n, int k, void *workspace,
                         size_t workspace_bytes, void *stream);

MatmulFn g_matmul = nullptr;
PyObject *g_workspaces = nullptr;  // the dict (device, stream) -> tensor that ops.py fills: there is no other record of them

// The workspace of a device and stream, with a reference of the caller's own: another thread may put a larger one in its
// place while this one is in use.  Null where there is none.
struct Workspace {
    PyObject *tensor = nullptr;
    Workspace(int device, void *stream)
    {
        PyObject *key = Py_BuildValue("(iK)", device, (unsigned long long)stream);
        PyObject *found = key ? PyDict_GetItemWithError(g_workspaces, key) : nullptr;
        Py_XDECREF(key);
        if (found && THPVariable_Check(found)) tensor = Py_NewRef(found);
        PyErr_Clear();
    }
    ~Workspace() { Py_XDECREF(tensor); }
    Workspace(const Workspace &) = delete;
    Workspace &operator=(const Workspace &) = delete;
    void *ptr() const { return THPVariable_Unpack(tensor).mutable_data_ptr(); }
    size_t bytes() const { return THPVariable_Unpack(tensor).nbytes(); }
};

// The interpreter lock is released for this object's life: a launch waits where the stream's queue is full, and other
// threads - one of which may be what the stream waits for - have to run meanwhile.
struct Unlocked {
    PyThreadState *state = PyEval_SaveThread();
    ~Unlocked() { PyEval_RestoreThread(state); }
};

// The tensor of `o` if it is a plain contiguous CUDA tensor of `numel` elements of `type` on `device` (-1: any), else null.
const at::Tensor *plain(PyObject *o, at::ScalarType type, int64_t numel, int device)
{
    if (!THPVariable_CheckExact(o)) return nullptr;  // subclasses take the Python way
    const at::Tensor &t = THPVariable_Unpack(o);
    if (!t.defined() || !t.is_cuda() || t.scalar_type() != type || t.layout() != at::kStrided || t.numel() != numel || !t.is_contiguous()) return nullptr;
    if (device >= 0 && t.get_device() != device) return nullptr;
    return &t;
}

constexpr int kPythonWay = 1;  // no status of the library: those are negative or TUNA_OK

int launch(PyObject *const *args)
{
    long long dim[3];
    for (int i = 0; i < 3; ++i) {
        if (!PyLong_CheckExact(args[5 + i])) return kPythonWay;
        int overflow = 0;
        dim[i] = PyLong_AsLongLongAndOverflow(args[5 + i], &overflow);
        if (overflow || dim[i] <= 0 || dim[i] > 0x7fffffff) return kPythonWay;
    }
    const long long m = dim[0], n = dim[1], k = dim[2];
    const at::Tensor *x = plain(args[0], at::kHalf, n * k, -1);
    if (!x) return kPythonWay;
    const int device = x->get_device();
    const at::Tensor *q = plain(args[1], at::kByte, m * k / 2, device), *s = plain(args[2], at::kFloat, m, device),
                     *c = plain(args[3], at::kFloat, 16, device), *o = plain(args[4], at::kHalf, n * m, device);
    if (!q || !s || !c || !o || device != c10::cuda::current_device()) return kPythonWay;
    void *stream = c10::cuda::getCurrentCUDAStream(device).stream();
    const Workspace ws(device, stream);
    if (!ws.tensor) return kPythonWay;
    const void *qp = q->const_data_ptr(), *xp = x->const_data_ptr(), *cp = c->const_data_ptr(), *sp = s->const_data_ptr();
    void *op = o->mutable_data_ptr(), *wp = ws.ptr();
    const size_t bytes = ws.bytes();
    const MatmulFn matmul = g_matmul;
    const Unlocked unlocked;  // the caller's arguments and `ws` keep the tensors
    const int st = matmul(qp, xp, cp, sp, op, (int)m, (int)n, (int)k, wp, bytes, stream);
    return st == TUNA_ERR_WORKSPACE ? kPythonWay : st;
}

// ---- the microscaled operators (mx.py): the same answers

struct {
    int (*quantize)(const void *x, int x_type, long long row_stride, void *q, void *s, int rows, int k, int batch, void *stream);
    int (*dequant)(const void *q, const void *s, void *o, int o_type, int rows, int k, int batch, void *stream);
    int (*matmul)(const void *x, int x_type, const void *xs, const void *q, const void *s, void *o, int o_type, int m, int n, int k, void *workspace,
                  size_t workspace_bytes, void *stream);
    int (*matmul_grouped)(const void *x, int x_type, const void *xs, const void *q, const void *s, const void *offsets, void *o, int o_type, int m, int n, int k,
                          int experts, void *workspace, size_t workspace_bytes, void *stream);
    size_t (*workspace_bytes)(int m, int n, int k, int experts, int x_type);
} g_mx = {};

int type_of(at::ScalarType t) { return t == at::kHalf ? TUNA_FP16 : t == at::kBFloat16 ? TUNA_BF16 : t == at::kFloat ? TUNA_FP32 : -1; }

// A size argument: positive and of 32 bits, else 0.
long long size_of(PyObject *o)
{
    if (!PyLong_CheckExact(o)) return 0;
    int overflow = 0;
    const long long v = PyLong_AsLongLongAndOverflow(o, &overflow);
    return overflow || v <= 0 || v > 0x7fffffff ? 0 : v;
}

// A plain contiguous tensor of one of the number types (`type` says which), else null.
const at::Tensor *numbers(PyObject *o, int64_t numel, int device, int *type)
{
    if (!THPVariable_CheckExact(o)) return nullptr;
    const at::Tensor &t = THPVariable_Unpack(o);
    if (!t.defined()) return nullptr;
    *type = type_of(t.scalar_type());
    return *type < 0 ? nullptr : plain(o, t.scalar_type(), numel, device);
}

int64_t code_bytes(int64_t rows, int64_t k) { return (k + 255) / 256 * rows * 128; }
int64_t scale_bytes(int64_t rows, int64_t k) { return (k + 127) / 128 * rows * 4; }

// x, xs, q, s, [offsets,] o, m, n, k
int launch_mx_product(PyObject *const *args, bool grouped)
{
    PyObject *const *tail = args + (grouped ? 5 : 4);
    const long long m = size_of(tail[1]), n = size_of(tail[2]), k = size_of(tail[3]);
    if (!m || !n || !k) return kPythonWay;
    int x_type = TUNA_MXFP4, o_type;
    const bool packed = args[1] != Py_None;
    const at::Tensor *x = packed ? plain(args[0], at::kByte, code_bytes(n, k), -1) : numbers(args[0], n * k, -1, &x_type);
    if (!x) return kPythonWay;
    const int device = x->get_device();
    const at::Tensor *xs = packed ? plain(args[1], at::kByte, scale_bytes(n, k), device) : nullptr;
    if ((packed && !xs) || x_type == TUNA_FP32 || device != c10::cuda::current_device()) return kPythonWay;
    long long experts = 1;
    const at::Tensor *offsets = nullptr;
    if (grouped) {
        if (!THPVariable_CheckExact(args[2])) return kPythonWay;
        const at::Tensor &q = THPVariable_Unpack(args[2]);
        if (!q.defined() || q.dim() != 4 || q.size(0) < 1 || q.size(0) > TUNA_MX_MAX_EXPERTS) return kPythonWay;
        experts = q.size(0);
        offsets = plain(args[4], at::kInt, experts + 1, device);
        if (!offsets) return kPythonWay;
    }
    const at::Tensor *q = plain(args[2], at::kByte, experts * code_bytes(m, k), device), *s = plain(args[3], at::kByte, experts * scale_bytes(m, k), device),
                     *o = numbers(tail[0], n * m, device, &o_type);
    if (!q || !s || !o) return kPythonWay;
    void *stream = c10::cuda::getCurrentCUDAStream(device).stream();
    const size_t bytes = packed ? 0 : g_mx.workspace_bytes((int)m, (int)n, (int)k, grouped ? (int)experts : 0, x_type);
    at::Tensor ws;  // this call's own, in stream order: what a graph captures comes from its pool
    if (bytes > 0) ws = at::detail::empty_cuda({(int64_t)bytes}, at::kByte, x->device(), std::nullopt);
    const void *xp = x->const_data_ptr(), *xsp = xs ? xs->const_data_ptr() : nullptr, *qp = q->const_data_ptr(), *sp = s->const_data_ptr(),
               *fp = offsets ? offsets->const_data_ptr() : nullptr;
    void *op = o->mutable_data_ptr(), *wp = bytes > 0 ? ws.mutable_data_ptr() : nullptr;
    const auto f = g_mx;
    const Unlocked unlocked;
    return grouped ? f.matmul_grouped(xp, x_type, xsp, qp, sp, fp, op, o_type, (int)m, (int)n, (int)k, (int)experts, wp, bytes, stream)
                   : f.matmul(xp, x_type, xsp, qp, sp, op, o_type, (int)m, (int)n, (int)k, wp, bytes, stream);
}

// q, s, o, m, k
int launch_mx_dequant(PyObject *const *args)
{
    const long long m = size_of(args[3]), k = size_of(args[4]);
    int o_type;
    if (!m || !k || !THPVariable_CheckExact(args[0])) return kPythonWay;
    const at::Tensor &t = THPVariable_Unpack(args[0]);
    if (!t.defined() || t.dim() != 3) return kPythonWay;  // one matrix
    const at::Tensor *q = plain(args[0], at::kByte, code_bytes(m, k), -1);
    if (!q) return kPythonWay;
    const int device = q->get_device();
    const at::Tensor *s = plain(args[1], at::kByte, scale_bytes(m, k), device), *o = numbers(args[2], m * k, device, &o_type);
    if (!s || !o || device != c10::cuda::current_device()) return kPythonWay;
    void *stream = c10::cuda::getCurrentCUDAStream(device).stream();
    const void *qp = q->const_data_ptr(), *sp = s->const_data_ptr();
    void *op = o->mutable_data_ptr();
    const auto f = g_mx.dequant;
    const Unlocked unlocked;
    return f(qp, sp, op, o_type, (int)m, (int)k, 1, stream);
}

// x [rows, k] -> (q, s) in `out`; a status
int launch_mx_quantize(PyObject *x, at::Tensor (&out)[2])
{
    if (!THPVariable_CheckExact(x)) return kPythonWay;
    const at::Tensor &t = THPVariable_Unpack(x);
    if (!t.defined() || t.dim() != 2 || t.numel() == 0) return kPythonWay;
    const int64_t rows = t.size(0), k = t.size(1);
    int type;
    if (!numbers(x, t.numel(), -1, &type) || rows > 0x7fffffff || k > 0x7fffffff || k % 32 || t.get_device() != c10::cuda::current_device()) return kPythonWay;
    void *stream = c10::cuda::getCurrentCUDAStream(t.get_device()).stream();
    // torch.empty without its way through the dispatcher, 1 us shorter
    out[0] = at::detail::empty_cuda({(k + 255) / 256, rows, 128}, at::kByte, t.device(), std::nullopt);
    out[1] = at::detail::empty_cuda({(k + 127) / 128, rows, 4}, at::kByte, t.device(), std::nullopt);
    const void *xp = t.const_data_ptr();
    void *qp = out[0].mutable_data_ptr(), *sp = out[1].mutable_data_ptr();
    const auto f = g_mx.quantize;
    const Unlocked unlocked;
    return f(xp, type, k, qp, sp, (int)rows, (int)k, 1, stream);
}

// ---- the 8-bit block-scaled operators (fp8.py): the same answers

struct {
    int (*quantize)(const void *x, int x_type, long long row_stride, int blocks, void *q, void *s, void *q2, void *s2, int rows, int k, void *stream);
    int (*dequant)(const void *q, const void *s, int blocks, void *o, int o_type, int rows, int k, void *stream);
    int (*matmul)(const void *x, int x_type, const void *xs, const void *q, const void *s, void *o, int o_type, int m, int n, int k, void *workspace,
                  size_t workspace_bytes, void *stream);
    int (*matmul_backward)(const void *dy, int dy_type, const void *x, int x_type, const void *xs, const void *q, const void *s, void *dx, int dx_type, void *dw, int dw_type,
                           int m, int n, int k, void *workspace, size_t workspace_bytes, void *stream);
    int (*gated)(const void *x, int x_type, const void *xs, const void *q, const void *s, void *h, int h_type, void *z, int f, int n, int k, int activation,
                 void *workspace, size_t workspace_bytes, void *stream);
    int (*gated_backward)(const void *dh, const void *z, int type, const void *x, int x_type, const void *xs, const void *q, const void *s, void *dx, int dx_type, void *dw,
                          int dw_type, int f, int n, int k, int activation, void *workspace, size_t workspace_bytes, void *stream);
    size_t (*workspace_bytes)(int call, int m, int n, int k, int x_type);
} g_fp8 = {};

constexpr at::ScalarType kFp8Codes = at::kFloat8_e4m3fn;

int64_t fp8_scales(int64_t rows, int64_t k, int blocks)
{
    if (blocks == TUNA_FP8_SQUARE) return (rows + 127) / 128 * ((k + 127) / 128);
    return blocks == TUNA_FP8_ROW ? (k + 511) / 512 * rows * 4 : (rows + 511) / 512 * k * 4;
}

// A small number that the caller has checked or looked up.
int code_of(PyObject *o) { return PyLong_CheckExact(o) ? (int)PyLong_AsLong(o) : -1; }

const void *address(const at::Tensor *t) { return t ? t->const_data_ptr() : nullptr; }
void *writable(const at::Tensor *t) { return t ? t->mutable_data_ptr() : nullptr; }

// Operands x and xs (None: x is numbers of 16 bits) of a call, with scales of `blocks`
struct Fp8Tokens {
    const at::Tensor *x = nullptr, *xs = nullptr;
    int type = TUNA_FP8;
    bool take(PyObject *x_arg, PyObject *xs_arg, int64_t n, int64_t k, int blocks, int device)
    {
        if (xs_arg == Py_None) {
            x = numbers(x_arg, n * k, device, &type);
            return x && type != TUNA_FP32;
        }
        x = plain(x_arg, kFp8Codes, n * k, device);
        xs = x ? plain(xs_arg, at::kByte, fp8_scales(n, k, blocks), x->get_device()) : nullptr;
        return xs != nullptr;
    }
};

at::Tensor fp8_workspace(int call, int64_t m, int64_t n, int64_t k, int x_type, const at::Tensor &like)
{
    const size_t bytes = g_fp8.workspace_bytes(call, (int)m, (int)n, (int)k, x_type);
    return bytes ? at::detail::empty_cuda({(int64_t)bytes}, at::kByte, like.device(), std::nullopt) : at::Tensor();
}

// x, xs, q, s, o, m, n, k, and gated: activation, z
int launch_fp8_product(PyObject *const *args, bool gated)
{
    const long long f = size_of(args[5]), m = gated ? 2 * f : f, n = size_of(args[6]), k = size_of(args[7]);
    if (!f || !n || !k || m > 0x7fffffff) return kPythonWay;
    Fp8Tokens t;
    if (!t.take(args[0], args[1], n, k, TUNA_FP8_ROW, -1)) return kPythonWay;
    const int device = t.x->get_device();
    if (device != c10::cuda::current_device()) return kPythonWay;
    int o_type;
    const at::Tensor *q = plain(args[2], kFp8Codes, m * k, device), *s = plain(args[3], at::kByte, fp8_scales(m, k, TUNA_FP8_SQUARE), device), *o = numbers(args[4], n * f, device, &o_type),
                     *z = nullptr;
    if (!q || !s || !o) return kPythonWay;
    const int activation = gated ? code_of(args[8]) : 0;
    if (gated && args[9] != Py_None && (o_type == TUNA_FP32 || !(z = plain(args[9], o->scalar_type(), n * m, device)))) return kPythonWay;
    void *stream = c10::cuda::getCurrentCUDAStream(device).stream();
    const at::Tensor ws = fp8_workspace(gated ? TUNA_FP8_GATED : TUNA_FP8_MATMUL, m, n, k, t.type, *t.x);
    const size_t bytes = ws.defined() ? ws.nbytes() : 0;
    const void *xp = address(t.x), *xsp = address(t.xs), *qp = address(q), *sp = address(s);
    void *op = writable(o), *zp = writable(z), *wp = ws.defined() ? ws.mutable_data_ptr() : nullptr;
    const auto fn = g_fp8;
    const Unlocked unlocked;
    return gated ? fn.gated(xp, t.type, xsp, qp, sp, op, o_type, zp, (int)f, (int)n, (int)k, activation, wp, bytes, stream)
                 : fn.matmul(xp, t.type, xsp, qp, sp, op, o_type, (int)m, (int)n, (int)k, wp, bytes, stream);
}

// dy, x, xs, q, s, dx, dw, m, n, k; gated: dh, z, x .. k, activation
int launch_fp8_backward(PyObject *const *args, bool gated)
{
    PyObject *const *rest = args + (gated ? 2 : 1);
    const long long f = size_of(rest[6]), m = gated ? 2 * f : f, n = size_of(rest[7]), k = size_of(rest[8]);
    if (!f || !n || !k || m > 0x7fffffff || (rest[4] == Py_None && rest[5] == Py_None)) return kPythonWay;
    int dy_type, dx_type = 0, dw_type = 0;
    const at::Tensor *dy = numbers(args[0], n * f, -1, &dy_type);
    if (!dy || dy_type == TUNA_FP32) return kPythonWay;
    const int device = dy->get_device();
    if (device != c10::cuda::current_device()) return kPythonWay;
    const at::Tensor *z = gated ? plain(args[1], dy->scalar_type(), n * m, device) : nullptr, *q = nullptr, *s = nullptr, *dx = nullptr, *dw = nullptr;
    if (gated && !z) return kPythonWay;
    Fp8Tokens t;
    if (rest[4] != Py_None) {
        q = plain(rest[2], kFp8Codes, m * k, device);
        s = plain(rest[3], at::kByte, fp8_scales(m, k, TUNA_FP8_SQUARE), device);
        dx = numbers(rest[4], n * k, device, &dx_type);
        if (!q || !s || !dx) return kPythonWay;
    }
    if (rest[5] != Py_None) {
        dw = numbers(rest[5], m * k, device, &dw_type);
        if (!dw || !t.take(rest[0], rest[1], n, k, TUNA_FP8_COLUMN, device)) return kPythonWay;
    }
    const int activation = gated ? code_of(rest[9]) : 0;
    void *stream = c10::cuda::getCurrentCUDAStream(device).stream();
    const at::Tensor ws = fp8_workspace(TUNA_FP8_BACKWARD, m, n, k, t.type, *dy);
    const size_t bytes = ws.defined() ? ws.nbytes() : 0;
    const void *dyp = address(dy), *zp = address(z), *xp = address(t.x), *xsp = address(t.xs), *qp = address(q), *sp = address(s);
    void *dxp = writable(dx), *dwp = writable(dw), *wp = ws.defined() ? ws.mutable_data_ptr() : nullptr;
    const auto fn = g_fp8;
    const Unlocked unlocked;
    return gated ? fn.gated_backward(dyp, zp, dy_type, xp, t.type, xsp, qp, sp, dxp, dx_type, dwp, dw_type, (int)f, (int)n, (int)k, activation, wp, bytes, stream)
                 : fn.matmul_backward(dyp, dy_type, xp, t.type, xsp, qp, sp, dxp, dx_type, dwp, dw_type, (int)m, (int)n, (int)k, wp, bytes, stream);
}

// q, s, o, m, k, blocks
int launch_fp8_dequant(PyObject *const *args)
{
    const long long m = size_of(args[3]), k = size_of(args[4]);
    const int blocks = code_of(args[5]);
    int o_type;
    if (!m || !k) return kPythonWay;
    const at::Tensor *q = plain(args[0], kFp8Codes, m * k, -1);
    if (!q) return kPythonWay;
    const int device = q->get_device();
    const at::Tensor *s = plain(args[1], at::kByte, fp8_scales(m, k, blocks), device), *o = numbers(args[2], m * k, device, &o_type);
    if (!s || !o || device != c10::cuda::current_device()) return kPythonWay;
    void *stream = c10::cuda::getCurrentCUDAStream(device).stream();
    const void *qp = address(q), *sp = address(s);
    void *op = writable(o);
    const auto fn = g_fp8.dequant;
    const Unlocked unlocked;
    return fn(qp, sp, blocks, op, o_type, (int)m, (int)k, stream);
}

// x [rows, k], blocks -> codes and scales in `out`, of both ways one after the other; a status
int launch_fp8_quantize(PyObject *const *args, at::Tensor (&out)[4])
{
    PyObject *x = args[0];
    const int blocks = code_of(args[1]);
    if (!THPVariable_CheckExact(x)) return kPythonWay;
    const at::Tensor &t = THPVariable_Unpack(x);
    if (!t.defined() || t.dim() != 2 || t.numel() == 0) return kPythonWay;
    const int64_t rows = t.size(0), k = t.size(1);
    int type;
    if (!numbers(x, t.numel(), -1, &type) || rows > 0x7fffffff || k > 0x7fffffff || k % 16 || t.get_device() != c10::cuda::current_device()) return kPythonWay;
    void *stream = c10::cuda::getCurrentCUDAStream(t.get_device()).stream();
    void *ptr[4] = {};
    for (int i = 0; i < (blocks == TUNA_FP8_BOTH ? 2 : 1); ++i) {
        const int way = blocks != TUNA_FP8_BOTH ? blocks : i ? TUNA_FP8_COLUMN : TUNA_FP8_ROW;
        out[2 * i] = at::detail::empty_cuda({rows, k}, kFp8Codes, t.device(), std::nullopt);
        out[2 * i + 1] = way == TUNA_FP8_SQUARE ? at::detail::empty_cuda({(rows + 127) / 128, (k + 127) / 128}, at::kByte, t.device(), std::nullopt)
                       : way == TUNA_FP8_ROW    ? at::detail::empty_cuda({(k + 511) / 512, rows, 4}, at::kByte, t.device(), std::nullopt)
                                                : at::detail::empty_cuda({(rows + 511) / 512, k, 4}, at::kByte, t.device(), std::nullopt);
        ptr[2 * i] = out[2 * i].mutable_data_ptr();
        ptr[2 * i + 1] = out[2 * i + 1].mutable_data_ptr();
    }
    const void *xp = t.const_data_ptr();
    const auto fn = g_fp8.quantize;
    const Unlocked unlocked;
    return fn(xp, type, k, blocks, ptr[0], ptr[1], ptr[2], ptr[3], (int)rows, (int)k, stream);
}

PyObject *answer(int st) { return st == TUNA_OK || st == kPythonWay ? PyBool_FromLong(st == TUNA_OK) : PyLong_FromLong(st); }

template <int NARGS, typename Launch>
PyObject *guarded(Py_ssize_t nargs, Launch launch, bool bound = g_mx.matmul != nullptr)
{
    int st = kPythonWay;
    try {
        if (nargs == NARGS && bound) st = launch();
    } catch (...) {
    }
    return answer(st);
}
PyObject *fast_mx_matmul(PyObject *, PyObject *const *args, Py_ssize_t nargs) { return guarded<8>(nargs, [&] { return launch_mx_product(args, false); }); }
PyObject *fast_mx_matmul_grouped(PyObject *, PyObject *const *args, Py_ssize_t nargs) { return guarded<9>(nargs, [&] { return launch_mx_product(args, true); }); }
PyObject *fast_mx_dequant(PyObject *, PyObject *const *args, Py_ssize_t nargs) { return guarded<5>(nargs, [&] { return launch_mx_dequant(args); }); }

// The pair of tensors, or the answers of the others
PyObject *fast_mx_quantize(PyObject *, PyObject *const *args, Py_ssize_t nargs)
{
    at::Tensor out[2];
    PyObject *st = guarded<1>(nargs, [&] { return launch_mx_quantize(args[0], out); });
    if (st != Py_True) return st;
    Py_DECREF(st);
    PyObject *q = THPVariable_Wrap(out[0]), *s = THPVariable_Wrap(out[1]);
    return q && s ? Py_BuildValue("(NN)", q, s) : nullptr;
}

bool fp8_bound() { return g_fp8.matmul != nullptr; }
PyObject *fast_fp8_matmul(PyObject *, PyObject *const *args, Py_ssize_t nargs) { return guarded<8>(nargs, [&] { return launch_fp8_product(args, false); }, fp8_bound()); }
PyObject *fast_fp8_gated(PyObject *, PyObject *const *args, Py_ssize_t nargs) { return guarded<10>(nargs, [&] { return launch_fp8_product(args, true); }, fp8_bound()); }
PyObject *fast_fp8_matmul_backward(PyObject *, PyObject *const *args, Py_ssize_t nargs) { return guarded<10>(nargs, [&] { return launch_fp8_backward(args, false); }, fp8_bound()); }
PyObject *fast_fp8_gated_backward(PyObject *, PyObject *const *args, Py_ssize_t nargs) { return guarded<12>(nargs, [&] { return launch_fp8_backward(args, true); }, fp8_bound()); }
PyObject *fast_fp8_dequant(PyObject *, PyObject *const *args, Py_ssize_t nargs) { return guarded<6>(nargs, [&] { return launch_fp8_dequant(args); }, fp8_bound()); }

// The two tensors, or four, or the answers of the others
PyObject *fast_fp8_quantize(PyObject *, PyObject *const *args, Py_ssize_t nargs)
{
    at::Tensor out[4];
    PyObject *st = guarded<2>(nargs, [&] { return launch_fp8_quantize(args, out); }, fp8_bound());
    if (st != Py_True) return st;
    Py_DECREF(st);
    const int count = out[2].defined() ? 4 : 2;
    PyObject *all = PyTuple_New(count);
    for (int i = 0; all && i < count; ++i) {
        PyObject *t = THPVariable_Wrap(out[i]);
        if (!t) Py_CLEAR(all);
        else PyTuple_SET_ITEM(all, i, t);
    }
    return all;
}

// bind_fp8(addresses of the seven functions)
PyObject *bind_fp8(PyObject *, PyObject *args)
{
    unsigned long long f[7];
    if (!PyArg_ParseTuple(args, "KKKKKKK", &f[0], &f[1], &f[2], &f[3], &f[4], &f[5], &f[6])) return nullptr;
    g_fp8 = {(decltype(g_fp8.quantize))f[0],        (decltype(g_fp8.dequant))f[1], (decltype(g_fp8.matmul))f[2], (decltype(g_fp8.matmul_backward))f[3], (decltype(g_fp8.gated))f[4],
             (decltype(g_fp8.gated_backward))f[5], (decltype(g_fp8.workspace_bytes))f[6]};
    Py_RETURN_NONE;
}

// bind_mx(addresses of the five functions)
PyObject *bind_mx(PyObject *, PyObject *args)
{
    unsigned long long f[5];
    if (!PyArg_ParseTuple(args, "KKKKK", &f[0], &f[1], &f[2], &f[3], &f[4])) return nullptr;
    g_mx = {(decltype(g_mx.quantize))f[0], (decltype(g_mx.dequant))f[1], (decltype(g_mx.matmul))f[2], (decltype(g_mx.matmul_grouped))f[3], (decltype(g_mx.workspace_bytes))f[4]};
    Py_RETURN_NONE;
}

PyObject *fast_matmul(PyObject *, PyObject *const *args, Py_ssize_t nargs)
{
    int st = kPythonWay;
    try {
        if (nargs == 8 && g_matmul) st = launch(args);
    } catch (...) {  // a tensor without storage of its own (vmap, a trace): the Python way says what is wrong
    }
    return answer(st);
}

// workspace(device, stream) -> (address, bytes) of the one that a launch there uses, or None
PyObject *workspace(PyObject *, PyObject *args)
{
    int device;
    unsigned long long stream;
    if (!PyArg_ParseTuple(args, "iK", &device, &stream)) return nullptr;
    if (!g_workspaces) Py_RETURN_NONE;
    const Workspace ws(device, (void *)stream);
    if (!ws.tensor) Py_RETURN_NONE;
    return Py_BuildValue("(KK)", (unsigned long long)ws.ptr(), (unsigned long long)ws.bytes());
}

// bind(address of tuna_matmul, dict of the workspaces)
PyObject *bind(PyObject *, PyObject *args)
{
    unsigned long long fn;
    PyObject *workspaces;
    if (!PyArg_ParseTuple(args, "KO!", &fn, &PyDict_Type, &workspaces)) return nullptr;
    g_matmul = (MatmulFn)fn;
    Py_XSETREF(g_workspaces, Py_NewRef(workspaces));
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"matmul", (PyCFunction)(void (*)(void))fast_matmul, METH_FASTCALL, nullptr},
    {"mx_quantize", (PyCFunction)(void (*)(void))fast_mx_quantize, METH_FASTCALL, nullptr},
    {"mx_dequant", (PyCFunction)(void (*)(void))fast_mx_dequant, METH_FASTCALL, nullptr},
    {"mx_matmul", (PyCFunction)(void (*)(void))fast_mx_matmul, METH_FASTCALL, nullptr},
    {"mx_matmul_grouped", (PyCFunction)(void (*)(void))fast_mx_matmul_grouped, METH_FASTCALL, nullptr},
    {"bind_mx", bind_mx, METH_VARARGS, nullptr},
    {"fp8_quantize", (PyCFunction)(void (*)(void))fast_fp8_quantize, METH_FASTCALL, nullptr},
    {"fp8_dequant", (PyCFunction)(void (*)(void))fast_fp8_dequant, METH_FASTCALL, nullptr},
    {"fp8_matmul", (PyCFunction)(void (*)(void))fast_fp8_matmul, METH_FASTCALL, nullptr},
    {"fp8_matmul_backward", (PyCFunction)(void (*)(void))fast_fp8_matmul_backward, METH_FASTCALL, nullptr},
    {"fp8_gated", (PyCFunction)(void (*)(void))fast_fp8_gated, METH_FASTCALL, nullptr},
    {"fp8_gated_backward", (PyCFunction)(void (*)(void))fast_fp8_gated_backward, METH_FASTCALL, nullptr},
    {"bind_fp8", bind_fp8, METH_VARARGS, nullptr},
    {"workspace", workspace, METH_VARARGS, nullptr},
    {"bind", bind, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fast_call", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// torch's layouts are compiled in: _lib.py uses the module, and build.py keeps it, only where this names the torch and Python at hand.
#ifndef FAST_CALL_STAMP
#error "build.py says what this is built for"
#endif
PyMODINIT_FUNC PyInit__fast_call()
{
    PyObject *m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "stamp", FAST_CALL_STAMP) < 0) Py_CLEAR(m);
    return m;
}
