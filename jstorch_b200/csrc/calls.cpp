// calls.cpp -- the Python extension _calls: torch CUDA tensors to the C entry
// points of jstorch_scan.h, jstorch_dropout.h and jstorch_quant.h.
//
// What a call does beside its launch (checks of a handful of tensors, the
// outputs' allocation, the stream, a dozen C arguments) is what the smallest calls
// wait for: 1 x 1 x 1024 steps of the scan take 2.6 us on the device, and the
// host 5.8 us from here, 13.2 from Python over ctypes; a call of 5 x 2048 x 512 of
// the 8-bit product takes 5.3 us, 4.4 of them the host's, 10.6 from Python.  The functions take all
// arguments by position; their documentation and defaults stand in rnn.py,
// dropout.py and quant.py.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <cstdint>
#include <string>
#include <tuple>

#include "../../include/jstorch_dropout.h"
#include "../../include/jstorch_quant.h"
#include "../../include/jstorch_scan.h"

namespace {

using at::Tensor;

[[noreturn]] void error(PyObject* type, const std::string& what) {
    PyErr_SetString(type, what.c_str());
    throw python_error();
}
[[noreturn]] void value_error(const std::string& what) { error(PyExc_ValueError, what); }
[[noreturn]] void type_error(const std::string& what) { error(PyExc_TypeError, what); }

std::string text(at::IntArrayRef v) {
    std::string s = "(";
    for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
    return s + (v.size() == 1 ? ",)" : ")");
}

// `o` as a CUDA tensor of one type.
const Tensor& tensor(PyObject* o, const char* name, at::ScalarType type, const char* type_name) {
    if (!THPVariable_Check(o)) type_error(std::string(name) + " must be a torch.Tensor");
    const Tensor& x = THPVariable_Unpack(o);
    if (x.scalar_type() != type)
        type_error(std::string(name) + " must be " + type_name + " (got " + at::toString(x.scalar_type()) + ")");
    if (!x.is_cuda()) value_error(std::string(name) + " must live on a CUDA device");
    // imag() of a conjugate: the memory holds the values' negatives
    if (x.is_neg()) value_error(std::string(name) + " is a negated view: give a tensor of its own (resolve_neg())");
    return x;
}
const Tensor& f32(PyObject* o, const char* name) { return tensor(o, name, at::kFloat, "float32"); }
const Tensor& i8(PyObject* o, const char* name) { return tensor(o, name, at::kChar, "int8"); }

// The same with a given shape and device.
const Tensor& f32(PyObject* o, const char* name, at::IntArrayRef shape, int index) {
    const Tensor& x = f32(o, name);
    if (x.get_device() != index || x.sizes() != shape)
        value_error(std::string(name) + " must be a float32 tensor of shape " + text(shape) + " on cuda:" + std::to_string(index));
    return x;
}

// Address of a contiguous one, or null for None.
float* packed(PyObject* o, const char* name, at::IntArrayRef shape, int index) {
    if (o == Py_None) return nullptr;
    const Tensor& x = f32(o, name, shape, index);
    if (!x.is_contiguous()) value_error(std::string(name) + " must be contiguous");
    return static_cast<float*>(x.data_ptr());
}

// Address of `n` adjacent values.
float* vector(PyObject* o, const char* name, int64_t n, int index) {
    (void)f32(o, name);  // None is not one
    return packed(o, name, {n}, index);
}

float* floats(const Tensor& x) { return static_cast<float*>(x.data_ptr()); }
int8_t* bytes(const Tensor& x) { return static_cast<int8_t*>(x.data_ptr()); }

// A reference that this holds.
struct Owned {
    PyObject* p;
    explicit Owned(PyObject* o) : p(o) {
        if (!p) throw python_error();
    }
    ~Owned() { Py_DECREF(p); }
    Owned(const Owned&) = delete;
    Owned& operator=(const Owned&) = delete;
};

PyObject* pair(const Tensor& a, const Tensor& b) {
    const Owned x(THPVariable_Wrap(a)), y(b.defined() ? THPVariable_Wrap(b) : Py_NewRef(Py_None));
    return PyTuple_Pack(2, x.p, y.p);
}

bool truth(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw python_error();
    return v != 0;
}

long integer(PyObject* o) {
    const long v = PyLong_AsLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
}

[[noreturn]] void bad_strides(const Tensor& x, const char* name) {
    value_error(std::string(name) + ": unsupported strides " + text(x.strides()) + " for shape " + text(x.sizes()));
}

// The device and stream of one call: current while it lasts.  `stream` is a
// torch.cuda.Stream or None (the device's current stream).  Memory made while a
// stream is current belongs to that stream: the allocator does not hand out what
// the stream could still be using in another stream's order.
class Call {
  public:
    Call(int index, PyObject* stream) : options_(at::TensorOptions().device(at::kCUDA, (c10::DeviceIndex)index)) {
        if (stream == Py_None) {
            device_.set_index((c10::DeviceIndex)index);
            handle_ = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)index).stream();
            return;
        }
        const long id = attribute(stream, "stream_id"), on = attribute(stream, "device_index"),
                   type = attribute(stream, "device_type");
        if (on != index)
            value_error("stream belongs to cuda:" + std::to_string(on) + ", the tensors to cuda:" + std::to_string(index));
        const auto s = c10::cuda::CUDAStream::unpack3(id, (c10::DeviceIndex)on, (c10::DeviceType)type);
        stream_.reset_stream(s);
        handle_ = s.stream();
    }

    Tensor empty(at::IntArrayRef shape, at::ScalarType type = at::kFloat) const { return at::empty(shape, options_.dtype(type)); }
    jst_stream_t handle() const { return reinterpret_cast<jst_stream_t>(handle_); }

    // entry() without the interpreter's lock; raises JstError on a status.
    template <typename F>
    static void run(F&& entry) {
        int status;
        Py_BEGIN_ALLOW_THREADS
        status = entry();
        Py_END_ALLOW_THREADS
        if (status == JST_OK) return;
        const Owned lib(PyImport_ImportModule("jstorch_b200._lib"));
        const Owned none(PyObject_CallMethod(lib.p, "check", "i", status));
    }

  private:
    static long attribute(PyObject* o, const char* name) {
        PyObject* v = PyObject_GetAttrString(o, name);
        const long n = v ? PyLong_AsLong(v) : -1;
        Py_XDECREF(v);
        if (n == -1 && PyErr_Occurred()) throw python_error();
        return n;
    }

    at::TensorOptions options_;
    c10::cuda::OptionalCUDAGuard device_;
    c10::cuda::OptionalCUDAStreamGuard stream_;
    cudaStream_t handle_ = nullptr;
};

void arguments(const char* name, Py_ssize_t given, Py_ssize_t wanted) {
    if (given != wanted) type_error(std::string(name) + " takes " + std::to_string(wanted) + " arguments");
}

// ------------------------------------------------------------ scan
// Row pitch of a tensor [seq, batch, cols] whose rows are equally far apart.
int64_t step_rows(const Tensor& x, const char* name) {
    const int64_t seq = x.size(0), batch = x.size(1), cols = x.size(2);
    if (x.is_contiguous()) return cols;
    const int64_t s0 = x.stride(0), s1 = x.stride(1), pitch = batch > 1 ? s1 : seq > 1 ? s0 : cols;
    if ((cols > 1 && x.stride(2) != 1) || pitch < cols || (seq > 1 && batch > 1 && s0 != batch * s1)) bad_strides(x, name);
    return pitch;
}

struct Scan {
    const Tensor& gates;
    int index;
    int64_t seq = 0, batch = 0, hidden = 0, ld = 0;
    const float* h0 = nullptr;
    const int32_t* lengths = nullptr;

    Scan(PyObject* g, PyObject* h, PyObject* l) : gates(f32(g, "gates")), index(gates.get_device()) {
        if (gates.dim() != 3 || gates.size(2) % 2) value_error("gates must be [seq, batch, 2 * hidden]");
        seq = gates.size(0);
        batch = gates.size(1);
        hidden = gates.size(2) / 2;
        if (std::max({seq, batch, 2 * hidden}) > INT32_MAX) value_error("gates: size > 2^31 - 1");
        ld = step_rows(gates, "gates");
        h0 = packed(h, "h0", {batch, hidden}, index);
        if (l == Py_None) return;
        if (!THPVariable_Check(l)) type_error("lengths must be a torch.Tensor");
        const Tensor& n = THPVariable_Unpack(l);
        if (n.scalar_type() != at::kInt || !n.is_cuda() || n.get_device() != index || n.dim() != 1 || n.size(0) != batch ||
            !n.is_contiguous())
            value_error("lengths must be a contiguous int32 tensor of shape (" + std::to_string(batch) + ",) on cuda:" +
                        std::to_string(index));
        lengths = static_cast<const int32_t*>(n.data_ptr());
    }
};

// (gates, h0, lengths, reverse, candidate, out, h_n, stream) -> (out, h_n)
PyObject* scan_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arguments("scan_forward", n, 8);
    const Scan s(a[0], a[1], a[2]);
    const int reverse = truth(a[3]), candidate = (int)integer(a[4]);
    const Call call(s.index, a[7]);
    const Tensor out = a[5] == Py_None ? call.empty({s.seq, s.batch, s.hidden})
                                       : f32(a[5], "out", {s.seq, s.batch, s.hidden}, s.index);
    const int64_t ld_out = step_rows(out, "out");
    float* last = packed(a[6], "h_n", {s.batch, s.hidden}, s.index);
    Tensor h_n;
    if (a[6] == Py_None) {
        h_n = call.empty({s.batch, s.hidden});
        last = floats(h_n);
    } else {
        h_n = THPVariable_Unpack(a[6]);
    }
    const float* gates = floats(s.gates);
    float* to = floats(out);
    Call::run([&] {
        return jst_scan_forward(gates, s.ld, (int)s.seq, (int)s.batch, (int)s.hidden, s.h0, s.lengths, reverse, candidate, to,
                                ld_out, last, call.handle());
    });
    return pair(out, h_n);
    END_HANDLE_TH_ERRORS
}

// (gates, out, dout, h0, dh_n, lengths, reverse, candidate, dgates, stream) -> (dgates, dh0)
PyObject* scan_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arguments("scan_backward", n, 10);
    const Scan s(a[0], a[3], a[5]);
    const int reverse = truth(a[6]), candidate = (int)integer(a[7]);
    const Tensor& out = f32(a[1], "out", {s.seq, s.batch, s.hidden}, s.index);
    const int64_t ld_out = step_rows(out, "out");
    const float* dout = nullptr;
    int64_t ld_dout = s.hidden;
    if (a[2] != Py_None) {
        const Tensor& d = f32(a[2], "dout", {s.seq, s.batch, s.hidden}, s.index);
        ld_dout = step_rows(d, "dout");
        dout = floats(d);
    }
    const float* dh_n = packed(a[4], "dh_n", {s.batch, s.hidden}, s.index);
    const Call call(s.index, a[9]);
    const Tensor dgates = a[8] == Py_None ? call.empty({s.seq, s.batch, 2 * s.hidden})
                                          : f32(a[8], "dgates", {s.seq, s.batch, 2 * s.hidden}, s.index);
    const int64_t ld_dgates = step_rows(dgates, "dgates");
    Tensor dh0;
    if (s.h0 || a[3] != Py_None) dh0 = call.empty({s.batch, s.hidden});
    const float *gates = floats(s.gates), *from = floats(out);
    float *to = floats(dgates), *first = dh0.defined() ? floats(dh0) : nullptr;
    Call::run([&] {
        return jst_scan_backward(gates, s.ld, (int)s.seq, (int)s.batch, (int)s.hidden, s.h0, s.lengths, reverse, candidate,
                                 from, ld_out, dout, ld_dout, dh_n, to, ld_dgates, first, call.handle());
    });
    return pair(dgates, dh0);
    END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------ dropout
struct Rows {
    int64_t rows, cols, pitch;
};

// x as a row-major matrix; contiguous tensors are one row.
Rows flat_rows(const Tensor& x, const char* name) {
    if (x.is_contiguous()) return {1, x.numel(), x.numel()};
    const auto shape = x.sizes(), stride = x.strides();
    const size_t last = shape.size() - 1;
    const int64_t cols = shape[last];
    if (cols > 1 && stride[last] != 1) bad_strides(x, name);
    int64_t pitch = 0, rows = 1;
    for (size_t i = last; i-- > 0;) {
        if (shape[i] == 1) continue;
        if (pitch == 0) pitch = stride[i];
        if (stride[i] != pitch * rows || pitch < cols) bad_strides(x, name);
        rows *= shape[i];
    }
    return {rows, cols, pitch ? pitch : cols};
}

uint64_t word64(PyObject* o) {
    const Owned i(PyNumber_Index(o));
    const unsigned long long v = PyLong_AsUnsignedLongLong(i.p);
    if (v == (unsigned long long)-1 && PyErr_Occurred()) {
        if (!PyErr_ExceptionMatches(PyExc_OverflowError)) throw python_error();
        PyErr_Clear();
        value_error("seed and offset must be 64-bit unsigned integers");
    }
    return v;
}

// (x, p, seed, offset, step, out, stream) -> out
PyObject* dropout(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arguments("dropout", n, 7);
    const Tensor& x = f32(a[0], "x");
    const int index = x.get_device();
    const double p = PyFloat_AsDouble(a[1]);
    if (p == -1.0 && PyErr_Occurred()) throw python_error();
    if (!(p >= 0.0 && p <= 1.0)) value_error("p must be in [0, 1] (got " + std::to_string(p) + ")");
    const uint64_t seed = word64(a[2]), offset = word64(a[3]);
    const int64_t* step = nullptr;
    if (a[4] != Py_None) {
        if (!THPVariable_Check(a[4])) type_error("step must be a torch.Tensor");
        const Tensor& s = THPVariable_Unpack(a[4]);
        if (s.scalar_type() != at::kLong || s.numel() != 1 || !s.is_cuda() || s.get_device() != index)
            value_error("step must be a one-element int64 tensor on x's device");
        step = static_cast<const int64_t*>(s.data_ptr());
    }
    const Call call(index, a[6]);
    const Tensor out = a[5] == Py_None ? call.empty(x.sizes()) : f32(a[5], "out", x.sizes(), index);
    Rows from = flat_rows(x, "x"), to = flat_rows(out, "out");
    // one of the two has gaps: the other has rows of the same length without any
    if (to.rows == 1 && from.rows > 1) to = {from.rows, from.cols, from.cols};
    if (from.rows == 1 && to.rows > 1) from = {to.rows, to.cols, to.cols};
    const float* src = floats(x);
    float* dst = floats(out);
    Call::run([&] {
        return jst_dropout(src, from.pitch, dst, to.pitch, from.rows, from.cols, p, seed, offset, step, call.handle());
    });
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------ 8-bit products
// A 2-D tensor whose columns are adjacent; the C entry points count its sizes
// in 32 bits.
Rows matrix(const Tensor& x, const char* name) {
    if (x.dim() != 2) value_error(std::string(name) + " must be 2-D");
    const int64_t rows = x.size(0), cols = x.size(1);
    if (std::max(rows, cols) > 0x7fff0000) value_error(std::string(name) + ": size > 0x7fff0000");
    const int64_t packed = std::max<int64_t>(cols, 1);
    if (x.is_contiguous()) return {rows, cols, packed};
    if ((cols > 1 && x.stride(1) != 1) || (rows > 1 && x.stride(0) < cols)) bad_strides(x, name);
    return {rows, cols, rows > 1 ? x.stride(0) : packed};
}

// (x, stream) -> (q, scale)
PyObject* quantize_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arguments("quantize_rows", n, 2);
    const Tensor& x = f32(a[0], "x");
    const Rows m = matrix(x, "x");
    const Call call(x.get_device(), a[1]);
    const int64_t pitch = std::max<int64_t>((m.cols + 15) / 16 * 16, 16);
    Tensor q = call.empty({m.rows, pitch}, at::kChar);
    const Tensor scale = call.empty({m.rows});
    const float* from = floats(x);
    int8_t* to = bytes(q);
    float* s = floats(scale);
    Call::run([&] { return jst_quantize_rows_i8(from, m.pitch, (int)m.rows, (int)m.cols, to, pitch, s, call.handle()); });
    if (pitch != m.cols) q = q.slice(1, 0, m.cols);
    return pair(q, scale);
    END_HANDLE_TH_ERRORS
}

// What gemm_i8 and linear_i8 share behind their first operand x [M, K]: the
// weight, its scales, bias, epilogue and output.
struct Product {
    int index;
    Rows x, w;
    const int8_t* weight;
    const float *scale, *bias;
    int epilogue;

    Product(const char* name, const char* x_name, const Tensor& first, PyObject* weight_o, PyObject* scale_o, PyObject* bias_o,
            PyObject* relu)
        : index(first.get_device()) {
        const Tensor& second = i8(weight_o, "w");
        if (second.get_device() != index) value_error(std::string(x_name) + " and w must live on one device");
        x = matrix(first, x_name);
        w = matrix(second, "w");
        if (x.cols != w.cols)
            value_error(std::string(name) + " shape mismatch: " + x_name + " is [" + std::to_string(x.rows) + ", " +
                        std::to_string(x.cols) + "], w is [" + std::to_string(w.rows) + ", " + std::to_string(w.cols) + "]");
        weight = bytes(second);
        scale = vector(scale_o, "w_scale", w.rows, index);
        bias = packed(bias_o, "bias", {w.rows}, index);
        epilogue = (bias_o != Py_None ? JST_EPI_BIAS : 0) | (truth(relu) ? JST_EPI_RELU : 0);
    }

    Tensor output(PyObject* out, const Call& call) const {
        return out == Py_None ? call.empty({x.rows, w.rows}) : f32(out, "out", {x.rows, w.rows}, index);
    }
};

// (a, w, a_scale, w_scale, out, bias, relu, stream) -> out
PyObject* gemm_i8(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arguments("gemm_i8", n, 8);
    const Tensor& tokens = i8(a[0], "a");
    const Product p("gemm_i8", "a", tokens, a[1], a[3], a[5], a[6]);
    jst_gemm_i8_desc d = {};
    d.M = (int)p.x.rows; d.N = (int)p.w.rows; d.K = (int)p.x.cols;
    d.A = bytes(tokens); d.lda = p.x.pitch;
    d.B = p.weight; d.ldb = p.w.pitch;
    d.a_scale = vector(a[2], "a_scale", p.x.rows, p.index);
    d.b_scale = p.scale; d.bias = p.bias; d.epilogue = p.epilogue;
    const Call call(p.index, a[7]);
    const Tensor out = p.output(a[4], call);
    d.C = floats(out); d.ldc = matrix(out, "out").pitch;
    d.stream = call.handle();
    Call::run([&] { return jst_gemm_i8(&d); });
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// (x, w, w_scale, out, bias, relu, stream) -> out
PyObject* linear_i8(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arguments("linear_i8", n, 7);
    const Tensor& x = f32(a[0], "x");
    const Product p("linear_i8", "x", x, a[1], a[2], a[4], a[5]);
    const Call call(p.index, a[6]);
    const Tensor out = p.output(a[3], call);
    const int64_t ldy = matrix(out, "out").pitch;
    const float* from = floats(x);
    float* to = floats(out);
    Call::run([&] {
        return jst_linear_i8(from, p.x.pitch, (int)p.x.rows, (int)p.x.cols, p.weight, p.w.pitch, p.scale, (int)p.w.rows,
                             p.bias, p.epilogue, to, ldy, call.handle());
    });
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

#define JST_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {JST_METHOD(scan_forward), JST_METHOD(scan_backward), JST_METHOD(dropout),
                         JST_METHOD(quantize_rows), JST_METHOD(gemm_i8), JST_METHOD(linear_i8),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__calls() {
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "torch_version", JST_TORCH_VERSION) < 0) {
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
