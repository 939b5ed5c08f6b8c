// opennpu_amd._kv8: the 8-bit key-value cache's calls for torch tensors (device.py kv8_write, kv8_read, kv8_attn),
// checked here and handed to the C entries of include/onpu.h, whose addresses device.py binds. A decode
// step's calls are bound by their issue: through ctypes and checks in Python kv8_attn took 9.9 us of the
// host to issue, here 4.2, 3.3 of them the launch.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "onpu.h"

namespace {

decltype(&onpu_kv8_write_dev) c_write;
decltype(&onpu_kv8_read_dev) c_read;
decltype(&onpu_kv8_attn_ws_bytes) c_ws_bytes;
decltype(&onpu_kv8_attn_dev) c_attn;
decltype(&onpu_last_error) c_error;

struct Refused {                              // becomes a ValueError
    std::string why;
};

[[noreturn]] void refuse(const char * what, const std::string & why) { throw Refused{std::string(what) + ": " + why}; }

const at::Tensor & tensor(PyObject * o, const char * what, const char * name) {
    if (!THPVariable_Check(o)) refuse(what, std::string(name) + " must be a tensor");
    return THPVariable_Unpack(o);
}

void on_gpu(const at::Tensor & t, int here, const char * what) {
    if (!t.is_cuda() || t.get_device() != here)
        refuse(what, "every tensor must be on the current GPU (cuda:" + std::to_string(here) + "), got " + t.device().str());
}

int64_t whole(PyObject * o) {
    const int64_t v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw Refused{""};
    return v;
}
int whole32(PyObject * o, const char * what, const char * name) {
    const int64_t v = whole(o);
    if (v < INT32_MIN || v > INT32_MAX) refuse(what, std::string(name) + " does not fit 32 bits");
    return (int) v;
}

// the arguments that the three calls share, as device.py documents them
struct Common {
    void * codes, * stream;
    float * scales;
    const int32_t * table, * pos, * off;
    int64_t pages, T, tld;
    int Hkv, D, P, nseq, here, bf16;
};

// rows: fp32 or bf16 [T][heads][D]
Common common(const at::Tensor & codes, const at::Tensor & scales, const at::Tensor & table, const at::Tensor & pos, PyObject * off_o,
              const at::Tensor & rows, const char * what) {
    Common c;
    c.here = c10::hip::current_device();
    if (codes.scalar_type() != at::kChar || codes.dim() != 4 || codes.size(2) != 2 || codes.size(3) % 64 || !codes.is_contiguous())
        refuse(what, "codes must be int8 [pages][Hkv][2][64 D], contiguous");
    if (scales.scalar_type() != at::kFloat || scales.dim() != 3 || scales.size(0) != codes.size(0) ||
        scales.size(1) != codes.size(1) || scales.size(2) != 2 || !scales.is_contiguous())
        refuse(what, "scales must be fp32 [pages][Hkv][2], contiguous");
    if (table.scalar_type() != at::kInt || table.dim() != 2 || (table.size(1) > 1 && table.stride(1) != 1))
        refuse(what, "table must be int32 [sequences][P] with rows of unit stride");
    if (pos.scalar_type() != at::kInt || pos.dim() != 1 || pos.size(0) != table.size(0) || !pos.is_contiguous())
        refuse(what, "positions or lengths must be int32, one per sequence, contiguous");
    for (const at::Tensor * t : {&codes, &scales, &table, &pos, &rows}) on_gpu(*t, c.here, what);
    c.off = nullptr;
    if (off_o != Py_None) {
        const at::Tensor & off = tensor(off_o, what, "off");
        if (off.scalar_type() != at::kInt || off.dim() != 1 || off.size(0) != table.size(0) + 1 || !off.is_contiguous())
            refuse(what, "off must be int32, one more than the sequences, contiguous");
        on_gpu(off, c.here, what);
        c.off = (const int32_t *) off.data_ptr();
    }
    c.bf16 = rows.scalar_type() == at::kBFloat16;
    if (rows.dim() != 3 || rows.size(2) * 64 != codes.size(3) || rows.stride(2) != 1 || (!c.bf16 && rows.scalar_type() != at::kFloat))
        refuse(what, "rows must be fp32 or bf16 [T][heads][" + std::to_string(codes.size(3) / 64) + "] with unit stride in the last dimension");
    if (codes.size(1) > INT32_MAX || table.size(0) > INT32_MAX || table.size(1) > INT32_MAX) refuse(what, "sizes past 32 bits");
    c.codes = codes.data_ptr();
    c.scales = (float *) scales.data_ptr();
    c.table = (const int32_t *) table.data_ptr();
    c.pos = (const int32_t *) pos.data_ptr();
    c.pages = codes.size(0);
    c.Hkv = (int) codes.size(1);
    c.D = (int) rows.size(2);
    c.nseq = (int) table.size(0);
    c.P = (int) table.size(1);
    c.tld = table.stride(0);
    c.T = rows.size(0);
    c.stream = c10::hip::getCurrentHIPStream((c10::DeviceIndex) c.here).stream();
    return c;
}

// the most rows of a sequence: given, or as many as there are; without off the same for all
int most(const Common & c, PyObject * max_n, const char * what) {
    int64_t n = c.T;
    if (!c.off) {
        const int64_t s = c.nseq > 0 ? c.nseq : 1;
        if (c.T % s) refuse(what, std::to_string(c.T) + " rows cannot be the same number for each of " + std::to_string(c.nseq) + " sequences: give off");
        n = c.T / s;
    } else if (max_n != Py_None) {
        n = whole(max_n);
    }
    if (n > INT32_MAX) refuse(what, "more rows than 32 bits count");
    return (int) n;
}

PyObject * done(int rc, PyObject * result, const char * what) {
    if (rc >= 0) return result;
    Py_XDECREF(result);
    PyErr_Format(PyExc_RuntimeError, "%s: %s", what, c_error());
    return nullptr;
}

// a call's body with C++ exceptions turned into Python's
template <class F> PyObject * guarded(Py_ssize_t n, Py_ssize_t want, F && body) {
    try {
        if (n != want || !c_attn) {
            PyErr_SetString(PyExc_TypeError, "opennpu_amd._kv8: called other than by opennpu_amd.device");
            return nullptr;
        }
        return body();
    } catch (const Refused & r) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, r.why.c_str());
    } catch (...) {                           // torch's own: out of memory and the like
        torch::translate_exception_to_python(std::current_exception());
    }
    return nullptr;
}

// codes, scales, k, v, table, pos, off, max_n
PyObject * py_write(PyObject *, PyObject * const * a, Py_ssize_t n) {
    return guarded(n, 8, [&]() -> PyObject * {
        const char * w = "kv8_write";
        const at::Tensor & k = tensor(a[2], w, "k"), & v = tensor(a[3], w, "v");
        const Common c = common(tensor(a[0], w, "codes"), tensor(a[1], w, "scales"), tensor(a[4], w, "table"), tensor(a[5], w, "pos"), a[6], k, w);
        on_gpu(v, c.here, w);
        if (k.size(1) != c.Hkv || v.dim() != 3 || v.sizes() != k.sizes() || v.scalar_type() != k.scalar_type() || v.stride(2) != 1)
            refuse(w, "k and v must have the same type and shape [T][Hkv][D], with unit stride in the last dimension");
        const int rc = c_write(c.codes, c.scales, c.pages, c.Hkv, c.D, k.data_ptr(), v.data_ptr(), c.bf16, k.stride(0), k.stride(1),
                               v.stride(0), v.stride(1), c.table, c.tld, c.P, c.pos, c.off, c.nseq, c.T, most(c, a[7], w), c.stream);
        return done(rc, Py_NewRef(Py_None), w);
    });
}

// codes, scales, table, pos, rows, off, max_n, dtype, k, v
PyObject * py_read(PyObject *, PyObject * const * a, Py_ssize_t n) {
    return guarded(n, 10, [&]() -> PyObject * {
        const char * w = "kv8_read";
        const at::Tensor & codes = tensor(a[0], w, "codes");
        const int64_t rows = whole(a[4]);
        at::Tensor k, v;
        if (a[7] != Py_None && (!THPDtype_Check(a[7]) || (((THPDtype *) a[7])->scalar_type != at::kFloat &&
                                                          ((THPDtype *) a[7])->scalar_type != at::kBFloat16)))
            refuse(w, "dtype must be fp32 or bf16");
        if (a[8] == Py_None) {
            if (rows < 0) refuse(w, "rows must not be negative");
            if (codes.dim() != 4) refuse(w, "codes must be int8 [pages][Hkv][2][64 D], contiguous");
            const auto t = a[7] == Py_None ? at::kBFloat16 : ((THPDtype *) a[7])->scalar_type;
            k = at::empty({rows, codes.size(1), codes.size(3) / 64}, codes.options().dtype(t));
            v = at::empty({rows, codes.size(1), codes.size(3) / 64}, codes.options().dtype(t));
        } else {
            k = tensor(a[8], w, "out");
            v = tensor(a[9], w, "out");
            if (k.dim() != 3 || k.size(0) != rows || codes.dim() != 4 || k.size(1) != codes.size(1) || v.sizes() != k.sizes() ||
                v.scalar_type() != k.scalar_type() || !k.is_contiguous() || !v.is_contiguous() ||
                (a[7] != Py_None && ((THPDtype *) a[7])->scalar_type != k.scalar_type()))
                refuse(w, "out must be two contiguous [rows][Hkv][D] tensors of one type");
        }
        const Common c = common(codes, tensor(a[1], w, "scales"), tensor(a[2], w, "table"), tensor(a[3], w, "pos"), a[5], k, w);
        on_gpu(v, c.here, w);
        const int rc = c_read(c.codes, c.scales, c.pages, c.Hkv, c.D, c.table, c.tld, c.P, c.pos, c.off, c.nseq, c.T, most(c, a[6], w),
                              k.data_ptr(), v.data_ptr(), c.bf16, c.stream);
        PyObject * r = PyTuple_New(2);
        if (!r) return nullptr;
        if (a[8] == Py_None) {
            PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(k)));
            PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(v)));
        } else {
            PyTuple_SET_ITEM(r, 0, Py_NewRef(a[8]));
            PyTuple_SET_ITEM(r, 1, Py_NewRef(a[9]));
        }
        return done(rc, r, w);
    });
}

// q, codes, scales, table, lens, off, max_n, max_len, mask, sinks, window, scale, out, ws
PyObject * py_attn(PyObject *, PyObject * const * a, Py_ssize_t n) {
    return guarded(n, 14, [&]() -> PyObject * {
        const char * w = "kv8_attn";
        const at::Tensor & q = tensor(a[0], w, "q"), & codes = tensor(a[1], w, "codes");
        const Common c = common(codes, tensor(a[2], w, "scales"), tensor(a[3], w, "table"), tensor(a[4], w, "lens"), a[5], q, w);
        if (q.size(1) > INT32_MAX) refuse(w, "sizes past 32 bits");
        const int Hq = (int) q.size(1), max_n = most(c, a[6], w), window = whole32(a[10], w, "window");
        const int64_t len = a[7] == Py_None ? 64 * (int64_t) c.P : whole(a[7]);
        const int max_len = len > INT32_MAX - 64 ? (a[7] == Py_None ? INT32_MAX - 64 : -1) : (len < 0 ? -1 : (int) len);
        const float * mask = nullptr, * sinks = nullptr;
        int64_t mld = 0;
        if (a[8] != Py_None) {
            const at::Tensor & m = tensor(a[8], w, "mask");
            if (m.scalar_type() != at::kFloat || m.dim() != 2 || m.size(0) != c.nseq || m.size(1) < max_len || (m.size(1) > 1 && m.stride(1) != 1))
                refuse(w, "mask must be fp32 [sequences][>= max_len], rows of unit stride");
            on_gpu(m, c.here, w);
            mask = (const float *) m.data_ptr();
            mld = c.nseq > 1 ? m.stride(0) : m.size(1);
        }
        if (a[9] != Py_None) {
            const at::Tensor & s = tensor(a[9], w, "sinks");
            if (s.scalar_type() != at::kFloat || s.dim() != 1 || s.size(0) != Hq || !s.is_contiguous())
                refuse(w, "sinks must be fp32 [Hq], contiguous");
            on_gpu(s, c.here, w);
            sinks = (const float *) s.data_ptr();
        }
        double scale = 1.0 / std::sqrt((double) c.D);
        if (a[11] != Py_None) {
            scale = PyFloat_AsDouble(a[11]);
            if (scale == -1.0 && PyErr_Occurred()) return nullptr;
        }
        at::Tensor out, ws;
        if (a[12] == Py_None) {
            out = at::empty(q.sizes(), q.options());
        } else {
            out = tensor(a[12], w, "out");
            if (out.sizes() != q.sizes() || out.scalar_type() != q.scalar_type() || !out.is_contiguous())
                refuse(w, "out must be contiguous, of q's shape and type");
            on_gpu(out, c.here, w);
        }
        const int64_t need = c_ws_bytes(c.bf16, Hq, c.D, c.Hkv, c.nseq, c.T, max_n, max_len, window);
        if (a[13] != Py_None) {
            ws = tensor(a[13], w, "ws");
            if (!ws.is_contiguous()) refuse(w, "ws must be contiguous");
            on_gpu(ws, c.here, w);
        } else if (need > 0) {
            ws = at::empty({need}, codes.options());
        }
        const int rc = c_attn(q.data_ptr(), c.bf16, Hq, q.stride(0), q.stride(1), c.codes, c.scales, c.pages, c.Hkv, c.D, c.table, c.tld,
                              c.P, c.pos, c.off, c.nseq, c.T, max_n, max_len, mask, mld, sinks, window, (float) scale, out.data_ptr(),
                              ws.defined() ? ws.data_ptr() : nullptr, ws.defined() ? (int64_t) ws.nbytes() : 0, c.stream);
        return done(rc, a[12] == Py_None ? THPVariable_Wrap(std::move(out)) : Py_NewRef(a[12]), w);
    });
}

// the C entries' addresses: write, read, attn_ws_bytes, attn, last_error
PyObject * py_bind(PyObject *, PyObject * const * a, Py_ssize_t n) {
    if (n != 5) {
        PyErr_SetString(PyExc_TypeError, "bind takes five addresses");
        return nullptr;
    }
    void * p[5];
    for (int i = 0; i < 5; i++)
        if (!(p[i] = PyLong_AsVoidPtr(a[i]))) return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_ValueError, "bind: a null address");
    c_write = (decltype(c_write)) p[0];
    c_read = (decltype(c_read)) p[1];
    c_ws_bytes = (decltype(c_ws_bytes)) p[2];
    c_error = (decltype(c_error)) p[4];
    c_attn = (decltype(c_attn)) p[3];
    Py_RETURN_NONE;
}

PyMethodDef METHODS[] = {
    {"bind", (PyCFunction) (void (*)(void)) py_bind, METH_FASTCALL, nullptr},
    {"write", (PyCFunction) (void (*)(void)) py_write, METH_FASTCALL, nullptr},
    {"read", (PyCFunction) (void (*)(void)) py_read, METH_FASTCALL, nullptr},
    {"attn", (PyCFunction) (void (*)(void)) py_attn, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef MODULE = {PyModuleDef_HEAD_INIT, "_kv8", nullptr, -1, METHODS, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__kv8() { return PyModule_Create(&MODULE); }
