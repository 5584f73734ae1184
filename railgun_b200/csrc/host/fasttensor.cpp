// What an operator does on the host around its launch, on tensors themselves instead of through their Python attributes: are the
// arguments what the kernel takes, outputs and scratch, and the launch.
//
// An attribute of a tensor costs Python 40 to 90 ns and a test of type, place and sizes needs five of them; a new tensor costs
// 2.0 to 2.5 us through torch.empty, a list of 32 caches 13 us.  (The committing of drafts in 32 layers took 37 us of host time with Python's attributes
// and takes 11.9 so, 2.7 of them the launch and 3.5 three new tensors.)  Launchers are called as in fastcall.cpp, whose comment says why one function type serves all of them.
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/Functions.h>
#include <algorithm>
#include <vector>

#if !defined(__linux__) || !(defined(__x86_64__) || defined(__aarch64__))
#error "the calling conventions relied on are those of 64-bit Linux on x86 and ARM"
#endif

#define MAX_INTS 48
#define MAX_FLOATS 8
typedef unsigned long long u64;
typedef int (*Launcher)(u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64,
                        u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64,
                        u64, u64, u64, u64, u64, u64, float, float, float, float, float, float, float, float);

static bool of_type(const at::Tensor& t, PyObject* dtype) {
    return dtype == Py_None || (THPDtype_Check(dtype) && t.scalar_type() == reinterpret_cast<THPDtype*>(dtype)->scalar_type);
}
static bool on_device(const at::Tensor& t, int64_t device) { return t.is_cuda() && t.get_device() == device; }

// One tensor of fits and fits_all: its sizes are a[0] .. a[n - 1].  -1: an error is set.
static int fits_one(PyObject* tensor, PyObject* dtype, long device, PyObject* const* a, Py_ssize_t n) {
    if (!THPVariable_Check(tensor)) return 0;
    const at::Tensor& t = THPVariable_Unpack(tensor);
    if (!on_device(t, device) || !of_type(t, dtype) || t.layout() != at::kStrided || t.dim() != n) return 0;
    for (Py_ssize_t i = 0; i < n; ++i) {
        if (a[i] == Py_None) continue;
        const long long want = PyLong_AsLongLong(a[i]);
        if (want == -1 && PyErr_Occurred()) return -1;
        if (t.size(i) != want) return 0;
    }
    return t.is_contiguous();
}

// fits(tensor, dtype or None, device, sizes..): a contiguous tensor of this type on this CUDA device, of as many dimensions and these
// sizes (None: any)?
static PyObject* ft_fits(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n < 3) {
        PyErr_SetString(PyExc_TypeError, "fits: a tensor, a type, a device and sizes");
        return nullptr;
    }
    const long device = PyLong_AsLong(a[2]);
    if (device == -1 && PyErr_Occurred()) return nullptr;
    const int fits = fits_one(a[0], a[1], device, a + 3, n - 3);
    if (fits < 0) return nullptr;
    return PyBool_FromLong(fits);
    END_HANDLE_TH_ERRORS
}

// fits_all(device, tensor, dtype, sizes.., tensor, dtype, sizes.., ..): the same of several tensors.
static PyObject* ft_fits_all(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n < 1) {
        PyErr_SetString(PyExc_TypeError, "fits_all: a device, and a tensor, a type and sizes for each");
        return nullptr;
    }
    const long device = PyLong_AsLong(a[0]);
    if (device == -1 && PyErr_Occurred()) return nullptr;
    for (Py_ssize_t i = 1; i < n;) {
        if (i + 1 >= n || !THPVariable_Check(a[i])) Py_RETURN_FALSE;
        Py_ssize_t end = i + 2;
        while (end < n && (a[end] == Py_None || (PyIndex_Check(a[end]) && !THPVariable_Check(a[end])))) ++end;
        const int fits = fits_one(a[i], a[i + 1], device, a + i + 2, end - i - 2);
        if (fits < 0) return nullptr;
        if (!fits) Py_RETURN_FALSE;
        i = end;
    }
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// rows(tensor, dtype, device, least columns): (rows, elements from one row to the next) of a matrix whose rows are contiguous and may be
// further apart than they are long; None where it is none.
static PyObject* ft_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 4) {
        PyErr_SetString(PyExc_TypeError, "rows: a tensor, a type, a device and columns");
        return nullptr;
    }
    const long device = PyLong_AsLong(a[2]);
    const long long columns = PyLong_AsLongLong(a[3]);
    if (PyErr_Occurred()) return nullptr;
    if (!THPVariable_Check(a[0])) Py_RETURN_NONE;
    const at::Tensor& t = THPVariable_Unpack(a[0]);
    if (!on_device(t, device) || !of_type(t, a[1]) || t.layout() != at::kStrided || t.dim() != 2 || t.stride(1) != 1 || t.size(1) < columns ||
        t.stride(0) < t.size(1))
        Py_RETURN_NONE;
    return Py_BuildValue("LL", (long long)t.size(0), (long long)t.stride(0));
    END_HANDLE_TH_ERRORS
}

// apart(matrix, matrix, columns): do two matrices of one type and as many rows, of which so many columns are used, share no memory?  The one may
// be columns beside the other's in a buffer.
static PyObject* ft_apart(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 3 || !THPVariable_Check(a[0]) || !THPVariable_Check(a[1]) || !PyLong_Check(a[2])) {
        PyErr_SetString(PyExc_TypeError, "apart: two matrices and columns");
        return nullptr;
    }
    const at::Tensor &x = THPVariable_Unpack(a[0]), &y = THPVariable_Unpack(a[1]);
    const long long columns = PyLong_AsLongLong(a[2]);
    if (columns == -1 && PyErr_Occurred()) return nullptr;
    if (x.dim() != 2 || y.dim() != 2 || x.size(0) != y.size(0) || x.scalar_type() != y.scalar_type()) {
        PyErr_SetString(PyExc_TypeError, "apart: matrices of one type and as many rows");
        return nullptr;
    }
    if (x.size(0) == 0 || columns <= 0) Py_RETURN_TRUE;
    const long long at = ((long long)y.data_ptr() - (long long)x.data_ptr()) / (long long)x.element_size(), before = x.size(0) - 1;
    if (at >= before * x.stride(0) + columns || -at >= before * y.stride(0) + columns) Py_RETURN_TRUE;
    const long long step = x.stride(0);
    if (step < 1 || step != y.stride(0)) Py_RETURN_FALSE;
    const long long beside = (at % step + step) % step;
    return PyBool_FromLong(columns <= beside && beside <= step - columns);
    END_HANDLE_TH_ERRORS
}

// addresses(list or tuple of tensors, device): where they are, as 64-bit numbers in a bytes object, if they are contiguous tensors of one shape and
// type on this CUDA device, no two of which share memory; None if not.
static PyObject* ft_addresses(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 2) {
        PyErr_SetString(PyExc_TypeError, "addresses: a list and a device");
        return nullptr;
    }
    const long device = PyLong_AsLong(a[1]);
    if (device == -1 && PyErr_Occurred()) return nullptr;
    if (!PyList_Check(a[0]) && !PyTuple_Check(a[0])) Py_RETURN_NONE;
    const Py_ssize_t m = PySequence_Fast_GET_SIZE(a[0]);
    PyObject** items = PySequence_Fast_ITEMS(a[0]);
    if (m == 0 || !THPVariable_Check(items[0])) Py_RETURN_NONE;
    const at::Tensor& first = THPVariable_Unpack(items[0]);
    PyObject* out = PyBytes_FromStringAndSize(nullptr, m * 8);
    if (!out) return nullptr;
    u64* to = reinterpret_cast<u64*>(PyBytes_AS_STRING(out));
    for (Py_ssize_t i = 0; i < m; ++i) {
        bool ok = THPVariable_Check(items[i]);
        if (ok) {
            const at::Tensor& t = THPVariable_Unpack(items[i]);
            ok = on_device(t, device) && t.layout() == at::kStrided && t.is_contiguous() && t.scalar_type() == first.scalar_type() &&
                 t.sizes() == first.sizes();
            if (ok) to[i] = (u64)t.data_ptr();
        }
        if (!ok) {
            Py_DECREF(out);
            Py_RETURN_NONE;
        }
    }
    std::vector<u64> places(to, to + m);
    std::sort(places.begin(), places.end());
    const u64 bytes = std::max<u64>(1, first.nbytes());
    if (std::adjacent_find(places.begin(), places.end(), [&](u64 x, u64 y) { return y - x < bytes; }) != places.end()) {
        Py_DECREF(out);
        Py_RETURN_NONE;
    }
    return out;
    END_HANDLE_TH_ERRORS
}

// empty(dtype, device, sizes..): a new tensor.
static PyObject* ft_empty(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n < 2 || n > 10 || !THPDtype_Check(a[0])) {
        PyErr_SetString(PyExc_TypeError, "empty: a type, a device and sizes");
        return nullptr;
    }
    const long device = PyLong_AsLong(a[1]);
    int64_t sizes[8];
    for (Py_ssize_t i = 2; i < n; ++i) sizes[i - 2] = PyLong_AsLongLong(a[i]);
    if (PyErr_Occurred()) return nullptr;
    const auto options = at::TensorOptions().dtype(reinterpret_cast<THPDtype*>(a[0])->scalar_type).device(at::kCUDA, (c10::DeviceIndex)device);
    return THPVariable_Wrap(at::empty(at::IntArrayRef(sizes, (size_t)n - 2), options));
    END_HANDLE_TH_ERRORS
}

// call(address, kinds, arguments..): a launcher's arguments, one letter of `kinds` each: i a whole number, f a number as a 32-bit float, p a
// tensor or bytes (where they are), an address or None (a null pointer).  The letters are the launcher's: a float in an integer's place
// would move every argument behind it.
static PyObject* ft_call(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    u64 v[MAX_INTS] = {0};
    float f[MAX_FLOATS] = {0};
    int nv = 0, nf = 0;
    Py_ssize_t n_kinds = 0;
    const char* kinds = n >= 2 && PyLong_Check(a[0]) && PyUnicode_Check(a[1]) ? PyUnicode_AsUTF8AndSize(a[1], &n_kinds) : nullptr;
    if (!kinds || n_kinds != n - 2) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "call: the launcher's address, its arguments' kinds and as many arguments");
        return nullptr;
    }
    const u64 address = PyLong_AsUnsignedLongLongMask(a[0]);
    for (Py_ssize_t i = 0; i < n_kinds; ++i) {
        PyObject* o = a[i + 2];
        if (kinds[i] == 'f') {
            const double x = PyFloat_AsDouble(o);
            if (x == -1.0 && PyErr_Occurred()) return nullptr;
            if (nf == MAX_FLOATS) {
                PyErr_SetString(PyExc_TypeError, "call: more than 8 floats");
                return nullptr;
            }
            f[nf++] = (float)x;
            continue;
        }
        if (nv == MAX_INTS) {
            PyErr_SetString(PyExc_TypeError, "call: more than 48 integers");
            return nullptr;
        }
        if (kinds[i] == 'i') {
            PyObject* whole = PyNumber_Index(o);                    // no float, no None
            if (!whole) return nullptr;
            v[nv++] = PyLong_AsUnsignedLongLongMask(whole);
            Py_DECREF(whole);
        } else if (kinds[i] != 'p') {
            PyErr_SetString(PyExc_TypeError, "call: a kind is i, f or p");
            return nullptr;
        } else if (o == Py_None) v[nv++] = 0;
        else if (PyLong_Check(o)) v[nv++] = PyLong_AsUnsignedLongLongMask(o);
        else if (THPVariable_Check(o)) v[nv++] = (u64)THPVariable_Unpack(o).data_ptr();
        else if (PyBytes_Check(o)) v[nv++] = (u64)PyBytes_AS_STRING(o);
        else {
            PyErr_Format(PyExc_TypeError, "call: argument %zd, a pointer, is a %.100s", i, Py_TYPE(o)->tp_name);
            return nullptr;
        }
        if (PyErr_Occurred()) return nullptr;
    }
    if (!address) {
        PyErr_SetString(PyExc_ValueError, "call: a null address");
        return nullptr;
    }
    const Launcher fn = reinterpret_cast<Launcher>(address);
    int r;
    Py_BEGIN_ALLOW_THREADS
    r = fn(v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7], v[8], v[9], v[10], v[11], v[12], v[13], v[14], v[15], v[16], v[17],
           v[18], v[19], v[20], v[21], v[22], v[23], v[24], v[25], v[26], v[27], v[28], v[29], v[30], v[31], v[32], v[33], v[34],
           v[35], v[36], v[37], v[38], v[39], v[40], v[41], v[42], v[43], v[44], v[45], v[46], v[47], f[0], f[1], f[2], f[3],
           f[4], f[5], f[6], f[7]);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(r);
    END_HANDLE_TH_ERRORS
}

static PyMethodDef methods[] = {
    {"call", (PyCFunction)(void (*)(void))ft_call, METH_FASTCALL, "call(address, kinds, *arguments) -> int"},
    {"fits", (PyCFunction)(void (*)(void))ft_fits, METH_FASTCALL, "is it a contiguous tensor of this type on this device, of these sizes (None: any)?"},
    {"fits_all", (PyCFunction)(void (*)(void))ft_fits_all, METH_FASTCALL, "are they all contiguous tensors of their types on this device, of their sizes?"},
    {"rows", (PyCFunction)(void (*)(void))ft_rows, METH_FASTCALL, "a matrix's rows and how far they are apart; None if it does not fit"},
    {"apart", (PyCFunction)(void (*)(void))ft_apart, METH_FASTCALL, "do two matrices, of which so many columns are used, share no memory?"},
    {"addresses", (PyCFunction)(void (*)(void))ft_addresses, METH_FASTCALL, "where tensors of one kind are, as bytes; None if they are not of one kind"},
    {"empty", (PyCFunction)(void (*)(void))ft_empty, METH_FASTCALL, "a new tensor of this type, on this device, of these sizes"},
    {nullptr, nullptr, 0, nullptr}};

static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "fasttensor", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

PyMODINIT_FUNC PyInit_fasttensor(void) { return PyModule_Create(&module); }
