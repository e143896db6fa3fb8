// Python entry points of the layer norm, AdamW and 8-bit product (stdiff_amd/ops.py documents them): arguments are checked and
// the C ABI is called without a detour through interpreted code, which took longer than the kernels of small calls (layer
// norm of one token: 8.5 us through ctypes, of which 1.8 are the kernel).  Refusals are ValueError / TypeError with the
// argument's name, raised before anything is allocated or launched; tensors that are not on a GPU come last, so that
// everything else is refused without one too.
#include <Python.h>
#include <ATen/ATen.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <vector>

#include "../../include/stdiff_hip.h"

namespace {

struct Refusal {
    PyObject* type;                        // NULL: a Python error is set already
    std::string text;
};
template <typename... A> [[noreturn]] void refuse(PyObject* type, const A&... a) { throw Refusal{type, c10::str(a...)}; }

// ---------------------------------------------------------------- the two libraries (bf16 and fp16 as the 16-bit type)
struct Library {
    decltype(&stdiff_layer_norm) layer_norm;
    decltype(&stdiff_layer_norm_bwd_workspace) layer_norm_bwd_workspace;
    decltype(&stdiff_layer_norm_bwd) layer_norm_bwd;
    decltype(&stdiff_adamw_multi_workspace) adamw_multi_workspace;
    decltype(&stdiff_adamw_multi) adamw_multi;
    decltype(&stdiff_quantize_rows) quantize_rows;
    decltype(&stdiff_gemm_i8) gemm_i8;
    decltype(&stdiff_error_string) error_string;
};
constexpr int ENTRIES = sizeof(Library) / sizeof(void*);
Library libraries[2];
PyObject *loader = nullptr, *stdiff_error = nullptr;

const Library& library(bool fp16) {
    Library& l = libraries[fp16];
    if (!l.layer_norm) {
        PyObject* t = loader ? PyObject_CallFunction(loader, "i", (int)fp16) : nullptr;
        if (!t) {
            if (!loader) refuse(PyExc_RuntimeError, "stdiff_amd._bind is not set up");
            throw Refusal{nullptr, ""};
        }
        void* at[ENTRIES];
        bool ok = PyTuple_Check(t) && PyTuple_GET_SIZE(t) == ENTRIES;
        for (int i = 0; ok && i < ENTRIES; ++i) {
            at[i] = PyLong_AsVoidPtr(PyTuple_GET_ITEM(t, i));
            ok = at[i] != nullptr;
        }
        Py_DECREF(t);
        if (!ok) refuse(PyExc_RuntimeError, "stdiff_amd._bind: a library lacks entry points");
        memcpy(&l, at, sizeof(l));
    }
    return l;
}
void check(const Library& l, int rc) {
    if (rc == STDIFF_OK) return;
    refuse(rc < 0 && rc != STDIFF_ERR_STATE ? PyExc_ValueError : stdiff_error, "stdiff_hip: ", l.error_string(rc), " (status ", rc, ")");
}

// ---------------------------------------------------------------- arguments
using at::ScalarType;
using at::Tensor;

const Tensor* tensor(PyObject* o, const char* name, bool needed = false) {
    if (o == Py_None && !needed) return nullptr;
    if (!THPVariable_Check(o)) refuse(PyExc_TypeError, name, ": a tensor is needed, got ", Py_TYPE(o)->tp_name);
    return &THPVariable_Unpack(o);
}
double number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Refusal{nullptr, ""};
    return v;
}
ScalarType dtype(PyObject* o, ScalarType otherwise) {
    if (o == Py_None) return otherwise;
    if (!THPDtype_Check(o)) refuse(PyExc_TypeError, "a torch.dtype is needed, got ", Py_TYPE(o)->tp_name);
    return reinterpret_cast<THPDtype*>(o)->scalar_type;
}

// the 16-bit type of a call, which chooses the library
struct Half {
    bool bf16 = false, fp16 = false;
    int code(ScalarType t) {               // the C ABI's code of a type
        if (t == ScalarType::Float) return STDIFF_F32;
        if (t == ScalarType::BFloat16) bf16 = true;
        else if (t == ScalarType::Half) fp16 = true;
        else refuse(PyExc_TypeError, "unsupported dtype ", t);
        if (bf16 && fp16) refuse(PyExc_TypeError, "float16 and bfloat16 tensors in one stdiff_hip call");
        return STDIFF_BF16;
    }
};

int64_t read_ld(const Tensor& t, const char* name, const Tensor* like = nullptr) {
    if (t.dim() != 2 || (like && t.sizes() != like->sizes()))
        refuse(PyExc_ValueError, name, ": a matrix is needed", like ? c10::str(" of ", like->sizes()) : std::string(), ", got ", t.sizes());
    if (t.size(0) > INT_MAX || t.size(1) > INT_MAX) refuse(PyExc_ValueError, name, ": too large, ", t.sizes());
    if (t.size(1) > 1 && t.stride(1) != 1) refuse(PyExc_ValueError, name, ": the elements of a row have to be neighbours, got strides ", t.strides());
    return t.size(0) > 1 ? t.stride(0) : t.size(1);
}
int64_t write_ld(const Tensor& t, const char* name) {
    const int64_t ld = read_ld(t, name);
    if (ld < t.size(1)) refuse(PyExc_ValueError, name, ": rows of an output may not overlap, got strides ", t.strides());
    return ld;
}
void* vector(const Tensor* t, const char* name, int64_t n, bool any_float = false) {
    if (!t) return nullptr;
    const ScalarType k = t->scalar_type();
    const bool fits = k == ScalarType::Float || (any_float && (k == ScalarType::BFloat16 || k == ScalarType::Half));
    if (t->dim() != 1 || t->numel() != n || !fits || !t->is_contiguous())
        refuse(PyExc_ValueError, name, ": a contiguous vector of ", n, any_float ? " floating elements" : " float32 elements", " is needed, got ", t->sizes(), " ", k);
    return t->data_ptr();
}
// rows that begin on 16-byte borders and may be touched up to the next border behind their end
int64_t rows16(const Tensor& t, const char* name) {
    if (t.scalar_type() != ScalarType::Char) refuse(PyExc_TypeError, name, ": int8 is needed, got ", t.scalar_type());
    const int64_t rows = t.dim() == 2 ? t.size(0) : 0, k = t.dim() == 2 ? t.size(1) : 0, kp = (k + 15) / 16 * 16;
    const int64_t ld = rows == 1 ? (read_ld(t, name), kp) : read_ld(t, name);
    if (rows && (ld % 16 || ld < kp || (uintptr_t)t.data_ptr() % 16 || t.storage_offset() + (rows - 1) * ld + kp > (int64_t)t.storage().nbytes()))
        refuse(PyExc_ValueError, name, ": rows have to begin on 16-byte borders and to reach the next border behind their end in memory, "
               "as quantize_rows lays them out; got shape ", t.sizes(), ", strides ", t.strides());
    return ld;
}

// Memory that a call reads or writes: rows of `width` bytes, `ld` bytes apart (a vector is one row).
struct Area {
    const char* name;
    uintptr_t at;
    int64_t rows, ld, width;               // no rows: nothing
    ScalarType type;
    bool empty() const { return rows <= 0 || width <= 0; }
    uintptr_t end() const { return at + (rows - 1) * ld + width; }
};
// columns: how many of a row are touched, where that is not the tensor's own number (padding included)
Area matrix(const Tensor* t, const char* name, int64_t ld, int64_t columns = -1) {
    if (!t || !t->numel()) return {name, 0, 0, 0, 0, ScalarType::Undefined};
    const int64_t size = t->element_size();
    return {name, (uintptr_t)t->data_ptr(), ld ? t->size(0) : 1, ld * size, (columns < 0 ? t->size(1) : columns) * size, t->scalar_type()};
}
Area flat(const Tensor* t, const char* name) {
    if (!t || !t->numel()) return {name, 0, 0, 0, 0, ScalarType::Undefined};
    const int64_t bytes = (int64_t)t->nbytes();
    return {name, (uintptr_t)t->data_ptr(), 1, bytes, bytes, t->scalar_type()};
}
// Side by side in the rows of one buffer, or in the gaps between rows, two areas are apart.
bool meet(const Area& a, const Area& b) {
    if (a.empty() || b.empty() || a.end() <= b.at || b.end() <= a.at) return false;
    if (a.rows == 1 && b.rows > 1) return meet(b, a);
    if (b.rows == 1) {                     // the first row of a that ends behind b's beginning: does it begin before b's end?
        const int64_t behind = (int64_t)(b.at - a.at) - a.width, row = behind < 0 ? 0 : behind / a.ld + 1;
        return row < a.rows && a.at + row * a.ld < b.end();
    }
    if (a.ld == b.ld) {
        const int64_t off = (int64_t)(b.at - a.at) % a.ld, d = off < 0 ? off + a.ld : off;
        if (d >= a.width && d + b.width <= a.ld) return false;
    }
    return true;
}
// Outputs share no memory with what a call reads, nor with each other, but where an operator may work in place: then they are
// the same elements.
void keep_apart(const Area& out, const Area& in, bool in_place = false) {
    if (!meet(out, in)) return;
    if (in_place && out.at == in.at && out.ld == in.ld && out.type == in.type) return;
    refuse(PyExc_ValueError, out.name, " and ", in.name, " share memory", in_place ? " and are not the same elements" : "");
}

// The device that all tensors of a call are on is current while this lives; its current stream.
struct Place {
    int device, was;
    hipStream_t stream;
    Place(const Tensor& first, std::initializer_list<const Tensor*> rest) {
        for (const Tensor* t : rest)
            if (t && t->device() != first.device()) {
                if (t->is_cuda() && first.is_cuda()) refuse(PyExc_ValueError, "tensors on ", first.device(), " and ", t->device(), " in one call");
                not_here();
            }
        if (!first.is_cuda()) not_here();
        enter(first.get_device());
    }
    explicit Place(int dev) { enter(dev); }
    Place(const Place&) = delete;
    ~Place() {
        if (was == device) return;
        try {
            c10::hip::set_device((c10::DeviceIndex)was);
        } catch (...) {                    // a destructor's exception would end the process
        }
    }
    [[noreturn]] static void not_here() { refuse(PyExc_RuntimeError, "stdiff_amd runs on MI355X only: got a CPU tensor (no CPU fallback exists)"); }

private:
    void enter(int dev) {
        device = dev;
        was = c10::hip::current_device();
        if (was != device) c10::hip::set_device((c10::DeviceIndex)device);
        stream = c10::hip::getCurrentHIPStream((c10::DeviceIndex)device).stream();
    }
};

// autograd refuses a backward through what it had saved of a tensor that was written since
void written(const Tensor* t) {
    if (t && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}
PyObject* same(PyObject* given, const Tensor& made) {
    if (given != Py_None) {
        Py_INCREF(given);
        return given;
    }
    return made.defined() ? THPVariable_Wrap(made) : Py_NewRef(Py_None);
}
Tensor floats(const Tensor& like, int64_t n) { return at::empty({n}, like.options().dtype(ScalarType::Float)); }

// ---------------------------------------------------------------- entry points
PyObject* layer_norm(PyObject* const* a) {
    const Tensor &x = *tensor(a[0], "x", true), *w = tensor(a[1], "weight"), *b = tensor(a[2], "bias"), *given = tensor(a[4], "out"),
                 *mean = tensor(a[6], "mean"), *rstd = tensor(a[7], "rstd");
    const double eps = number(a[3]);
    const int64_t ldx = read_ld(x, "x"), R = x.size(0), H = x.size(1);
    if (given && given->sizes() != x.sizes()) read_ld(*given, "out", &x);
    int64_t ldy = given ? write_ld(*given, "out") : H;
    if (w && b && w->scalar_type() != b->scalar_type())
        refuse(PyExc_TypeError, "weight is ", w->scalar_type(), ", bias ", b->scalar_type(), ": one dtype is needed");
    void *wp = vector(w, "weight", H, true), *bp = vector(b, "bias", H, true), *mp = vector(mean, "mean", R), *rp = vector(rstd, "rstd", R);
    const Area ax = matrix(&x, "x", ldx), ao = matrix(given, "out", ldy), am = flat(mean, "mean"), ar = flat(rstd, "rstd");
    const Area aw = flat(w, "weight"), ab = flat(b, "bias");
    keep_apart(ao, ax, true);
    keep_apart(am, ar);
    for (const Area* in : {&aw, &ab, &am, &ar}) keep_apart(ao, *in);
    for (const Area* stat : {&am, &ar})
        for (const Area* in : {&ax, &aw, &ab}) keep_apart(*stat, *in);
    Half half;
    const ScalarType yt = given ? given->scalar_type() : dtype(a[5], x.scalar_type());
    const int xc = half.code(x.scalar_type()), yc = half.code(yt), wc = w ? half.code(w->scalar_type()) : b ? half.code(b->scalar_type()) : STDIFF_F32;
    Place here(x, {w, b, given, mean, rstd});
    const Tensor out = given ? *given : at::empty({R, H}, x.options().dtype(yt));
    const Library& l = library(half.fp16);
    check(l, l.layer_norm(x.data_ptr(), ldx, xc, wp, bp, wc, (float)eps, out.data_ptr(), ldy, yc, (float*)mp, (float*)rp, (int)R, (int)H, here.stream));
    for (const Tensor* t : {given, mean, rstd}) written(t);
    return same(a[4], out);
}

PyObject* layer_norm_bwd(PyObject* const* a) {
    const Tensor &dy = *tensor(a[0], "dy", true), &x = *tensor(a[1], "x", true), *mean = tensor(a[2], "mean"), *rstd = tensor(a[3], "rstd"),
                 *w = tensor(a[4], "weight"), *dx_ = tensor(a[5], "dx"), *dw_ = tensor(a[6], "dweight"), *db_ = tensor(a[7], "dbias"),
                 *ws_ = tensor(a[9], "workspace");
    const int accumulate = PyObject_IsTrue(a[8]);
    if (accumulate < 0) throw Refusal{nullptr, ""};
    const int64_t ldx = read_ld(x, "x"), lddy = read_ld(dy, "dy", &x), R = x.size(0), H = x.size(1);
    if (accumulate && !dw_ && !db_) refuse(PyExc_ValueError, "accumulate: there is no dweight or dbias to add to");
    if (!mean || !rstd) refuse(PyExc_ValueError, "mean and rstd of the forward are needed");
    if (dx_ && dx_->scalar_type() != x.scalar_type()) refuse(PyExc_TypeError, "dx is ", dx_->scalar_type(), ", x ", x.scalar_type());
    if (dx_) read_ld(*dx_, "dx", &x);
    const int64_t lddx = dx_ ? write_ld(*dx_, "dx") : H;
    void *wp = vector(w, "weight", H, true), *mp = vector(mean, "mean", R), *rp = vector(rstd, "rstd", R);
    vector(dw_, "dweight", H);
    vector(db_, "dbias", H);
    if (ws_ && !ws_->is_contiguous()) refuse(PyExc_ValueError, "workspace: a contiguous tensor is needed");
    const Area ax = matrix(&x, "x", ldx), ady = matrix(&dy, "dy", lddy), adx = matrix(dx_, "dx", lddx), adw = flat(dw_, "dweight"), adb = flat(db_, "dbias");
    const Area aw = flat(w, "weight"), am = flat(mean, "mean"), ar = flat(rstd, "rstd"), aws = flat(ws_, "workspace");
    keep_apart(adx, ax, true);
    keep_apart(adx, ady, true);
    keep_apart(adw, adb);
    for (const Area* o : {&aw, &am, &ar, &adw, &adb}) keep_apart(adx, *o);
    for (const Area* o : {&adw, &adb})
        for (const Area* in : {&ax, &ady, &aw, &am, &ar}) keep_apart(*o, *in);
    for (const Area* o : {&ax, &ady, &adx, &aw, &am, &ar, &adw, &adb}) keep_apart(aws, *o);
    Half half;
    const int xc = half.code(x.scalar_type()), dc = half.code(dy.scalar_type()), wc = w ? half.code(w->scalar_type()) : STDIFF_F32;
    Place here(x, {&dy, mean, rstd, w, dx_, dw_, db_, ws_});
    const Library& l = library(half.fp16);
    const Tensor dx = dx_ ? *dx_ : at::empty({R, H}, x.options());
    const bool both = w && !accumulate;    // with a weight both gradients are formed
    const Tensor dw = dw_ ? *dw_ : both ? floats(x, H) : Tensor(), db = db_ ? *db_ : both ? floats(x, H) : Tensor();
    Tensor ws = ws_ ? *ws_ : Tensor();
    if (!ws_ && (dw.defined() || db.defined())) {
        const int64_t need = l.layer_norm_bwd_workspace((int)R, (int)H, xc, dc);
        if (need > 0) ws = floats(x, need / 4);
    }
    check(l, l.layer_norm_bwd(dy.data_ptr(), lddy, dc, x.data_ptr(), ldx, xc, (float*)mp, (float*)rp, wp, wc, dx.data_ptr(), lddx,
                              dw.defined() ? (float*)dw.data_ptr() : nullptr, db.defined() ? (float*)db.data_ptr() : nullptr, accumulate,
                              ws.defined() ? (float*)ws.data_ptr() : nullptr, ws.defined() ? (long long)ws.nbytes() : 0, (int)R, (int)H, here.stream));
    for (const Tensor* t : {dx_, dw_, db_}) written(t);
    PyObject* r = PyTuple_New(3);
    if (!r) throw Refusal{nullptr, ""};
    PyTuple_SET_ITEM(r, 0, same(a[5], dx));
    PyTuple_SET_ITEM(r, 1, same(a[6], dw));
    PyTuple_SET_ITEM(r, 2, same(a[7], db));
    return r;
}

PyObject* quantize_rows(PyObject* const* a) {
    const Tensor &x = *tensor(a[0], "x", true), *out_ = tensor(a[1], "out"), *scale_ = tensor(a[2], "scale");
    const int64_t ldx = read_ld(x, "x"), R = x.size(0), K = x.size(1), kp = (K + 15) / 16 * 16;
    if (out_) read_ld(*out_, "out", &x);
    const int64_t ldq = out_ ? rows16(*out_, "out") : kp;
    vector(scale_, "scale", R);
    const Area ax = matrix(&x, "x", ldx), aq = matrix(out_, "out", ldq, kp), as = flat(scale_, "scale");
    keep_apart(aq, ax);
    keep_apart(aq, as);
    keep_apart(as, ax);
    Half half;
    const int xc = half.code(x.scalar_type());
    Place here(x, {out_, scale_});
    Tensor out = out_ ? *out_ : at::empty({R, kp}, x.options().dtype(ScalarType::Char));
    if (!out_ && kp != K) out = out.narrow(1, 0, K);
    const Tensor scale = scale_ ? *scale_ : floats(x, R);
    const Library& l = library(half.fp16);
    check(l, l.quantize_rows(x.data_ptr(), ldx, xc, out.data_ptr(), ldq, (float*)scale.data_ptr(), (int)R, (int)K, here.stream));
    for (const Tensor* t : {out_, scale_}) written(t);
    PyObject* r = PyTuple_New(2);
    if (!r) throw Refusal{nullptr, ""};
    PyTuple_SET_ITEM(r, 0, same(a[1], out));
    PyTuple_SET_ITEM(r, 1, same(a[2], scale));
    return r;
}

PyObject* gemm_i8(PyObject* const* a) {
    const Tensor &A = *tensor(a[0], "A", true), *sa = tensor(a[1], "a_scale"), &W = *tensor(a[2], "W", true), *sw = tensor(a[3], "w_scale"),
                 *bias = tensor(a[4], "bias"), *out_ = tensor(a[5], "out");
    const int64_t lda = rows16(A, "A"), ldw = rows16(W, "W"), M = A.size(0), K = A.size(1), N = W.size(0);
    if (W.size(1) != K) refuse(PyExc_ValueError, "A has ", K, " columns, W ", W.size(1));
    if (!sa || !sw) refuse(PyExc_ValueError, "a_scale and w_scale are needed");
    stdiff_gemm_i8_args g = {};
    g.M = (int)M, g.N = (int)N, g.K = (int)K;
    g.A = A.data_ptr(), g.lda = lda, g.W = W.data_ptr(), g.ldw = ldw;
    g.a_scale = (const float*)vector(sa, "a_scale", M), g.w_scale = (const float*)vector(sw, "w_scale", N), g.bias = (const float*)vector(bias, "bias", N);
    if (out_ && (out_->dim() != 2 || out_->size(0) != M || out_->size(1) != N))
        refuse(PyExc_ValueError, "out: a matrix of [", M, ", ", N, "] is needed, got ", out_->sizes());
    g.ldc = out_ ? write_ld(*out_, "out") : N;
    const Area ao = matrix(out_, "out", g.ldc);
    keep_apart(ao, matrix(&A, "A", lda));
    keep_apart(ao, matrix(&W, "W", ldw));
    keep_apart(ao, flat(sa, "a_scale"));
    keep_apart(ao, flat(sw, "w_scale"));
    keep_apart(ao, flat(bias, "bias"));
    Half half;
    const ScalarType ct = out_ ? out_->scalar_type() : dtype(a[6], ScalarType::Float);
    g.c_dtype = half.code(ct);
    Place here(A, {sa, &W, sw, bias, out_});
    const Tensor out = out_ ? *out_ : at::empty({M, N}, A.options().dtype(ct));
    g.C = out.data_ptr();
    const Library& l = library(half.fp16);
    check(l, l.gemm_i8(&g, here.stream));
    written(out_);
    return same(a[5], out);
}

// ---- AdamW: the table of an AdamWTensors, in a capsule
struct Table {
    std::vector<stdiff_adamw_tensor> rows;
    std::vector<int64_t> sizes;
    std::vector<c10::Storage> memory;      // alive even where a tensor is given other memory
    std::vector<std::pair<Tensor, void*>> states;
    std::vector<std::pair<uintptr_t, uintptr_t>> taken;    // beginning and end of all of it, in order
    Half half;
    int bits = 32, device = -1;
};
// Whether memory lies apart from a table's.  What was asked about last lies in some gap between the parameters and states; the next
// gradient is often in the same one, and no search is needed.
struct Apart {
    const Table& t;
    uintptr_t from = 1, to = 0;
    bool operator()(const Area& a) {
        if (a.empty() || (a.at >= from && a.end() <= to)) return true;
        const auto next = std::upper_bound(t.taken.begin(), t.taken.end(), a.at, [](uintptr_t v, const auto& r) { return v < r.first; });
        const uintptr_t below = next == t.taken.begin() ? 0 : (next - 1)->second, above = next == t.taken.end() ? UINTPTR_MAX : next->first;
        if (a.at < below || a.end() > above) return false;
        from = below, to = above;
        return true;
    }
};
constexpr const char* TABLE = "stdiff_amd.adamw_table";

struct Items {                             // of a Python sequence
    PyObject* fast;
    Py_ssize_t n;
    Items(PyObject* o, const char* name) : fast(PySequence_Fast(o, name)), n(0) {
        if (!fast) throw Refusal{nullptr, ""};
        n = PySequence_Fast_GET_SIZE(fast);
    }
    Items(const Items&) = delete;
    ~Items() { Py_XDECREF(fast); }
    PyObject* operator[](Py_ssize_t i) const { return PySequence_Fast_GET_ITEM(fast, i); }
};

PyObject* adamw_table(PyObject* const* a) {
    const char* names[] = {"param", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale"};
    const Items p(a[0], "params"), m(a[1], "exp_avg"), v(a[2], "exp_avg_sq"), ms(a[3], "exp_avg_scale"), vs(a[4], "exp_avg_sq_scale"),
        decay(a[5], "weight_decay");
    for (const Items* k : {&m, &v, &ms, &vs, &decay})
        if (k->n != p.n) refuse(PyExc_ValueError, "adamw_multi_args: lists of different lengths");
    std::unique_ptr<Table> t(new Table);
    const Tensor *first = nullptr, *away = nullptr;
    for (Py_ssize_t i = 0; i < p.n; ++i) {
        const Tensor* k[5];
        int j = 0;
        for (const Items* s : {&p, &m, &v, &ms, &vs}) {
            k[j] = tensor((*s)[i], names[j], j < 3);
            if (k[j]) {
                if (!first) first = k[j];
                if (k[j]->device() != first->device()) away = k[j];
            }
            ++j;
        }
        const bool eight = k[1]->scalar_type() == ScalarType::Float8_e4m3fn;
        if (i == 0) t->bits = eight ? 8 : 32;
        const ScalarType kind = t->bits == 8 ? ScalarType::Float8_e4m3fn : ScalarType::Float;
        if (k[1]->scalar_type() != kind || k[2]->scalar_type() != kind)
            refuse(PyExc_TypeError, "tensor ", i, ": states are ", k[1]->scalar_type(), " and ", k[2]->scalar_type(), ", ", kind, " is needed");
        const int64_t n = k[0]->numel();
        if (k[1]->numel() != n || k[2]->numel() != n)
            refuse(PyExc_ValueError, "tensor ", i, ": states of ", k[1]->numel(), " and ", k[2]->numel(), " elements for ", n, " parameters");
        for (j = 0; j < 3; ++j)
            if (!k[j]->is_contiguous()) refuse(PyExc_ValueError, "tensor ", i, ": ", names[j], " is not contiguous");
        if (t->bits == 32 && (k[3] || k[4])) refuse(PyExc_ValueError, "32-bit states have no scales");
        if (t->bits == 8 && (!k[3] || !k[4])) refuse(PyExc_ValueError, "8-bit states need exp_avg_scale and exp_avg_sq_scale");
        stdiff_adamw_tensor r = {};
        r.param = k[0]->data_ptr(), r.exp_avg = k[1]->data_ptr(), r.exp_avg_sq = k[2]->data_ptr();
        r.exp_avg_scale = (float*)vector(k[3], "exp_avg_scale", (n + 255) / 256);
        r.exp_avg_sq_scale = (float*)vector(k[4], "exp_avg_sq_scale", (n + 255) / 256);
        r.n = n, r.param_dtype = t->half.code(k[0]->scalar_type()), r.weight_decay = (float)number(decay[i]);
        t->rows.push_back(r);
        t->sizes.push_back(n);
        for (j = 0; j < 5; ++j)
            if (k[j]) {
                t->memory.push_back(k[j]->storage());
                if (j) t->states.push_back({*k[j], k[j]->data_ptr()});
                if (k[j]->numel()) t->taken.push_back({(uintptr_t)k[j]->data_ptr(), (uintptr_t)k[j]->data_ptr() + k[j]->nbytes()});
            }
    }
    if (first) {
        if (away && away->is_cuda() && first->is_cuda()) refuse(PyExc_ValueError, "tensors on ", first->device(), " and ", away->device(), " in one call");
        if (away || !first->is_cuda()) Place::not_here();
        t->device = first->get_device();
    }
    std::sort(t->taken.begin(), t->taken.end());
    for (size_t i = 1; i < t->taken.size(); ++i)
        if (t->taken[i - 1].second > t->taken[i].first)
            refuse(PyExc_ValueError, "adamw_multi_args: two of the parameters and states share memory");
    PyObject* c = PyCapsule_New(t.get(), TABLE, [](PyObject* o) { delete (Table*)PyCapsule_GetPointer(o, TABLE); });
    if (!c) throw Refusal{nullptr, ""};
    t.release();
    return c;
}

PyObject* adamw_multi(PyObject* const* a) {
    Table* t = (Table*)PyCapsule_GetPointer(a[0], TABLE);
    if (!t) throw Refusal{nullptr, ""};
    const Items params(a[1], "params"), grads(a[2], "grads");
    const Py_ssize_t n = (Py_ssize_t)t->rows.size();
    if (params.n != n || grads.n != n) refuse(PyExc_ValueError, "adamw_multi: ", grads.n, " gradients for ", n, " parameters");
    const Tensor &step = *tensor(a[3], "step_dev", true), *norm = tensor(a[10], "norm"), *ws_ = tensor(a[11], "workspace");
    stdiff_adamw_multi_args g = {};
    g.lr = number(a[4]), g.max_norm = a[5] == Py_None ? 0.0 : number(a[5]), g.grad_scale = number(a[6]);
    g.beta1 = number(a[7]), g.beta2 = number(a[8]), g.eps = number(a[9]);
    if (a[5] != Py_None && !(g.max_norm > 0.0)) refuse(PyExc_ValueError, "max_norm has to be positive (or None), got ", g.max_norm);
    if (step.scalar_type() != ScalarType::Int || step.numel() != 1) refuse(PyExc_ValueError, "step_dev: one int32 element is needed, got ", step.sizes(), " ", step.scalar_type());
    g.norm = (float*)vector(norm, "norm", 1);
    if (ws_ && !ws_->is_contiguous()) refuse(PyExc_ValueError, "workspace: a contiguous tensor is needed");
    for (const auto& s : t->states)
        if (s.first.data_ptr() != s.second) refuse(PyExc_ValueError, "adamw_multi: a state was given other memory since adamw_multi_args");
    const Area cells[] = {flat(ws_, "workspace"), flat(norm, "norm"), flat(&step, "step_dev")};
    Apart apart{*t};
    for (int i = 0; i < 3; ++i) {
        if (!apart(cells[i])) refuse(PyExc_ValueError, "adamw_multi: ", cells[i].name, " shares memory with a parameter or state");
        for (int j = i + 1; j < 3; ++j) keep_apart(cells[i], cells[j]);
    }
    Half half = t->half;
    std::vector<stdiff_adamw_tensor> rows = t->rows;       // of this call: two calls do not see each other's gradients
    for (Py_ssize_t i = 0; i < n; ++i) {
        const Tensor& p = *tensor(params[i], "param", true);
        if (p.data_ptr() != t->rows[i].param) refuse(PyExc_ValueError, "adamw_multi: parameter ", i, " was given other memory since adamw_multi_args");
        const Tensor* d = tensor(grads[i], "gradient");
        if (!d) {
            rows[i].n = 0;
            continue;
        }
        if (d->numel() != t->sizes[i] || !d->is_contiguous())
            refuse(PyExc_ValueError, "adamw_multi: gradient ", i, ": ", t->sizes[i], " contiguous elements are needed, got ", d->sizes(), " with strides ", d->strides());
        if (!d->is_cuda() || d->get_device() != t->device) refuse(PyExc_ValueError, "adamw_multi: gradient ", i, " is on ", d->device(), ", its parameter on device ", t->device);
        rows[i].grad = d->data_ptr();
        rows[i].grad_dtype = half.code(d->scalar_type());
        const int64_t bytes = t->sizes[i] * (rows[i].grad_dtype == STDIFF_F32 ? 4 : 2);
        const Area grad = {"gradient", (uintptr_t)rows[i].grad, bytes ? 1 : 0, bytes, bytes, ScalarType::Undefined};
        if (!apart(grad)) refuse(PyExc_ValueError, "adamw_multi: gradient ", i, " shares memory with a parameter or state");
        for (const Area& c : cells)
            if (bytes && !c.empty() && c.at < grad.at + bytes && grad.at < c.end())
                refuse(PyExc_ValueError, "adamw_multi: ", c.name, " and gradient ", i, " share memory");
    }
    Place here(step, {norm, ws_});
    if (n && here.device != t->device) refuse(PyExc_ValueError, "step_dev is on ", step.device(), ", the parameters on device ", t->device);
    const Library& l = library(half.fp16);
    const Tensor ws = ws_ ? *ws_ : floats(step, l.adamw_multi_workspace((int)n) / 4);
    g.tensors = rows.data(), g.n_tensors = (int)n, g.state_bits = t->bits;
    g.step_dev = (int32_t*)step.data_ptr(), g.workspace = (float*)ws.data_ptr(), g.workspace_bytes = (long long)ws.nbytes();
    check(l, l.adamw_multi(&g, here.stream));
    // who keeps copies of the parameters (DiT_stDiff's packed operands) sees by their version counters that they changed
    const size_t per = t->bits == 8 ? 4 : 2;               // states of a tensor
    for (Py_ssize_t i = 0; i < n; ++i)
        if (rows[i].n) {
            written(&THPVariable_Unpack(params[i]));
            for (size_t j = 0; j < per; ++j) written(&t->states[i * per + j].first);
        }
    written(&step);
    written(norm);
    return Py_NewRef(Py_None);
}

PyObject* setup(PyObject* const* a) {
    Py_XDECREF(loader);
    Py_XDECREF(stdiff_error);
    loader = Py_NewRef(a[0]);
    stdiff_error = Py_NewRef(a[1]);
    return Py_NewRef(Py_None);
}

// no exception leaves an entry point
template <PyObject* (*F)(PyObject* const*), int N> PyObject* entry(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != N) {
        PyErr_Format(PyExc_TypeError, "stdiff_amd._bind: %d arguments are needed, got %zd", N, n);
        return nullptr;
    }
    try {
        return F(a);
    } catch (const Refusal& r) {
        if (r.type) PyErr_SetString(r.type, r.text.c_str());
    } catch (const std::bad_alloc&) {
        PyErr_NoMemory();
    } catch (const c10::OutOfMemoryError& e) {
        PyObject* torch = PyImport_ImportModule("torch");
        PyObject* type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
        PyErr_Clear();
        PyErr_SetString(type ? type : PyExc_RuntimeError, e.what_without_backtrace());
        Py_XDECREF(type);
        Py_XDECREF(torch);
    } catch (const c10::Error& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}
#define ENTRY(name, args) {#name, (PyCFunction)(void*)entry<name, args>, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {ENTRY(setup, 2), ENTRY(layer_norm, 8), ENTRY(layer_norm_bwd, 10), ENTRY(quantize_rows, 3), ENTRY(gemm_i8, 7),
                         ENTRY(adamw_table, 6), ENTRY(adamw_multi, 12), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_bind", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__bind() { return PyModule_Create(&module); }
