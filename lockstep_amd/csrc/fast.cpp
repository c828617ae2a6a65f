// The plain calls of the Python modules in native code: argument checks, output
// allocation and the launches of one public call in one extension call.
//
// Issued from Python through ctypes, a call costs 9 to 50 us of interpreter
// time (shape tests, torch.empty, stream lookups, argument conversion) for 4
// to 30 us of kernels: the M = 1 weight product took 14.2 us for an 8.3 us
// kernel, a small MXFP4Linear forward 48 us for 30.  Every function here
// takes the arguments of its Python caller and handles the form that programs
// pass in a loop -- exact torch tensors on one GPU, the layouts the kernels
// read in place -- and returns None for anything else (other strides,
// alignments, types, empty shapes, wrong arguments, tensor subclasses,
// functorch wrappers, calls under a dispatch mode or a functorch transform):
// the caller then runs its general path, which converts,
// or raises as it always has.  The launches go through the same C ABI
// (include/lsmx.h), on torch's current stream, with the GIL released.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <ATen/autocast_mode.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>

#include <cmath>

#include "../../include/lsmx.h"

namespace {

using at::Tensor;

PyObject *g_error = nullptr;      // _capi.check(rc): raises LsmxError
PyObject *g_workspace = nullptr;  // _capi.workspace(device, nbytes)
PyObject *g_epoch = nullptr;      // _capi.next_epoch()

// A dispatch mode or a functorch transform around the call: at::empty gives
// that mode's tensors, which may have no data pointer.
bool transformed() {
    return c10::impl::TorchDispatchModeTLS::any_modes_set() ||
           c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode);
}

// A plain GPU tensor: exactly torch.Tensor (or Parameter), with storage, and no
// dispatch key that changes what its data means.
const Tensor *plain(PyObject *o) {
    if (!THPVariable_CheckExact(o) || transformed()) return nullptr;
    const Tensor &t = THPVariable_Unpack(o);
    if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || !t.has_storage()) return nullptr;
    constexpr c10::DispatchKeySet odd{c10::DispatchKey::Python, c10::DispatchKey::Conjugate, c10::DispatchKey::Negative,
                                      c10::DispatchKey::ZeroTensor, c10::DispatchKey::FuncTorchBatched,
                                      c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Functionalize};
    return t.key_set().has_any(odd) ? nullptr : &t;
}

bool al(const Tensor &t, uintptr_t a) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % a == 0; }

// rows of a 2-D tensor with unit stride and 16-byte aligned starts
bool rows16(const Tensor &t) {
    return t.dim() == 2 && t.stride(1) == 1 && al(t, 16) && t.stride(0) >= t.size(1) &&
           (t.stride(0) * t.element_size()) % 16 == 0;
}

int dtype_of(at::ScalarType s) {
    return s == at::kFloat ? LSMX_F32 : s == at::kBFloat16 ? LSMX_BF16 : s == at::kHalf ? LSMX_F16 : -1;
}

// scalar type of a torch.dtype argument, or Undefined (None included: only
// weight()'s callers give it a meaning)
at::ScalarType out_type(PyObject *o) {
    if (!THPDtype_Check(o)) return at::ScalarType::Undefined;
    const at::ScalarType s = reinterpret_cast<THPDtype *>(o)->scalar_type;
    return dtype_of(s) >= 0 ? s : at::ScalarType::Undefined;
}

Tensor make(at::IntArrayRef shape, at::ScalarType s, const Tensor &like) {
    return at::empty(shape, at::TensorOptions().dtype(s).device(like.device()));
}
void *stream_of(const Tensor &t) {
    return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

// Holds the GIL released; takes it back when a C++ exception leaves the scope
// too, so that HANDLE_TH_ERRORS sets the Python error with it held.
struct NoGil {
    PyThreadState *s = PyEval_SaveThread();
    ~NoGil() { PyEval_RestoreThread(s); }
};

// Runs launches with the GIL released; returns false with a Python error set
// (LsmxError through _capi.check) if one fails.
template <typename F>
bool launch(F &&f) {
    int rc;
    {
        NoGil released;
        rc = f();
    }
    if (rc == LSMX_OK) return true;
    PyObject *r = PyObject_CallFunction(g_error, "i", rc);
    Py_XDECREF(r);
    return false;
}

PyObject *wrap2(const Tensor &a, const Tensor &b) {
    PyObject *t = PyTuple_New(2);
    if (!t) return nullptr;
    PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(a));
    PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(b));
    return t;
}

#define NONE_IF(c) \
    if (c) Py_RETURN_NONE

// ---------------------------------------------------------------- quantizers
// what the row quantizer reads in place: fp32 / bf16 / fp16 rows, K % 32 == 0
bool quant_rows(const Tensor *x, int64_t kmult) {
    return x && rows16(*x) && dtype_of(x->scalar_type()) >= 0 && x->size(0) > 0 && x->size(1) > 0 &&
           x->size(1) % kmult == 0;
}

struct Quantized {
    Tensor codes, scale;
};
Quantized packed_out(const Tensor &x, bool km) {
    const int64_t R = x.size(0), K = x.size(1);
    return {make({R, K / 2}, at::kByte, x), km ? make({K / 128, R, 4}, at::kByte, x) : make({R, K / 32}, at::kByte, x)};
}
int quant_launch(const Tensor &x, const Quantized &q, bool km, void *s) {
    const int64_t R = x.size(0), K = x.size(1);
    return lsmx_quantize_mxfp4(x.data_ptr(), dtype_of(x.scalar_type()), R, K, R > 1 ? x.stride(0) : K, 32,
                               q.codes.data_ptr(), LSMX_CODES_PACKED, K / 2, q.scale.data_ptr(),
                               km ? LSMX_SCALE_E8M0_KMAJOR : LSMX_SCALE_E8M0, km ? R : K / 32, s);
}
// two tensors: one launch when they share a dtype
int quant2_launch(const Tensor &x, const Quantized &qx, const Tensor &w, const Quantized &qw, bool km, void *s) {
    if (x.scalar_type() != w.scalar_type()) {
        const int rc = quant_launch(x, qx, km, s);
        return rc == LSMX_OK ? quant_launch(w, qw, km, s) : rc;
    }
    lsmx_q_item it[2];
    const Tensor *ts[2] = {&x, &w};
    const Quantized *qs[2] = {&qx, &qw};
    for (int i = 0; i < 2; ++i) {
        const int64_t R = ts[i]->size(0), K = ts[i]->size(1);
        it[i] = lsmx_q_item{ts[i]->data_ptr(),       R,     K,
                            R > 1 ? ts[i]->stride(0) : K, qs[i]->codes.data_ptr(), K / 2,
                            qs[i]->scale.data_ptr(), km ? R : K / 32};
    }
    return lsmx_quantize_mxfp4_batch(it, 2, dtype_of(x.scalar_type()), km ? LSMX_SCALE_E8M0_KMAJOR : LSMX_SCALE_E8M0, s);
}

// quantize_pack(x, kmajor) -> (packed, e8m0)
PyObject *quantize_pack(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    NONE_IF(n != 2);
    const bool km = a[1] == Py_True;
    const Tensor *x = plain(a[0]);
    NONE_IF(!quant_rows(x, km ? 128 : 32));
    const Quantized q = packed_out(*x, km);
    void *s = stream_of(*x);
    if (!launch([&] { return quant_launch(*x, q, km, s); })) return nullptr;
    return wrap2(q.codes, q.scale);
    END_HANDLE_TH_ERRORS
}

// quantize_pack2([x, w], kmajor) -> [(packed, e8m0), (packed, e8m0)]
PyObject *quantize_pack2(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    NONE_IF(n != 2 || !PyList_CheckExact(a[0]) || PyList_GET_SIZE(a[0]) != 2);
    const bool km = a[1] == Py_True;
    const Tensor *x = plain(PyList_GET_ITEM(a[0], 0)), *w = plain(PyList_GET_ITEM(a[0], 1));
    NONE_IF(!quant_rows(x, km ? 128 : 32) || !quant_rows(w, km ? 128 : 32) || x->scalar_type() != w->scalar_type() ||
            x->device() != w->device());
    const Quantized qx = packed_out(*x, km), qw = packed_out(*w, km);
    void *s = stream_of(*x);
    if (!launch([&] { return quant2_launch(*x, qx, *w, qw, km, s); })) return nullptr;
    PyObject *l = PyList_New(2);
    if (!l) return nullptr;
    PyList_SET_ITEM(l, 0, wrap2(qx.codes, qx.scale));
    PyList_SET_ITEM(l, 1, wrap2(qw.codes, qw.scale));
    return l;
    END_HANDLE_TH_ERRORS
}

// quantize(x) -> (codes, fp32 scale): fp4.quantize_mxfp4 with 32-blocks
PyObject *quantize(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    NONE_IF(n != 1);
    const Tensor *x = plain(a[0]);
    NONE_IF(!quant_rows(x, 32));
    const int64_t R = x->size(0), K = x->size(1);
    const Tensor codes = make({R, K}, at::kByte, *x), scale = make({R, K / 32}, at::kFloat, *x);
    void *s = stream_of(*x);
    if (!launch([&] {
            return lsmx_quantize_mxfp4(x->data_ptr(), dtype_of(x->scalar_type()), R, K, R > 1 ? x->stride(0) : K, 32,
                                       codes.data_ptr(), LSMX_CODES_UNPACKED, K, scale.data_ptr(), LSMX_SCALE_F32,
                                       K / 32, s);
        }))
        return nullptr;
    return wrap2(codes, scale);
    END_HANDLE_TH_ERRORS
}

// quantize_2d(x) -> (row_packed, row_scale, col_packed, col_scale), K-major
PyObject *quantize_2d(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    NONE_IF(n != 1);
    const Tensor *x = plain(a[0]);
    NONE_IF(!quant_rows(x, 128) || x->size(0) % 128 || x->scalar_type() == at::kFloat);
    const int64_t R = x->size(0), K = x->size(1);
    const Tensor rp = make({R, K / 2}, at::kByte, *x), rs = make({K / 128, R, 4}, at::kByte, *x);
    const Tensor cp = make({K, R / 2}, at::kByte, *x), cs = make({R / 128, K, 4}, at::kByte, *x);
    void *s = stream_of(*x);
    if (!launch([&] {
            return lsmx_quantize_mxfp4_2d(x->data_ptr(), dtype_of(x->scalar_type()), R, K, x->stride(0),
                                          rp.data_ptr<uint8_t>(), K / 2, rs.data_ptr<uint8_t>(), R,
                                          cp.data_ptr<uint8_t>(), R / 2, cs.data_ptr<uint8_t>(), K,
                                          LSMX_SCALE_E8M0_KMAJOR, s);
        }))
        return nullptr;
    PyObject *t = PyTuple_New(4);
    if (!t) return nullptr;
    const Tensor *o[4] = {&rp, &rs, &cp, &cs};
    for (int i = 0; i < 4; ++i) PyTuple_SET_ITEM(t, i, THPVariable_Wrap(*o[i]));
    return t;
    END_HANDLE_TH_ERRORS
}

// pack(codes) -> packed
PyObject *pack(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    NONE_IF(n != 1);
    const Tensor *c = plain(a[0]);
    NONE_IF(!c || c->scalar_type() != at::kByte || c->dim() != 2 || !c->is_contiguous() || c->size(1) % 2 ||
            c->numel() == 0 || !al(*c, 16));
    const Tensor out = make({c->size(0), c->size(1) / 2}, at::kByte, *c);
    void *s = stream_of(*c);
    if (!launch([&] { return lsmx_pack_fp4(c->data_ptr<uint8_t>(), out.data_ptr<uint8_t>(), out.numel(), s); }))
        return nullptr;
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------ f4 x f4 GEMM
int gemm_km(const Tensor &a, const Tensor &as, const Tensor &b, const Tensor &bs, const Tensor &c, int64_t K, void *s) {
    const int64_t M = a.size(0), N = b.size(0);
    return lsmx_gemm_f4f4(a.data_ptr<uint8_t>(), M > 1 ? a.stride(0) : K / 2, as.data_ptr(), M, b.data_ptr<uint8_t>(),
                          N > 1 ? b.stride(0) : K / 2, bs.data_ptr(), N, LSMX_SCALE_E8M0_KMAJOR, c.data_ptr(),
                          dtype_of(c.scalar_type()), N, M, N, K, s);
}

// fp32 block scales of the two operands -> K-major E8M0 in one launch, with the
// flag that lsmx_gemm_mx_promote tests unless the caller knows them exact
struct ScaleConv {
    Tensor a, b, flag;
    uint64_t epoch = 0;
    lsmx_e8m0_item it[2];
};
bool scales_f32(const Tensor *s, int64_t r, int64_t c) {
    return s && s->scalar_type() == at::kFloat && s->dim() == 2 && s->size(0) == r && s->size(1) == c &&
           s->stride(1) == 1 && s->stride(0) >= c;
}
bool conv_prepare(ScaleConv &v, const Tensor &sa, int64_t M, const Tensor &sb, bool sb_t, int64_t N, int64_t K,
                  bool flagged) {
    v.a = make({K / 128, M, 4}, at::kByte, sa);
    v.b = make({K / 128, N, 4}, at::kByte, sa);
    const Tensor *ss[2] = {&sa, &sb};
    for (int i = 0; i < 2; ++i) {
        const Tensor &s = *ss[i];
        v.it[i] = lsmx_e8m0_item{s.data_ptr<float>(), s.size(0), s.size(1), s.size(0) > 1 ? s.stride(0) : s.size(1),
                                 i == 1 && sb_t ? LSMX_E8M0_IN_T : 0, (i ? v.b : v.a).data_ptr<uint8_t>(), i ? N : M};
    }
    if (flagged) {
        v.flag = make({1}, at::kLong, sa);
        PyObject *e = PyObject_CallNoArgs(g_epoch);
        if (!e) return false;
        v.epoch = PyLong_AsUnsignedLongLong(e);
        Py_DECREF(e);
        if (PyErr_Occurred()) return false;
    }
    return true;
}
uint64_t *flag_of(const ScaleConv &v) { return v.flag.defined() ? reinterpret_cast<uint64_t *>(v.flag.data_ptr()) : nullptr; }
int conv_launch(const ScaleConv &v, void *s) { return lsmx_scale_to_e8m0_batch(v.it, 2, flag_of(v), v.epoch, s); }

// gemm_packed(a_pk, bt_pk, a_scale, b_scale, out_dtype, exact)
PyObject *gemm_packed(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    NONE_IF(n != 6);
    const Tensor *ap = plain(a[0]), *bp = plain(a[1]), *as = plain(a[2]), *bs = plain(a[3]);
    const at::ScalarType ot = out_type(a[4]);
    NONE_IF(!ap || !bp || !as || !bs || ot == at::ScalarType::Undefined || ap->scalar_type() != at::kByte ||
            bp->scalar_type() != at::kByte || !rows16(*ap) || !rows16(*bp) || ap->size(1) != bp->size(1));
    const int64_t M = ap->size(0), N = bp->size(0), K = 2 * ap->size(1);
    NONE_IF(M == 0 || N == 0 || K == 0 || K % 128 || bp->device() != ap->device() || as->device() != ap->device() ||
            bs->device() != ap->device() || as->scalar_type() != bs->scalar_type());
    if (as->scalar_type() == at::kByte) {
        for (int i = 0; i < 2; ++i) {
            const Tensor &s = i ? *bs : *as;
            NONE_IF(s.dim() != 3 || s.size(0) != K / 128 || s.size(1) != (i ? N : M) || s.size(2) != 4 ||
                    !s.is_contiguous());
        }
        const Tensor c = make({M, N}, ot, *ap);
        void *s = stream_of(c);
        if (!launch([&] { return gemm_km(*ap, *as, *bp, *bs, c, K, s); })) return nullptr;
        return THPVariable_Wrap(c);
    }
    NONE_IF(!scales_f32(as, M, K / 32) || !scales_f32(bs, N, K / 32));
    const bool flagged = a[5] != Py_True;
    const Tensor c = make({M, N}, ot, *ap);
    void *s = stream_of(c);
    ScaleConv v;
    if (!conv_prepare(v, *as, M, *bs, false, N, K, flagged)) return nullptr;
    if (!launch([&] {
            int rc = conv_launch(v, s);
            if (rc == LSMX_OK) rc = gemm_km(*ap, v.a, *bp, v.b, c, K, s);
            if (rc == LSMX_OK && flagged)
                rc = lsmx_gemm_mx_promote(ap->data_ptr<uint8_t>(), M > 1 ? ap->stride(0) : K / 2, as->data_ptr<float>(),
                                          M > 1 ? as->stride(0) : K / 32, 1, bp->data_ptr<uint8_t>(),
                                          N > 1 ? bp->stride(0) : K / 2, bs->data_ptr<float>(),
                                          N > 1 ? bs->stride(0) : K / 32, 1, LSMX_CODES_PACKED, c.data_ptr(),
                                          dtype_of(ot), N, M, N, K, flag_of(v), v.epoch, s);
            return rc;
        }))
        return nullptr;
    return THPVariable_Wrap(c);
    END_HANDLE_TH_ERRORS
}

// linear(x, w, out_dtype): quantize both operands along K and multiply, the
// forward of MXFP4Linear
PyObject *linear(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    NONE_IF(n != 3);
    const Tensor *x = plain(a[0]), *w = plain(a[1]);
    const at::ScalarType ot = out_type(a[2]);
    NONE_IF(ot == at::ScalarType::Undefined || !quant_rows(x, 128) || !quant_rows(w, 128) || x->size(1) != w->size(1) ||
            x->device() != w->device());
    const int64_t K = x->size(1);
    const Quantized qx = packed_out(*x, true), qw = packed_out(*w, true);
    const Tensor c = make({x->size(0), w->size(0)}, ot, *x);
    void *s = stream_of(c);
    if (!launch([&] {
            const int rc = quant2_launch(*x, qx, *w, qw, true, s);
            return rc == LSMX_OK ? gemm_km(qx.codes, qx.scale, qw.codes, qw.scale, c, K, s) : rc;
        }))
        return nullptr;
    return THPVariable_Wrap(c);
    END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------- weight-only GEMMs
// weight(a0, a1 or None, w_pk, w_scale, out_dtype or None): a0 @ deq(W)^T (and
// a1 @ deq(W)^T); E8M0 weight scales
PyObject *weight(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    NONE_IF(n != 5);
    const Tensor *a0 = plain(a[0]), *w = plain(a[2]), *ws = plain(a[3]);
    const bool dual = a[1] != Py_None;
    const Tensor *a1 = dual ? plain(a[1]) : nullptr;
    NONE_IF(!a0 || !w || !ws || (dual && !a1) || !rows16(*a0) || !rows16(*w) || dtype_of(a0->scalar_type()) < 0 ||
            w->scalar_type() != at::kByte || ws->scalar_type() != at::kByte);
    const at::ScalarType at_ = a0->scalar_type(), ot = a[4] == Py_None ? at_ : out_type(a[4]);
    const int64_t M = a0->size(0), K = a0->size(1), N = w->size(0);
    NONE_IF(ot == at::ScalarType::Undefined || M == 0 || N == 0 || K == 0 || K % 128 || 2 * w->size(1) != K ||
            w->device() != a0->device() || ws->device() != a0->device());
    NONE_IF(ws->dim() != 2 || ws->size(0) != N || ws->size(1) != K / 32 || ws->stride(1) != 1 ||
            ws->stride(0) < K / 32 || (N > 1 && ws->stride(0) % 4) || !al(*ws, 4));
    NONE_IF(dual && (at_ != at::kBFloat16 || a1->scalar_type() != at_ || !rows16(*a1) || a1->size(0) != M ||
                     a1->size(1) != K || a1->stride(0) != a0->stride(0) || a1->device() != a0->device()));
    const int64_t lda = M > 1 ? a0->stride(0) : K, ldw = N > 1 ? w->stride(0) : K / 2, lds = N > 1 ? ws->stride(0) : K / 32;
    const Tensor c0 = make({M, N}, ot, *a0), c1 = dual ? make({M, N}, ot, *a0) : Tensor();
    void *s = stream_of(c0);
    if (at_ == at::kBFloat16) {
        const int64_t nws = lsmx_gemm_bf16f4_slices(M, N, K) > 1 ? lsmx_gemm_bf16f4_workspace(M, N, K, dual) : 0;
        void *wsp = nullptr;
        PyObject *keep = nullptr;
        if (nws > 0) {   // the split-K workspace of this device and stream
            PyObject *dev = PyObject_GetAttrString(a[0], "device");
            if (!dev) return nullptr;
            keep = PyObject_CallFunction(g_workspace, "OL", dev, (long long)nws);
            Py_DECREF(dev);
            if (!keep) return nullptr;
            wsp = THPVariable_Unpack(keep).data_ptr();
        }
        const bool ok = launch([&] {
            return lsmx_gemm_bf16f4_ws(a0->data_ptr(), dual ? a1->data_ptr() : nullptr, lda, w->data_ptr<uint8_t>(), ldw,
                                       ws->data_ptr(), lds, LSMX_SCALE_E8M0, c0.data_ptr(),
                                       dual ? c1.data_ptr() : nullptr, dtype_of(ot), N, M, N, K, wsp, nws, s);
        });
        Py_XDECREF(keep);
        if (!ok) return nullptr;
    } else if (!launch([&] {
                   return lsmx_gemm_wonly_f4(a0->data_ptr(), dtype_of(at_), lda, w->data_ptr<uint8_t>(), ldw,
                                             ws->data_ptr(), lds, LSMX_SCALE_E8M0, c0.data_ptr(), dtype_of(ot), N, M, N,
                                             K, s);
               })) {
        return nullptr;
    }
    return dual ? wrap2(c0, c1) : THPVariable_Wrap(c0);
    END_HANDLE_TH_ERRORS
}

// -------------------------------------------------------------- E4M3 GEMM
// gemm_fp8(a_fp8, b_fp8, a_scale, b_scale, out_dtype, exact): B [K, N] with N
// contiguous, fp32 scales
PyObject *gemm_fp8(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    NONE_IF(n != 6);
    const Tensor *x = plain(a[0]), *b = plain(a[1]), *as = plain(a[2]), *bs = plain(a[3]);
    const at::ScalarType ot = out_type(a[4]);
    auto bytes = [](const Tensor &t) { return t.scalar_type() == at::kFloat8_e4m3fn || t.scalar_type() == at::kByte; };
    NONE_IF(!x || !b || !as || !bs || ot == at::ScalarType::Undefined || !bytes(*x) || !bytes(*b) || !rows16(*x) ||
            !rows16(*b) || x->size(1) != b->size(0));
    const int64_t M = x->size(0), K = x->size(1), N = b->size(1);
    NONE_IF(M == 0 || N == 0 || K == 0 || K % 128 || N % 16 || b->stride(0) >= 0x7FFFFFFF / 256 ||
            b->device() != x->device() || as->device() != x->device() || bs->device() != x->device() ||
            !scales_f32(as, M, K / 32) || !scales_f32(bs, K / 32, N));
    const bool flagged = a[5] != Py_True;
    const Tensor c = make({M, N}, ot, *x);
    void *s = stream_of(c);
    ScaleConv v;
    if (!conv_prepare(v, *as, M, *bs, true, N, K, flagged)) return nullptr;
    const uint8_t *xp = reinterpret_cast<const uint8_t *>(x->data_ptr()), *bp = reinterpret_cast<const uint8_t *>(b->data_ptr());
    const int64_t lda = M > 1 ? x->stride(0) : K, ldb = b->stride(0);
    if (!launch([&] {
            int rc = conv_launch(v, s);
            if (rc == LSMX_OK)
                rc = lsmx_gemm_f8f8_nb(xp, lda, v.a.data_ptr<uint8_t>(), M, bp, ldb, v.b.data_ptr<uint8_t>(), N,
                                       c.data_ptr(), dtype_of(ot), N, M, N, K, s);
            if (rc == LSMX_OK && flagged)
                rc = lsmx_gemm_mx_promote(xp, lda, as->data_ptr<float>(), M > 1 ? as->stride(0) : K / 32, 1, bp, ldb,
                                          bs->data_ptr<float>(), 1, K / 32 > 1 ? bs->stride(0) : N,
                                          LSMX_E4M3 | LSMX_B_NCONTIG, c.data_ptr(), dtype_of(ot), N, M, N, K,
                                          flag_of(v), v.epoch, s);
            return rc;
        }))
        return nullptr;
    return THPVariable_Wrap(c);
    END_HANDLE_TH_ERRORS
}

// -------------------------------------------------------------- attention
// What the attention kernels read in place: unit stride along the last axis, 16-byte
// aligned vectors, tokens and the heads of a group within 32-bit offsets.
bool in_reach(const Tensor &t, int64_t group) {
    const int64_t d = t.dim();
    if (t.numel() == 0 || t.stride(d - 1) != 1 || !al(t, 16)) return false;
    for (int64_t i = 0; i < d - 1; ++i)
        if (t.size(i) > 1 && t.stride(i) % 8) return false;
    return (t.size(d - 3) <= 1 || t.stride(d - 3) < (1 << 22)) && (t.size(d - 2) <= 1 || t.stride(d - 2) * group < (1 << 29));
}
void strides_of(const Tensor &t, int64_t *s) {
    const int64_t d = t.dim();
    for (int i = 0; i < 3; ++i) {
        const int64_t k = d - 4 + i;
        s[i] = k >= 0 && t.size(k) > 1 ? t.stride(k) : 0;
    }
}
bool bf16_or_f16(const Tensor &t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf; }
// an int >= lo, or None as 0
bool int_arg(PyObject *o, int64_t lo, bool none, int64_t &v) {
    if (none && o == Py_None) {
        v = 0;
        return true;
    }
    if (!PyLong_CheckExact(o)) return false;
    int over = 0;
    v = PyLong_AsLongLongAndOverflow(o, &over);
    return !over && v >= lo;
}
// scale, or None as 1 / sqrt(D); positive and finite
bool scale_arg(PyObject *o, int64_t D, double &v) {
    if (o == Py_None)
        v = 1.0 / std::sqrt((double)D);
    else if (PyFloat_CheckExact(o))
        v = PyFloat_AS_DOUBLE(o);
    else
        return false;
    return v > 0.0 && v <= 3.0e38;
}
bool int32_on(const Tensor *t, const Tensor &like, int64_t dims) {
    return t && t->scalar_type() == at::kInt && t->dim() == dims && t->is_contiguous() && t->device() == like.device();
}

// Under torch.jit.trace the Python path refuses the call; forward-mode
// derivatives are refused by its node.
bool traced() { return at::tracer::impl::is_dispatch_enabled(); }
bool dual(const Tensor &t) { return t._fw_grad(0).defined(); }

struct Failed {
    int rc;
};

lsmx_attention attention_args(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &o, const Tensor &rest,
                              const Tensor &lse, const Tensor &offsets, int64_t window, int64_t sinks, double scale) {
    lsmx_attention a{};
    a.q = q.data_ptr(), a.k = k.data_ptr(), a.v = v.data_ptr(), a.o = o.data_ptr();
    a.o_rest = rest.defined() ? rest.data_ptr() : nullptr;
    a.lse = lse.data_ptr<float>();
    a.dtype = dtype_of(q.scalar_type());
    const int64_t d = q.dim();
    a.batch = offsets.defined() ? offsets.numel() - 1 : q.size(0);
    a.q_len = q.size(d - 3), a.k_len = k.size(d - 3), a.heads = q.size(d - 2), a.kv_heads = k.size(d - 2);
    a.head_dim = q.size(d - 1);
    strides_of(q, a.q_stride), strides_of(k, a.k_stride), strides_of(v, a.v_stride), strides_of(o, a.o_stride);
    a.offsets = offsets.defined() ? offsets.data_ptr<int32_t>() : nullptr;
    a.window = window, a.sinks = sinks, a.scale = (float)scale;
    return a;
}

struct Forward {
    Tensor o, rest, lse;
};
Forward attention_forward(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &offsets, int64_t window,
                          int64_t sinks, double scale, bool grad) {
    Forward f;
    const int64_t d = q.dim();
    f.o = make(q.sizes(), q.scalar_type(), q);
    if (grad) f.rest = make(q.sizes(), q.scalar_type(), q);
    f.lse = d == 4 ? make({q.size(0), q.size(2), q.size(1)}, at::kFloat, q) : make({q.size(1), q.size(0)}, at::kFloat, q);
    const lsmx_attention a = attention_args(q, k, v, f.o, f.rest, f.lse, offsets, window, sinks, scale);
    if (const int rc = lsmx_attention_fwd(&a, stream_of(q))) throw Failed{rc};
    return f;
}

// The same node as attention._SinkWindowAttention, in native code.
struct Attention : torch::autograd::Function<Attention> {
    static Tensor forward(torch::autograd::AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v,
                          const std::optional<Tensor> &offsets, int64_t window, int64_t sinks, double scale) {
        const Tensor off = offsets ? *offsets : Tensor();
        const Forward f = attention_forward(q, k, v, off, window, sinks, scale, true);
        ctx->save_for_backward({q, k, v, f.o, f.rest, f.lse, off});
        ctx->saved_data["window"] = window;
        ctx->saved_data["sinks"] = sinks;
        ctx->saved_data["scale"] = scale;
        return f.o;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
        const auto s = ctx->get_saved_variables();
        const Tensor &q = s[0], &k = s[1], &v = s[2];
        std::vector<Tensor> d(3);
        {
            at::AutoGradMode off(false);
            Tensor d_o = grads[0].defined() ? grads[0].to(q.scalar_type()) : at::zeros_like(q);
            const int64_t group = q.size(-2) / k.size(-2);
            if (!in_reach(d_o, group)) {
                d_o = d_o.contiguous();
                if (!al(d_o, 16)) d_o = d_o.clone();
            }
            for (int i = 0; i < 3; ++i) d[i] = make(s[i].sizes(), q.scalar_type(), q);
            const lsmx_attention a = attention_args(q, k, v, s[3], s[4], s[5], s[6], ctx->saved_data["window"].toInt(),
                                                    ctx->saved_data["sinks"].toInt(), ctx->saved_data["scale"].toDouble());
            const int64_t n = lsmx_attention_workspace(&a);
            const Tensor ws = make({n}, at::kByte, q);
            int64_t st[3];
            strides_of(d_o, st);
            TORCH_CHECK(lsmx_attention_bwd(&a, d_o.data_ptr(), st, d[0].data_ptr(), d[1].data_ptr(), d[2].data_ptr(),
                                           ws.data_ptr(), n, stream_of(q)) == LSMX_OK,
                        lsmx_last_error());
        }
        if (at::GradMode::is_enabled()) {  // create_graph: the gradients have none
            auto err = std::make_shared<torch::autograd::DelayedError>(
                "trying to differentiate twice a function that was marked with @once_differentiable", 3);
            torch::autograd::variable_list in;
            for (auto &t : d) in.push_back(t.detach().set_requires_grad(true));
            d = (*err)(std::move(in));
        }
        return {d[0], d[1], d[2], Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

// attention(q, k, v, offsets, window, sinks, scale) -> o
PyObject *attention(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    NONE_IF(n != 7);
    const Tensor *q = plain(a[0]), *k = plain(a[1]), *v = plain(a[2]), *off = a[3] == Py_None ? nullptr : plain(a[3]);
    NONE_IF(!q || !k || !v || (a[3] != Py_None && !off) || at::autocast::is_autocast_enabled(at::kCUDA) || traced() || dual(*q) ||
            dual(*k) || dual(*v));
    const int64_t d = off ? 3 : 4;
    NONE_IF(q->dim() != d || k->dim() != d || !k->sizes().equals(v->sizes()) || !bf16_or_f16(*q) ||
            k->scalar_type() != q->scalar_type() || v->scalar_type() != q->scalar_type() || k->device() != q->device() ||
            v->device() != q->device() || (off && !int32_on(off, *q, 1)));
    const int64_t H = q->size(d - 2), Hkv = k->size(d - 2), D = q->size(d - 1);
    NONE_IF(q->numel() == 0 || k->numel() == 0 || k->size(0) != q->size(0) || k->size(d - 1) != D || H % Hkv || D % 8 ||
            D > 128 || (off && off->numel() < 1) || !in_reach(*q, H / Hkv) || !in_reach(*k, 1) || !in_reach(*v, 1));
    int64_t window, sinks;
    double scale;
    NONE_IF(!int_arg(a[4], 1, true, window) || !int_arg(a[5], 0, false, sinks) || !scale_arg(a[6], D, scale));
    const Tensor none, &offsets = off ? *off : none;
    const bool grad = at::GradMode::is_enabled() && (q->requires_grad() || k->requires_grad() || v->requires_grad());
    Tensor o;
    int rc = LSMX_OK;
    {
        NoGil released;
        try {
            o = grad ? Attention::apply(*q, *k, *v, off ? std::optional<Tensor>(*off) : std::nullopt, window, sinks, scale)
                     : attention_forward(*q, *k, *v, offsets, window, sinks, scale, false).o;
        } catch (const Failed &f) {
            rc = f.rc;
        }
    }
    if (rc != LSMX_OK) {
        Py_XDECREF(PyObject_CallFunction(g_error, "i", rc));
        return nullptr;
    }
    return THPVariable_Wrap(o);
    END_HANDLE_TH_ERRORS
}

// -------------------------------------------------------------- cache
// The cache of kv_cache._cache, or false for any form that it would refuse.
bool cache_of(PyObject *pages, PyObject *table, PyObject *lengths, lsmx_kv_cache &c, const Tensor *&like) {
    if (!PyTuple_Check(pages) || PyTuple_GET_SIZE(pages) != 4) return false;
    const Tensor *p[4], *t = plain(table), *l = plain(lengths);
    for (int i = 0; i < 4; ++i)
        if (!(p[i] = plain(PyTuple_GET_ITEM(pages, i))) || p[i]->scalar_type() != at::kByte || p[i]->dim() != 4 ||
            !p[i]->is_contiguous() || p[i]->numel() == 0)
            return false;
    const int64_t n = p[0]->size(0), h = p[0]->size(1), page = p[0]->size(2), D = 2 * p[0]->size(3);
    const int64_t want[4] = {n, h, page, D / 32};
    if ((D != 64 && D != 128) || page < 16 || page > 1024 || (page & (page - 1)) || !p[2]->sizes().equals(p[0]->sizes()) ||
        !p[1]->sizes().equals(want) || !p[3]->sizes().equals(want))
        return false;
    like = p[0];
    for (int i = 0; i < 4; ++i)
        if (p[i]->device() != like->device() || !al(*p[i], 16)) return false;
    if (!int32_on(t, *like, 2) || !int32_on(l, *like, 1) || l->size(0) != t->size(0) || t->numel() == 0) return false;
    c = lsmx_kv_cache{p[0]->data_ptr<uint8_t>(), p[1]->data_ptr<uint8_t>(), p[2]->data_ptr<uint8_t>(), p[3]->data_ptr<uint8_t>(),
                      n, page, h, D, t->data_ptr<int32_t>(), l->data_ptr<int32_t>(), t->size(0), t->size(1)};
    return true;
}
// weights as kv_cache._check_weights wants them
bool weights_ok(const Tensor *w, const lsmx_kv_cache &c, const Tensor &like) {
    return w && w->scalar_type() == at::kFloat && w->is_contiguous() && w->dim() == 3 && w->size(0) == c.batch &&
           w->size(1) == c.kv_heads && w->size(2) >= c.max_pages * c.page && w->device() == like.device();
}

// kv_append(pages, k, v, table, lengths, offsets, values) -> (k, v), or True
PyObject *kv_append(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    NONE_IF(n != 7);
    lsmx_kv_cache c;
    const Tensor *like, *k = plain(a[1]), *v = plain(a[2]), *off = a[5] == Py_None ? nullptr : plain(a[5]);
    NONE_IF(!k || !v || traced() || (a[5] != Py_None && !off) || !cache_of(a[0], a[3], a[4], c, like));
    const int64_t d = off ? 3 : 4;
    NONE_IF(k->dim() != d || !k->sizes().equals(v->sizes()) || !bf16_or_f16(*k) || v->scalar_type() != k->scalar_type() ||
            k->device() != like->device() || v->device() != like->device() || k->size(d - 2) != c.kv_heads ||
            k->size(d - 1) != c.head_dim || (off ? !int32_on(off, *like, 1) || off->size(0) != c.batch + 1 : k->size(0) != c.batch) ||
            k->numel() == 0);
    int64_t st[2][2];
    const Tensor *kv[2] = {k, v};
    for (int i = 0; i < 2; ++i) {
        const Tensor &t = *kv[i];
        NONE_IF(t.stride(d - 1) != 1 || !al(t, 16) || (t.size(d - 2) > 1 && t.stride(d - 2) % 8) ||
                (t.size(d - 3) > 1 && t.stride(d - 3) % 8));
        st[i][0] = t.size(d - 3) > 1 ? t.stride(d - 3) : d == 4 && t.size(0) > 1 ? t.stride(0) : 0;
        st[i][1] = t.size(d - 2) > 1 ? t.stride(d - 2) : 0;
        // the sequences of a dense call one after another
        NONE_IF(d == 4 && t.size(0) > 1 && (st[i][0] % 8 || t.stride(0) != st[i][0] * t.size(1)));
    }
    const int values = PyObject_IsTrue(a[6]);
    if (values < 0) return nullptr;
    const int64_t tokens = off ? k->size(0) : k->size(0) * k->size(1);
    Tensor ko, vo;
    if (values) ko = make(k->sizes(), at::kBFloat16, *k), vo = make(k->sizes(), at::kBFloat16, *k);
    void *s = stream_of(*k);
    if (!launch([&] {
            return lsmx_kv_append(&c, k->data_ptr(), st[0], v->data_ptr(), st[1], dtype_of(k->scalar_type()), tokens,
                                  off ? 0 : k->size(1), off ? off->data_ptr<int32_t>() : nullptr,
                                  values ? ko.data_ptr() : nullptr, values ? vo.data_ptr() : nullptr, s);
        }))
        return nullptr;
    if (values) return wrap2(ko, vo);
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// kv_attend(q, pages, table, lengths, window, sinks, scale, weights) -> o
PyObject *kv_attend(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    NONE_IF(n != 8);
    lsmx_kv_cache c;
    const Tensor *like, *q = plain(a[0]), *w = a[7] == Py_None ? nullptr : plain(a[7]);
    NONE_IF(!q || traced() || (a[7] != Py_None && !w) || !cache_of(a[1], a[2], a[3], c, like));
    NONE_IF(q->dim() != 4 || !bf16_or_f16(*q) || q->device() != like->device() || q->numel() == 0 || q->size(0) != c.batch ||
            q->size(3) != c.head_dim || q->size(2) % c.kv_heads || (w && !weights_ok(w, c, *like)) || q->stride(3) != 1 || !al(*q, 16));
    for (int i = 0; i < 3; ++i) NONE_IF(q->size(i) > 1 && q->stride(i) % 8);
    int64_t window, sinks, st[3];
    double scale;
    NONE_IF(!int_arg(a[4], 1, true, window) || !int_arg(a[5], 0, false, sinks) || !scale_arg(a[6], c.head_dim, scale));
    strides_of(*q, st);
    const Tensor o = make(q->sizes(), q->scalar_type(), *q);
    const int64_t T = q->size(1), H = q->size(2), nws = lsmx_kv_attend_workspace(&c, T, H, window, sinks, w != nullptr);
    PyObject *keep = nullptr;
    if (nws) {
        PyObject *dev = PyObject_GetAttrString(a[0], "device");
        if (!dev) return nullptr;
        keep = PyObject_CallFunction(g_workspace, "OL", dev, (long long)nws);
        Py_DECREF(dev);
        if (!keep) return nullptr;
    }
    void *ws = keep ? THPVariable_Unpack(keep).data_ptr() : nullptr, *s = stream_of(*q);
    const bool ok = launch([&] {
        return lsmx_kv_attend(&c, q->data_ptr(), st, dtype_of(q->scalar_type()), T, H, window, sinks, (float)scale,
                              o.data_ptr(), w ? w->data_ptr<float>() : nullptr, w ? w->size(2) : 0, ws, nws, s);
    });
    Py_XDECREF(keep);
    return ok ? THPVariable_Wrap(o) : nullptr;
    END_HANDLE_TH_ERRORS
}

// kv_evict(pages, table, lengths, weights, keep, out_table, sinks, recent) -> (index, weights, lengths)
PyObject *kv_evict(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    NONE_IF(n != 8);
    lsmx_kv_cache c;
    const Tensor *like, *w = plain(a[3]), *out = plain(a[5]);
    int64_t keep, sinks, recent;
    NONE_IF(!w || !out || traced() || !cache_of(a[0], a[1], a[2], c, like) || !weights_ok(w, c, *like) || !int32_on(out, *like, 2) ||
            !int_arg(a[4], 1, false, keep) || !int_arg(a[6], 0, false, sinks) || !int_arg(a[7], 0, false, recent));
    const int64_t cap = c.max_pages * c.page, most = keep < cap ? keep : cap;
    NONE_IF(keep >= (1 << 30) || sinks > keep || recent > keep - sinks || out->size(0) != c.batch || out->size(1) * c.page < most);
    const Tensor index = make({c.batch, c.kv_heads, keep}, at::kInt, *like), kept = make({c.batch, c.kv_heads, keep}, at::kFloat, *like);
    const Tensor len = make({c.batch}, at::kInt, *like);
    void *s = stream_of(*like);
    if (!launch([&] {
            return lsmx_kv_evict(&c, w->data_ptr<float>(), w->size(2), keep, sinks, recent, out->data_ptr<int32_t>(),
                                 out->size(1), index.data_ptr<int32_t>(), kept.data_ptr<float>(), len.data_ptr<int32_t>(), s);
        }))
        return nullptr;
    PyObject *t = PyTuple_New(3);
    if (!t) return nullptr;
    PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(index));
    PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(kept));
    PyTuple_SET_ITEM(t, 2, THPVariable_Wrap(len));
    return t;
    END_HANDLE_TH_ERRORS
}

// --------------------------------------------- norm, router, experts' products
// dense storage of a type on the current device, which launches need;
// forward-mode derivatives go to the Python path's nodes, which refuse them
bool dense(const Tensor *t, at::ScalarType s) { return t && t->scalar_type() == s && t->is_contiguous(); }
bool here(const Tensor &t) { return t.device().index() == c10::hip::current_device(); }
bool bool_arg(PyObject *o, bool &v) {
    v = o == Py_True;
    return PyBool_Check(o);
}
std::vector<int64_t> with_last(at::IntArrayRef shape, std::initializer_list<int64_t> last, int64_t drop) {
    std::vector<int64_t> v(shape.begin(), shape.end() - drop);
    v.insert(v.end(), last);
    return v;
}
PyObject *wrap_all(const std::vector<Tensor> &ts) {
    PyObject *r = PyTuple_New((Py_ssize_t)ts.size());
    if (!r) return nullptr;
    for (size_t i = 0; i < ts.size(); ++i) PyTuple_SET_ITEM(r, (Py_ssize_t)i, THPVariable_Wrap(ts[i]));
    return r;
}

// Raises for a failed call made inside a node, where the engine carries C++
// exceptions.
void must(int rc) { TORCH_CHECK(rc == LSMX_OK, lsmx_last_error()); }

// Gradients that have none of their own (create_graph), as once_differentiable
// gives them.
torch::autograd::variable_list once(torch::autograd::variable_list d) {
    if (!at::GradMode::is_enabled()) return d;
    auto err = std::make_shared<torch::autograd::DelayedError>(
        "trying to differentiate twice a function that was marked with @once_differentiable", (int)d.size());
    torch::autograd::variable_list in;
    for (auto &t : d) in.push_back(t.defined() ? t.detach().set_requires_grad(true) : t);
    return (*err)(std::move(in));
}

// Refuses a differentiable call that is being captured into a graph while a node
// that its gradients would go to belongs to the default stream, as a leaf's does
// of which an eager graph is still alive: in the backward pass the engine would
// make that stream wait for the captured one, which ends the process.  (Any other
// stream becomes part of the capture, and is joined at the pass's end.)
// `capturing`: of the current stream, or as a test has it.
bool capturing() { return c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None; }
void one_stream(const Tensor &t, bool capturing) {
    if (!capturing || !t.requires_grad()) return;
    const auto node = t.grad_fn() ? t.grad_fn() : torch::autograd::impl::try_get_grad_accumulator(t);
    if (!node) return;
    const auto there = node->stream();
    TORCH_CHECK(!there || there->device_type() != at::kCUDA ||
                    there->id() != c10::hip::getDefaultHIPStreamMasqueradingAsCUDA(there->device_index()).id() ||
                    there->id() == c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(there->device_index()).id(),
                "a differentiable call cannot be captured while a graph of its tensors made on the default stream is alive: free that "
                "graph's outputs first, make it on another stream, or capture the call under torch.no_grad()");
}

// captures(tensors, capturing): the same for the nodes in Python; capturing None:
// of the current stream
PyObject *captures(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    NONE_IF(n != 2 || !PyTuple_Check(a[0]));
    bool c = false;
    if (!bool_arg(a[1], c)) c = capturing();
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(a[0]); ++i)
        if (const Tensor *t = plain(PyTuple_GET_ITEM(a[0], i))) one_stream(*t, c);
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

struct NormOut {
    Tensor y, h, codes, scale;
};
NormOut norm_forward(const Tensor &x, const Tensor &w, const Tensor &r, double eps, bool mx) {
    const int64_t D = x.size(-1);
    NormOut o;
    o.y = make(x.sizes(), x.scalar_type(), x);
    if (r.defined()) o.h = make(x.sizes(), x.scalar_type(), x);
    if (mx) {
        o.codes = make(x.sizes(), at::kFloat8_e4m3fn, x);
        o.scale = make(with_last(x.sizes(), {D / 32}, 1), at::kByte, x);
    }
    if (const int rc = lsmx_rms_norm(x.data_ptr(), D, r.defined() ? r.data_ptr() : nullptr, r.defined() ? D : 0, dtype_of(x.scalar_type()),
                                     w.data_ptr(), dtype_of(w.scalar_type()), x.numel() / D, D, (float)eps,
                                     r.defined() ? o.h.data_ptr() : nullptr, o.y.data_ptr(), mx ? (uint8_t *)o.codes.data_ptr() : nullptr,
                                     mx ? o.scale.data_ptr<uint8_t>() : nullptr, stream_of(x)))
        throw Failed{rc};
    return o;
}

// The same node as norm._AddRMSNorm, in native code.
struct Norm : torch::autograd::Function<Norm> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext *ctx, const Tensor &x, const Tensor &w,
                                                  const std::optional<Tensor> &r, double eps, bool mx) {
        NormOut o = norm_forward(x, w, r ? *r : Tensor(), eps, mx);
        ctx->save_for_backward({r ? o.h : x, w});
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["residual"] = r.has_value();
        ctx->set_materialize_grads(false);
        torch::autograd::variable_list out{o.y};
        if (r) out.push_back(o.h);
        if (mx) {
            out.push_back(o.codes), out.push_back(o.scale);
            ctx->mark_non_differentiable({o.codes, o.scale});
        }
        return out;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
        const auto s = ctx->get_saved_variables();
        const Tensor &h = s[0], &w = s[1];
        const bool residual = ctx->saved_data["residual"].toBool();
        Tensor dy = grads[0], dh = residual ? grads[1] : Tensor(), dx, dw;
        if (!dy.defined()) {
            dx = dh;
        } else {
            at::AutoGradMode off(false);
            const int64_t D = h.size(-1), rows = h.numel() / D;
            const int dt = dtype_of(h.scalar_type());
            dy = dy.to(h.scalar_type()).contiguous();
            if (dh.defined()) dh = dh.to(h.scalar_type()).contiguous();
            dx = make(h.sizes(), h.scalar_type(), h);
            Tensor ws;
            int64_t n = 0;
            if (ctx->needs_input_grad(1)) {
                dw = make(w.sizes(), w.scalar_type(), w);
                n = lsmx_rms_norm_bwd_workspace(rows, D, dt);
                ws = make({n}, at::kByte, h);
            }
            must(lsmx_rms_norm_bwd(h.data_ptr(), D, dy.data_ptr(), D, dh.defined() ? dh.data_ptr() : nullptr, dh.defined() ? D : 0, dt,
                                   w.data_ptr(), dtype_of(w.scalar_type()), rows, D, (float)ctx->saved_data["eps"].toDouble(),
                                   dx.data_ptr(), dw.defined() ? dw.data_ptr() : nullptr, n ? ws.data_ptr() : nullptr, n, stream_of(h)));
        }
        auto d = once({dx, dw, residual ? dx : Tensor()});
        return {d[0], d[1], d[2], Tensor(), Tensor()};
    }
};

// rms_norm(x, weight, residual, eps, mxfp8) -> y, or (y, h), with (codes, scale)
PyObject *rms_norm(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    NONE_IF(n != 5);
    const Tensor *x = plain(a[0]), *w = plain(a[1]), *r = a[2] == Py_None ? nullptr : plain(a[2]);
    bool mx;
    NONE_IF(!x || !w || (a[2] != Py_None && !r) || !PyFloat_CheckExact(a[3]) || !bool_arg(a[4], mx) || traced());
    const double eps = PyFloat_AS_DOUBLE(a[3]);
    const at::ScalarType dt = x->scalar_type();
    NONE_IF(dtype_of(dt) < 0 || x->dim() < 1 || x->numel() == 0 || !x->is_contiguous() || (r && (!dense(r, dt) || !r->sizes().equals(x->sizes()))) ||
            (w->scalar_type() != dt && w->scalar_type() != at::kFloat) || w->dim() != 1 || !w->is_contiguous() ||
            w->size(0) != x->size(-1) || w->device() != x->device() || (r && r->device() != x->device()) || !here(*x) ||
            dual(*x) || dual(*w) || (r && dual(*r)) || !(eps >= 0.0 && eps <= 3.0e38));
    NONE_IF(mx && (x->size(-1) % 32 || !al(*x, 16) || !al(*w, 16) || (r && !al(*r, 16))));
    const bool grad = at::GradMode::is_enabled() && (x->requires_grad() || w->requires_grad() || (r && r->requires_grad()));
    torch::autograd::variable_list out;
    int rc = LSMX_OK;
    if (grad) {
        const bool c = capturing();
        one_stream(*x, c), one_stream(*w, c);
        if (r) one_stream(*r, c);
    }
    {
        NoGil released;
        try {
            if (grad) {
                out = Norm::apply(*x, *w, r ? std::optional<Tensor>(*r) : std::nullopt, eps, mx);
            } else {
                NormOut o = norm_forward(*x, *w, r ? *r : Tensor(), eps, mx);
                for (const Tensor &t : {o.y, o.h, o.codes, o.scale})
                    if (t.defined()) out.push_back(t);
            }
        } catch (const Failed &f) {
            rc = f.rc;
        }
    }
    if (rc != LSMX_OK) {
        Py_XDECREF(PyObject_CallFunction(g_error, "i", rc));
        return nullptr;
    }
    return out.size() > 1 ? wrap_all(out) : THPVariable_Wrap(out[0]);
    END_HANDLE_TH_ERRORS
}

lsmx_route route_args(const Tensor &l, int64_t k, bool sigmoid, int64_t groups, int64_t top, bool renorm, double scale) {
    lsmx_route g{};
    const int64_t E = l.size(-1);
    g.logits = l.data_ptr(), g.dtype = dtype_of(l.scalar_type()), g.rows = l.numel() / E, g.ld = E, g.experts = E, g.k = k;
    g.sigmoid = sigmoid, g.groups = groups, g.top_groups = top, g.renorm = renorm, g.scale = (float)scale;
    return g;
}
struct RouteOut {
    Tensor weights, ids;
};
RouteOut route_forward(const Tensor &l, lsmx_route g) {
    const std::vector<int64_t> shape = with_last(l.sizes(), {g.k}, 1);
    RouteOut o{make(shape, at::kFloat, l), make(shape, at::kInt, l)};
    g.weights = o.weights.data_ptr<float>(), g.ids = o.ids.data_ptr<int32_t>();
    if (const int rc = lsmx_route_fwd(&g, stream_of(l))) throw Failed{rc};
    return o;
}

// The same node as experts._Route, in native code.
struct Route : torch::autograd::Function<Route> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext *ctx, const Tensor &l, const std::optional<Tensor> &bias,
                                                  const std::optional<Tensor> &mask, int64_t k, bool sigmoid, int64_t groups, int64_t top,
                                                  bool renorm, double scale) {
        lsmx_route g = route_args(l, k, sigmoid, groups, top, renorm, scale);
        g.bias = bias ? bias->data_ptr<float>() : nullptr;
        g.mask = mask ? (const uint8_t *)mask->data_ptr() : nullptr;
        const RouteOut o = route_forward(l, g);
        ctx->save_for_backward({l, o.ids});
        ctx->saved_data["k"] = k, ctx->saved_data["sigmoid"] = sigmoid, ctx->saved_data["renorm"] = renorm, ctx->saved_data["scale"] = scale;
        ctx->mark_non_differentiable({o.ids});
        return {o.weights, o.ids};
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
        const auto s = ctx->get_saved_variables();
        const Tensor &l = s[0], &ids = s[1];
        Tensor dl;
        {
            at::AutoGradMode off(false);
            dl = make(l.sizes(), l.scalar_type(), l);
            const Tensor dw = grads[0].defined() ? grads[0].to(at::kFloat).contiguous() : at::zeros_like(ids, at::kFloat);
            // the groups only decide the choice
            lsmx_route g = route_args(l, ctx->saved_data["k"].toInt(), ctx->saved_data["sigmoid"].toBool(), 1, 1,
                                      ctx->saved_data["renorm"].toBool(), ctx->saved_data["scale"].toDouble());
            g.ids = ids.data_ptr<int32_t>();
            must(lsmx_route_bwd(&g, dw.data_ptr<float>(), dl.data_ptr(), stream_of(l)));
        }
        return {once({dl})[0], Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

// route(logits, k, bias, scoring, groups, top_groups, renormalize, scale, mask) -> (weights, experts)
PyObject *route(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    NONE_IF(n != 9);
    const Tensor *l = plain(a[0]), *b = a[2] == Py_None ? nullptr : plain(a[2]), *m = a[8] == Py_None ? nullptr : plain(a[8]);
    int64_t k, groups, top;
    bool renorm;
    NONE_IF(!l || (a[2] != Py_None && !b) || (a[8] != Py_None && !m) || traced() || !int_arg(a[1], 1, false, k) ||
            !int_arg(a[4], 1, false, groups) || !int_arg(a[5], 1, false, top) || !bool_arg(a[6], renorm) ||
            !PyFloat_CheckExact(a[7]) || !PyUnicode_CheckExact(a[3]));
    const bool soft = PyUnicode_CompareWithASCIIString(a[3], "softmax") == 0;
    NONE_IF(!soft && PyUnicode_CompareWithASCIIString(a[3], "sigmoid") != 0);
    NONE_IF(dtype_of(l->scalar_type()) < 0 || l->dim() < 1 || l->numel() == 0 || !l->is_contiguous() || !here(*l) || dual(*l));
    const int64_t E = l->size(-1);
    const at::IntArrayRef lead = l->sizes().slice(0, l->dim() - 1);
    const double scale = PyFloat_AS_DOUBLE(a[7]);
    NONE_IF(E > 1024 || groups > 64 || E % groups || top > groups || k > 64 || k > E / groups * top || !(scale > 0.0 && scale <= 3.0e38) ||
            (b && (!dense(b, at::kFloat) || b->dim() != 1 || b->size(0) != E || b->device() != l->device() || dual(*b))) ||
            (m && (!dense(m, at::kBool) || !m->sizes().equals(lead) || m->device() != l->device())));
    RouteOut o;
    int rc = LSMX_OK;
    const bool grad = at::GradMode::is_enabled() && l->requires_grad();
    if (grad) one_stream(*l, capturing());
    {
        NoGil released;
        try {
            if (grad) {
                const auto v = Route::apply(*l, b ? std::optional<Tensor>(b->detach()) : std::nullopt, m ? std::optional<Tensor>(*m) : std::nullopt,
                                            k, !soft, groups, top, renorm, scale);
                o = {v[0], v[1]};
            } else {
                lsmx_route g = route_args(*l, k, !soft, groups, top, renorm, scale);
                g.bias = b ? b->data_ptr<float>() : nullptr;
                g.mask = m ? (const uint8_t *)m->data_ptr() : nullptr;
                o = route_forward(*l, g);
            }
        } catch (const Failed &f) {
            rc = f.rc;
        }
    }
    if (rc != LSMX_OK) {
        Py_XDECREF(PyObject_CallFunction(g_error, "i", rc));
        return nullptr;
    }
    return wrap2(o.weights, o.ids);
    END_HANDLE_TH_ERRORS
}

// dispatch(experts, num_experts) -> (order, offsets)
PyObject *dispatch(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    NONE_IF(n != 2);
    const Tensor *ids = plain(a[0]);
    int64_t E;
    NONE_IF(!dense(ids, at::kInt) || ids->dim() < 1 || traced() || !int_arg(a[1], 1, false, E) || E > 1024 || ids->numel() == 0 ||
            ids->numel() > (1 << 21) || !here(*ids));
    const int64_t pairs = ids->numel(), nws = lsmx_dispatch_workspace(pairs, E);
    const Tensor order = make({pairs}, at::kInt, *ids), offsets = make({E + 1}, at::kInt, *ids);
    const Tensor ws = nws ? make({nws}, at::kByte, *ids) : Tensor();
    void *s = stream_of(*ids);
    if (!launch([&] {
            return lsmx_dispatch(ids->data_ptr<int32_t>(), pairs, E, order.data_ptr<int32_t>(), offsets.data_ptr<int32_t>(),
                                 nws ? ws.data_ptr() : nullptr, nws, s);
        }))
        return nullptr;
    return wrap2(order, offsets);
    END_HANDLE_TH_ERRORS
}

// The product of experts._check, or false for any form that it would convert or
// refuse.  slots: rows are [.., k, K], else [.., K].
bool experts_of(PyObject *const *a, bool slots, lsmx_experts &g, const Tensor *&x, const Tensor *&ids) {
    if (!PyTuple_Check(a[4]) || PyTuple_GET_SIZE(a[4]) != 3 || traced()) return false;
    const Tensor *xs = plain(a[1]), *w = plain(a[2]), *ws = plain(a[3]);
    const Tensor *order = plain(PyTuple_GET_ITEM(a[4], 1)), *off = plain(PyTuple_GET_ITEM(a[4], 2));
    x = plain(a[0]), ids = plain(PyTuple_GET_ITEM(a[4], 0));
    if (!x || !(dense(x, at::kFloat8_e4m3fn) || dense(x, at::kByte)) || !dense(xs, at::kByte) || !dense(w, at::kByte) ||
        !dense(ws, at::kByte) || !dense(ids, at::kInt) || !dense(order, at::kInt) || !dense(off, at::kInt))
        return false;
    for (const Tensor *t : {xs, w, ws, ids, order, off})
        if (t->device() != x->device()) return false;
    if (!here(*x) || w->dim() != 3 || w->numel() == 0 || ids->dim() < 1 || ids->numel() == 0 || !al(*x, 16) || !al(*w, 16) ||
        !al(*xs, 4) || !al(*ws, 4))
        return false;
    const int64_t E = w->size(0), N = w->size(1), K = 2 * w->size(2), k = ids->size(-1);
    const at::IntArrayRef lead = slots ? ids->sizes() : ids->sizes().slice(0, ids->dim() - 1);
    if (K % 128 || E > 1024 || k > 1024 || ids->numel() > (1 << 21) || N * K / 2 >= ((int64_t)1 << 31) ||
        !ws->sizes().equals({E, N, K / 32}) || !x->sizes().equals(with_last(lead, {K}, 0)) ||
        !xs->sizes().equals(with_last(lead, {K / 32}, 0)) || order->dim() != 1 || order->numel() != ids->numel() ||
        off->dim() != 1 || off->numel() != E + 1)
        return false;
    g = lsmx_experts{(const uint8_t *)x->data_ptr(), xs->data_ptr<uint8_t>(), w->data_ptr<uint8_t>(), ws->data_ptr<uint8_t>(),
                     ids->data_ptr<int32_t>(), order->data_ptr<int32_t>(), off->data_ptr<int32_t>(), ids->numel() / k, k, E, N, K};
    return true;
}

// expert_gated(x, x_scale, w, w_scale, d) -> (h, h_scale)
PyObject *expert_gated(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    NONE_IF(n != 5);
    lsmx_experts g;
    const Tensor *x, *ids;
    NONE_IF(!experts_of(a, false, g, x, ids) || g.N % 64);
    const Tensor h = make(with_last(ids->sizes(), {g.N / 2}, 0), at::kFloat8_e4m3fn, *x);
    const Tensor hs = make(with_last(ids->sizes(), {g.N / 64}, 0), at::kByte, *x);
    void *s = stream_of(*x);
    if (!launch([&] { return lsmx_expert_gated(&g, (uint8_t *)h.data_ptr(), hs.data_ptr<uint8_t>(), s); })) return nullptr;
    return wrap2(h, hs);
    END_HANDLE_TH_ERRORS
}

// expert_combine(h, h_scale, w, w_scale, d, weights, out_dtype) -> y
PyObject *expert_combine(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    NONE_IF(n != 7);
    lsmx_experts g;
    const Tensor *x, *ids, *w = plain(a[5]);
    const at::ScalarType ot = out_type(a[6]);
    NONE_IF(ot == at::ScalarType::Undefined || !dense(w, at::kFloat) || !experts_of(a, true, g, x, ids) ||
            !w->sizes().equals(ids->sizes()) || w->device() != x->device());
    const Tensor y = make(with_last(ids->sizes(), {g.N}, 1), ot, *x);
    const int64_t nws = lsmx_expert_combine_workspace(&g);
    const Tensor ws = make({nws}, at::kByte, *x);
    void *s = stream_of(*x);
    if (!launch([&] { return lsmx_expert_combine(&g, w->data_ptr<float>(), y.data_ptr(), dtype_of(ot), ws.data_ptr(), nws, s); }))
        return nullptr;
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

// init(check, workspace, next_epoch): the _capi functions the calls above use
PyObject *init(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (n != 3) {
        PyErr_SetString(PyExc_TypeError, "init(check, workspace, next_epoch)");
        return nullptr;
    }
    PyObject **g[3] = {&g_error, &g_workspace, &g_epoch};
    for (int i = 0; i < 3; ++i) {
        Py_INCREF(a[i]);
        Py_XDECREF(*g[i]);
        *g[i] = a[i];
    }
    Py_RETURN_NONE;
}

#define FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(init),   FAST(quantize_pack), FAST(quantize_pack2), FAST(quantize), FAST(quantize_2d), FAST(pack),
                         FAST(gemm_packed), FAST(linear), FAST(weight), FAST(gemm_fp8),
                         FAST(attention), FAST(kv_append), FAST(kv_attend), FAST(kv_evict), FAST(rms_norm), FAST(route), FAST(captures),
                         FAST(dispatch), FAST(expert_gated), FAST(expert_combine), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fast", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fast() { return PyModule_Create(&module); }
