// Native host path of the calls that are mostly host work: a prompt into a fresh cache, a dense result, the row codec.  Each of them made ten
// to forty small steps in Python (allocations, views, argument blocks field by field, a library call at a time): 160 us of host for 45 us of
// kernels where 4000 tokens of 8 heads go into a cache that hands dense tensors back, 25 us for the codec's two calls.
//
// Every function takes tensors as they are and checks what the launch relies on: CUDA, current device, types, strides.  Anything but the plain
// case is None, and the caller in Python takes its own path, with its conversions and its errors.  A library error is its negative code.
// The GIL is released around library calls, as ctypes does.
#include <torch/csrc/python_headers.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include <cmath>
#include <cstring>

#include "../../include/tq_abi.h"

namespace {

struct Release {                                        // the GIL, around library calls
    PyThreadState* s = PyEval_SaveThread();
    ~Release() { PyEval_RestoreThread(s); }
};

PyObject* none() { Py_RETURN_NONE; }
PyObject* status(int rc) { return PyLong_FromLong(rc); }
bool is_tensor(PyObject* o) { return THPVariable_Check(o); }
const at::Tensor& tensor(PyObject* o) { return THPVariable_Unpack(o); }
int64_t integer(PyObject* o) { return PyLong_AsLongLong(o); }

int type_code(at::ScalarType t) { return t == at::kHalf ? TQ_F16 : t == at::kBFloat16 ? TQ_BF16 : t == at::kFloat ? TQ_F32 : -1; }
bool here(const at::Tensor& t, int device) { return t.is_cuda() && t.get_device() == device && t.layout() == at::kStrided; }
at::Tensor empty(at::IntArrayRef size, at::ScalarType type, int device) { return at::empty(size, at::TensorOptions().dtype(type).device(at::kCUDA, device)); }
void* stream_of(int device) { return c10::cuda::getCurrentCUDAStream(device).stream(); }

// Rows (B, H, T, D) with one stride per lane and one per row
struct Rows { int64_t b, h, t, d, lane, row; };
bool rows_of(const at::Tensor& x, Rows& r) {
    if (x.dim() != 4 || x.stride(3) != 1) return false;
    r = Rows{x.size(0), x.size(1), x.size(2), x.size(3), 0, 0};
    if (r.b > 1 && r.h > 1 && x.stride(0) != r.h * x.stride(1)) return false;
    r.lane = r.h > 1 ? x.stride(1) : r.b > 1 ? x.stride(0) : 0;
    r.row = r.t > 1 ? x.stride(2) : r.d;
    return true;
}
// ... rows next to one another, lanes a whole number of rows apart that do not overlap: what the row copies take.  src_ls: rows between lanes.
bool copyable(const at::Tensor& x, int64_t first, int64_t n, Rows& r, int64_t& src_ls) {
    if (!rows_of(x, r) || r.row != r.d || first + n > r.t || (r.d * int64_t(x.element_size())) % 16) return false;
    src_ls = r.b * r.h > 1 ? r.lane / r.d : first + n;
    return r.b * r.h == 1 || (r.lane % r.d == 0 && src_ls >= first + n);
}
const char* at_row(const at::Tensor& x, int64_t row) { return static_cast<const char*>(x.data_ptr()) + row * x.size(-1) * int64_t(x.element_size()); }

// ---- row codec -------------------------------------------------------------------------------------------------
// codec_quantize(block, width, x, table): contiguous rows (..., d) -> packed, norms
PyObject* codec_quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 4 || !PyBytes_Check(a[0]) || PyBytes_GET_SIZE(a[0]) != sizeof(tq_quantize_args) || !is_tensor(a[2]) || !is_tensor(a[3])) return none();
    const at::Tensor &x = tensor(a[2]), &table = tensor(a[3]);
    tq_quantize_args q;
    std::memcpy(&q, PyBytes_AS_STRING(a[0]), sizeof q);
    const int device = c10::cuda::current_device(), code = type_code(x.scalar_type());
    if (code < 0 || !here(x, device) || !here(table, device) || x.dim() < 1 || x.size(-1) != q.d || !x.is_contiguous()) return none();
    auto size = x.sizes().vec();
    size.back() = integer(a[1]);
    at::Tensor packed = empty(size, at::kByte, device);
    size.pop_back();
    at::Tensor norms = empty(size, at::kFloat, device);
    q.x = x.data_ptr(); q.x_dtype = code;
    q.packed_hi = packed.data_ptr<uint8_t>(); q.norms = norms.data_ptr<float>();
    q.n_rows = q.out_lane_stride = norms.numel();
    int rc;
    {
        Release gil;
        rc = tq_quantize_pack(&q, stream_of(device));
    }
    if (rc) return status(rc);
    return PyTuple_Pack(2, THPObjectPtr(THPVariable_Wrap(packed)).get(), THPObjectPtr(THPVariable_Wrap(norms)).get());
    END_HANDLE_TH_ERRORS
}
// codec_dequantize(block, width, packed, norms, table): -> float32 rows
PyObject* codec_dequantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 5 || !PyBytes_Check(a[0]) || PyBytes_GET_SIZE(a[0]) != sizeof(tq_dequantize_args) || !is_tensor(a[2]) || !is_tensor(a[3]) || !is_tensor(a[4])) return none();
    const at::Tensor &packed = tensor(a[2]), &norms = tensor(a[3]), &table = tensor(a[4]);
    tq_dequantize_args r;
    std::memcpy(&r, PyBytes_AS_STRING(a[0]), sizeof r);
    const int device = c10::cuda::current_device();
    if (!here(packed, device) || !here(norms, device) || !here(table, device) || packed.scalar_type() != at::kByte || norms.scalar_type() != at::kFloat ||
        !packed.is_contiguous() || !norms.is_contiguous() || packed.numel() != norms.numel() * integer(a[1]))
        return none();
    auto size = norms.sizes().vec();
    size.push_back(r.d);
    at::Tensor out = empty(size, at::kFloat, device);
    r.packed_hi = packed.data_ptr<uint8_t>(); r.norms = norms.data_ptr<float>(); r.out = out.data_ptr();
    r.n_rows = r.in_lane_stride = norms.numel();
    r.out_lane_stride = r.n_rows * r.d;
    int rc;
    {
        Release gil;
        rc = tq_dequantize(&r, stream_of(device));
    }
    return rc ? status(rc) : THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// ---- token buffers ---------------------------------------------------------------------------------------------
// Whether keys and values (and the buffers they go with) agree in type, shape and strides
bool pair_of(const at::Tensor& k, const at::Tensor& v, int device) {
    return here(k, device) && here(v, device) && k.dim() == 4 && k.scalar_type() == v.scalar_type() && k.sizes() == v.sizes() && k.strides() == v.strides();
}
bool buffers_of(const at::Tensor& k, const at::Tensor& v, const at::Tensor& like, int device) {
    return pair_of(k, v, device) && k.scalar_type() == like.scalar_type() && k.size(0) == like.size(0) && k.size(1) == like.size(1) && k.size(3) == like.size(3) &&
           k.is_contiguous();
}
// append(k_buf, v_buf, k_new, v_new, first, n, row): rows [first, first + n) of the new tokens to rows row, ... of the buffers -> status
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    if (n_args != 7) return none();
    for (int i = 0; i < 4; ++i)
        if (!is_tensor(a[i])) return none();
    const at::Tensor &kb = tensor(a[0]), &vb = tensor(a[1]), &k = tensor(a[2]), &v = tensor(a[3]);
    const int64_t first = integer(a[4]), n = integer(a[5]), row = integer(a[6]);
    const int device = c10::cuda::current_device();
    Rows r;
    int64_t src_ls;
    if (!pair_of(k, v, device) || !buffers_of(kb, vb, k, device) || !copyable(k, first, n, r, src_ls) || row + n > kb.size(2)) return none();
    int rc;
    {
        Release gil;
        rc = tq_append_tokens(at_row(k, first), at_row(v, first), kb.data_ptr(), vb.data_ptr(), r.b * r.h, n, r.d * int64_t(k.element_size()), src_ls, kb.size(2), row, stream_of(device));
    }
    return rc == TQ_ERR_UNSUPPORTED ? none() : status(rc);
    END_HANDLE_TH_ERRORS
}
// buffers(k_new, v_new, first, n, capacity, k_old, v_old, old_first, kept): fresh buffers (B, H, capacity, D) x 2: kept rows of the old ones, then
// rows [first, first + n) of the new tokens, then zeros
PyObject* buffers(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    if (n_args != 9 || !is_tensor(a[0]) || !is_tensor(a[1])) return none();
    const at::Tensor &k = tensor(a[0]), &v = tensor(a[1]);
    const int64_t first = integer(a[2]), n = integer(a[3]), cap = integer(a[4]), old_first = integer(a[7]), kept = integer(a[8]);
    const int device = c10::cuda::current_device();
    Rows r;
    int64_t src_ls;
    if (!pair_of(k, v, device) || type_code(k.scalar_type()) < 0 || !copyable(k, first, n, r, src_ls)) return none();
    const char *k_old = nullptr, *v_old = nullptr;
    int64_t old_ls = 0;
    if (kept > 0) {
        if (!is_tensor(a[5]) || !is_tensor(a[6])) return none();
        const at::Tensor &ko = tensor(a[5]), &vo = tensor(a[6]);
        if (!buffers_of(ko, vo, k, device) || old_first + kept > ko.size(2)) return none();
        k_old = at_row(ko, old_first); v_old = at_row(vo, old_first); old_ls = ko.size(2);
    }
    const int64_t size[4] = {r.b, r.h, cap, r.d};
    at::Tensor kb = empty(size, k.scalar_type(), device), vb = empty(size, k.scalar_type(), device);
    int rc;
    {
        Release gil;
        rc = tq_fill_tokens(k_old, v_old, kept, old_ls, n > 0 ? at_row(k, first) : nullptr, n > 0 ? at_row(v, first) : nullptr, n, src_ls, kb.data_ptr(), vb.data_ptr(), r.b * r.h,
                            r.d * int64_t(k.element_size()), cap, stream_of(device));
    }
    if (rc) return rc == TQ_ERR_UNSUPPORTED ? none() : status(rc);
    return PyTuple_Pack(2, THPObjectPtr(THPVariable_Wrap(kb)).get(), THPObjectPtr(THPVariable_Wrap(vb)).get());
    END_HANDLE_TH_ERRORS
}

// ---- packed storage --------------------------------------------------------------------------------------------
// storage(b, h, capacity, width_hi, width_lo, sketches, device): codes, second codes or None, norms, sign words or None, residual norms or None
PyObject* storage(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 7) return none();
    const int64_t b = integer(a[0]), h = integer(a[1]), cap = integer(a[2]), w_hi = integer(a[3]), w_lo = integer(a[4]);
    const bool sketches = PyObject_IsTrue(a[5]) == 1;
    const int device = int(integer(a[6]));
    const int64_t hi[4] = {b, h, cap, w_hi}, lo[4] = {b, h, cap, w_lo}, one[3] = {b, h, cap};
    auto wrap = [](at::Tensor t) { return THPVariable_Wrap(std::move(t)); };
    auto absent = [] { Py_INCREF(Py_None); return Py_None; };
    THPObjectPtr t0(wrap(empty(hi, at::kByte, device))), t1(w_lo > 0 ? wrap(empty(lo, at::kByte, device)) : absent()), t2(wrap(empty(one, at::kFloat, device))),
        t3(sketches ? wrap(empty(one, at::kInt, device)) : absent()), t4(sketches ? wrap(empty(one, at::kFloat, device)) : absent());
    return PyTuple_Pack(5, t0.get(), t1.get(), t2.get(), t3.get(), t4.get());
    END_HANDLE_TH_ERRORS
}
// quantize(at, sides...): per side (block, buffer or None, old, new, n_new, hi, lo or None, norms, sign words or None, residual norms or None): the
// first `old` rows of the buffer and the first n_new of the new tokens to packed rows at, at + old, ... -> status
PyObject* quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n < 2 || n > 3) return none();
    const int64_t at0 = integer(a[0]);
    const int device = c10::cuda::current_device();
    tq_quantize_args jobs[4];
    int count = 0;
    for (Py_ssize_t i = 1; i < n; ++i) {
        if (!PyTuple_Check(a[i]) || PyTuple_GET_SIZE(a[i]) != 10) return none();
        PyObject* const* f = &PyTuple_GET_ITEM(a[i], 0);
        if (!PyBytes_Check(f[0]) || PyBytes_GET_SIZE(f[0]) != sizeof(tq_quantize_args) || !is_tensor(f[5]) || !is_tensor(f[7])) return none();
        const at::Tensor &hi = tensor(f[5]), &norms = tensor(f[7]);
        if (!here(hi, device) || !here(norms, device) || !hi.is_contiguous() || !norms.is_contiguous()) return none();
        const int64_t rows[2] = {integer(f[2]), integer(f[4])};
        int64_t row = at0;
        for (int part = 0; part < 2; ++part) {
            if (rows[part] == 0) continue;
            PyObject* src = f[part ? 3 : 1];
            if (!is_tensor(src)) return none();
            const at::Tensor& x = tensor(src);
            const int code = type_code(x.scalar_type());
            Rows r;
            // (one stride per lane and per row; an expanded axis, stride 0, is not for the tensor-core kernel)
            if (code < 0 || !here(x, device) || !rows_of(x, r) || rows[part] > r.t || (r.h > 1 && x.stride(1) == 0) || (r.b > 1 && x.stride(0) == 0) || (r.t > 1 && x.stride(2) == 0) ||
                r.b != hi.size(0) || r.h != hi.size(1) || row + rows[part] > hi.size(2))
                return none();
            tq_quantize_args& q = jobs[count++];
            std::memcpy(&q, PyBytes_AS_STRING(f[0]), sizeof q);
            if (r.d != q.d) return none();
            q.x = x.data_ptr(); q.x_dtype = code; q.n_lanes = r.b * r.h; q.n_rows = rows[part];
            q.x_lane_stride = r.lane; q.x_row_stride = r.row;
            q.packed_hi = hi.data_ptr<uint8_t>() + row * hi.size(3); q.norms = norms.data_ptr<float>() + row; q.out_lane_stride = hi.size(2);
            if (is_tensor(f[6])) {
                const at::Tensor& lo = tensor(f[6]);
                q.packed_lo = lo.data_ptr<uint8_t>() + row * lo.size(3);
            }
            if (q.qjl_proj_rot && is_tensor(f[8]) && is_tensor(f[9])) {
                q.qjl_bits = reinterpret_cast<uint32_t*>(tensor(f[8]).data_ptr<int32_t>()) + row;
                q.qjl_gamma = tensor(f[9]).data_ptr<float>() + row;
            }
            row += rows[part];
        }
    }
    int rc;
    {
        Release gil;
        rc = tq_quantize_pack_many(jobs, count, stream_of(device));
    }
    return status(rc);
    END_HANDLE_TH_ERRORS
}

// ---- dense result ----------------------------------------------------------------------------------------------
// fetch(sink_k, sink_v, sink_len, keys, values, recent_len, packed_len, k_side, v_side, dense_k, dense_v): dense keys and values
// [sink | packed | recent]; a side is (block, hi, lo or None, norms); with dense tensors the middle is copied from them
PyObject* fetch(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 11) return none();
    const int device = c10::cuda::current_device();
    const int64_t len[3] = {integer(a[2]), integer(a[5]), integer(a[6])};
    tq_fetch_args f;
    std::memset(&f, 0, sizeof f);
    const int64_t rows = len[0] + len[1] + len[2];
    int64_t b = 0, h = 0, d = 0;
    at::ScalarType type = at::kFloat;
    auto part = [&](int i, PyObject* ko, PyObject* vo, int64_t count, int64_t dst) -> bool {
        if (count == 0) return true;
        if (!is_tensor(ko) || !is_tensor(vo)) return false;
        const at::Tensor &k = tensor(ko), &v = tensor(vo);
        if (!pair_of(k, v, device) || type_code(k.scalar_type()) < 0 || !k.is_contiguous() || count > k.size(2)) return false;
        if (d == 0) { b = k.size(0); h = k.size(1); d = k.size(3); if (len[2] == 0) type = k.scalar_type(); }
        if (k.size(0) != b || k.size(1) != h || k.size(3) != d || (type != at::kFloat && k.scalar_type() != type)) return false;
        tq_fetch_part& p = f.part[i];
        p.k = k.data_ptr(); p.v = v.data_ptr(); p.dtype = type_code(k.scalar_type()); p.rows = count; p.lane_stride = k.size(2); p.dst_row = dst;
        return true;
    };
    // (the recent tokens' type is the result's where nothing is packed)
    if (!part(1, a[3], a[4], len[1], len[0] + len[2]) || !part(0, a[0], a[1], len[0], 0) || d == 0 || d % 8) return none();
    const bool expanded = is_tensor(a[9]);
    if (len[2] > 0 && expanded && !part(2, a[9], a[10], len[2], len[0])) return none();
    tq_dequantize_args jobs[2];
    const bool unpack = len[2] > 0 && !expanded;
    for (int i = 0; unpack && i < 2; ++i) {
        PyObject* side = a[7 + i];
        if (!PyTuple_Check(side) || PyTuple_GET_SIZE(side) != 4) return none();
        PyObject* const* s = &PyTuple_GET_ITEM(side, 0);
        if (!PyBytes_Check(s[0]) || PyBytes_GET_SIZE(s[0]) != sizeof(tq_dequantize_args) || !is_tensor(s[1]) || !is_tensor(s[3])) return none();
        const at::Tensor &hi = tensor(s[1]), &norms = tensor(s[3]);
        if (!here(hi, device) || !here(norms, device) || !hi.is_contiguous() || !norms.is_contiguous() || hi.size(0) != b || hi.size(1) != h || len[2] > hi.size(2)) return none();
        std::memcpy(&jobs[i], PyBytes_AS_STRING(s[0]), sizeof jobs[i]);
        if (jobs[i].d != d) return none();
        jobs[i].packed_hi = hi.data_ptr<uint8_t>(); jobs[i].norms = norms.data_ptr<float>();
        if (is_tensor(s[2])) jobs[i].packed_lo = tensor(s[2]).data_ptr<uint8_t>();
        jobs[i].n_lanes = b * h; jobs[i].n_rows = len[2]; jobs[i].in_lane_stride = hi.size(2);
    }
    const int64_t size[4] = {b, h, rows, d};
    at::Tensor k = empty(size, type, device), v = empty(size, type, device);
    for (int i = 0; unpack && i < 2; ++i) {
        jobs[i].out = (i ? v : k).data_ptr<float>() + len[0] * d;
        jobs[i].out_dtype = TQ_F32; jobs[i].out_lane_stride = rows * d;
    }
    f.lanes = b * h; f.out_rows = rows; f.d = int(d); f.out_dtype = type_code(type); f.k_out = k.data_ptr(); f.v_out = v.data_ptr();
    int rc;
    {
        Release gil;
        rc = tq_fetch_dense(&f, unpack ? &jobs[0] : nullptr, unpack ? &jobs[1] : nullptr, stream_of(device));
    }
    if (rc) return rc == TQ_ERR_UNSUPPORTED ? none() : status(rc);
    return PyTuple_Pack(2, THPObjectPtr(THPVariable_Wrap(k)).get(), THPObjectPtr(THPVariable_Wrap(v)).get());
    END_HANDLE_TH_ERRORS
}

// ---- rotary positions, 8-bit blocks ----------------------------------------------------------------------------------
// Inference only: what asks for a gradient goes back to Python, which refuses it.
bool plain(const at::Tensor& t, int device) { return here(t, device) && !(t.requires_grad() && c10::GradMode::is_enabled()); }
// Rows (B, H, T, D) of contiguous coordinates that start on 16 bytes
bool rows16(const at::Tensor& x, tq_new_rows& r) {
    const int64_t n = 16 / int64_t(x.element_size());
    if (x.stride(3) != 1 || reinterpret_cast<uintptr_t>(x.data_ptr()) % 16) return false;
    int64_t st[3];
    for (int i = 0; i < 3; ++i) {
        st[i] = x.size(i) > 1 ? x.stride(i) : 0;
        if (st[i] % n) return false;
    }
    r = tq_new_rows{x.data_ptr(), st[0], st[1], st[2]};
    return true;
}
// rotary(q, k or None, freqs, offset, positions or None, interleaved, factor) -> (q, k or None)
PyObject* rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 7 || !is_tensor(a[0]) || !is_tensor(a[2])) return none();
    const int device = c10::cuda::current_device();
    const at::Tensor &q = tensor(a[0]), &f = tensor(a[2]);
    const int code = type_code(q.scalar_type());
    if (code < 0 || !plain(q, device) || q.dim() != 4 || !here(f, device) || f.scalar_type() != at::kDouble || f.dim() != 1 || !f.is_contiguous() || f.numel() == 0 ||
        2 * f.numel() > q.size(3) || !PyLong_Check(a[3]))
        return none();
    tq_rotary_args r;
    std::memset(&r, 0, sizeof r);
    r.dtype = code; r.batch = int(q.size(0)); r.length = q.size(2); r.d = int(q.size(3)); r.dims = int(2 * f.numel());
    r.freqs = f.data_ptr<double>(); r.offset = integer(a[3]); r.interleaved = PyObject_IsTrue(a[5]) == 1;
    r.factor = float(PyFloat_AsDouble(a[6]));
    if (PyErr_Occurred()) { PyErr_Clear(); return none(); }
    if (a[4] != Py_None) {
        if (!is_tensor(a[4])) return none();
        const at::Tensor& pos = tensor(a[4]);
        const bool each = pos.dim() == 2;
        if (!here(pos, device) || pos.scalar_type() != at::kLong || pos.dim() < 1 || pos.dim() > 2 || pos.size(-1) != r.length || (each && pos.size(0) != r.batch) ||
            (r.length > 1 && pos.stride(-1) != 1))
            return none();
        r.positions = pos.data_ptr<int64_t>();
        r.pos_sb = each && r.batch > 1 ? pos.stride(0) : 0;
    }
    at::Tensor out[2];
    for (int i = 0; i < 2; ++i) {
        if (i && a[1] == Py_None) continue;
        if (!is_tensor(a[i])) return none();
        const at::Tensor& x = tensor(a[i]);
        if (!plain(x, device) || x.dim() != 4 || x.scalar_type() != q.scalar_type() || x.size(0) != r.batch || x.size(2) != r.length || x.size(3) != r.d || x.stride(3) != 1) return none();
        out[i] = empty(x.sizes(), x.scalar_type(), device);
        r.part[i] = tq_rotary_rows{x.data_ptr(), x.stride(0), x.stride(1), x.stride(2), out[i].data_ptr(), int(x.size(1))};
    }
    int rc;
    {
        Release gil;
        rc = tq_rotary(&r, stream_of(device));
    }
    if (rc) return status(rc);
    THPObjectPtr first(THPVariable_Wrap(out[0])), second(out[1].defined() ? THPVariable_Wrap(out[1]) : none());
    return PyTuple_Pack(2, first.get(), second.get());
    END_HANDLE_TH_ERRORS
}
// k_codes, k_scales, v_codes, v_scales, k_tail, v_tail
bool store_of(PyObject* const* a, int64_t length, int device, tq_block_store& s) {
    for (int i = 0; i < 6; ++i)
        if (!is_tensor(a[i]) || !here(tensor(a[i]), device) || !tensor(a[i]).is_contiguous()) return false;
    const at::Tensor &kc = tensor(a[0]), &ks = tensor(a[1]), &vc = tensor(a[2]), &vs = tensor(a[3]), &kt = tensor(a[4]), &vt = tensor(a[5]);
    const auto type = kc.scalar_type();
    const int code = type_code(kt.scalar_type());
    if ((type != at::kChar && type != at::kFloat8_e4m3fn) || vc.scalar_type() != type || ks.scalar_type() != at::kFloat || vs.scalar_type() != at::kFloat || code < 0 ||
        vt.scalar_type() != kt.scalar_type() || kc.dim() != 4 || ks.dim() != 3 || kt.dim() != 4)
        return false;
    const int64_t b = kc.size(0), h = kc.size(1), cap = kc.size(2), d = kc.size(3), block = kt.size(2);
    if ((block != 16 && block != 32 && block != 64 && block != 128) || vc.sizes() != kc.sizes() || kt.size(0) != b || kt.size(1) != h || kt.size(3) != d || vt.sizes() != kt.sizes() ||
        cap % block || ks.size(0) != b || ks.size(1) != h || ks.size(2) != cap / block || vs.sizes() != ks.sizes() || length < 0 || length / block * block > cap)
        return false;
    s = tq_block_store{int(b), int(h), int(d), int(block), type == at::kChar ? TQ_CODE_INT8 : TQ_CODE_E4M3, code, kc.data_ptr(), vc.data_ptr(), ks.data_ptr<float>(), vs.data_ptr<float>(),
                       kt.data_ptr(), vt.data_ptr(), cap, length};
    return true;
}
bool new_rows(PyObject* ko, PyObject* vo, const at::Tensor& tail, int device, tq_new_rows& k, tq_new_rows& v, int64_t& t) {
    if (!is_tensor(ko) || !is_tensor(vo)) return false;
    const at::Tensor &kn = tensor(ko), &vn = tensor(vo);
    if (!plain(kn, device) || !plain(vn, device) || kn.dim() != 4 || kn.sizes() != vn.sizes() || kn.scalar_type() != tail.scalar_type() || vn.scalar_type() != tail.scalar_type() ||
        kn.size(0) != tail.size(0) || kn.size(1) != tail.size(1) || kn.size(3) != tail.size(3) || !rows16(kn, k) || !rows16(vn, v))
        return false;
    t = kn.size(2);
    return true;
}
// blocks_write(keys, values, storage x 6, length) -> the new length
PyObject* blocks_write(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 9 || !PyLong_Check(a[8])) return none();
    const int device = c10::cuda::current_device();
    const int64_t length = integer(a[8]);
    tq_block_store s;
    tq_new_rows k, v;
    int64_t t = 0;
    if (!store_of(a + 2, length, device, s) || !new_rows(a[0], a[1], tensor(a[6]), device, k, v, t) || (length + t) / s.block * s.block > s.capacity) return none();
    int rc;
    {
        Release gil;
        rc = tq_blocks_write(&s, &k, &v, t, stream_of(device));
    }
    return rc ? status(rc) : PyLong_FromLongLong(length + t);
    END_HANDLE_TH_ERRORS
}
// blocks_read(storage x 6, length) -> dense keys and values of the tails' type
PyObject* blocks_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 7 || !PyLong_Check(a[6])) return none();
    const int device = c10::cuda::current_device();
    const int64_t length = integer(a[6]);
    tq_block_store s;
    if (!store_of(a, length, device, s)) return none();
    const int64_t size[4] = {s.batch, s.n_kv_heads, length, s.d};
    const auto type = tensor(a[4]).scalar_type();
    at::Tensor k = empty(size, type, device), v = empty(size, type, device);
    int rc;
    {
        Release gil;
        rc = tq_blocks_read(&s, k.data_ptr(), v.data_ptr(), s.dtype, stream_of(device));
    }
    if (rc) return status(rc);
    return PyTuple_Pack(2, THPObjectPtr(THPVariable_Wrap(k)).get(), THPObjectPtr(THPVariable_Wrap(v)).get());
    END_HANDLE_TH_ERRORS
}
// blocks_attend(queries, storage x 6, length, window or 0, sinks, scale or None, new keys or None, new values or None, out or None) -> result
PyObject* blocks_attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 14 || !is_tensor(a[0]) || !PyLong_Check(a[7]) || !PyLong_Check(a[8]) || !PyLong_Check(a[9])) return none();
    const int device = c10::cuda::current_device();
    const at::Tensor& q = tensor(a[0]);
    tq_blocks_attend_args r;
    std::memset(&r, 0, sizeof r);
    const int64_t length = integer(a[7]);
    if (!store_of(a + 1, length, device, r.store)) return none();
    const tq_block_store& s = r.store;
    if (!plain(q, device) || q.dim() != 4 || q.scalar_type() != tensor(a[5]).scalar_type() || q.size(0) != s.batch || q.size(3) != s.d || s.n_kv_heads == 0 || q.size(1) % s.n_kv_heads ||
        q.numel() == 0 || !rows16(q, r.q))
        return none();
    r.n_q_heads = int(q.size(1)); r.t_q = q.size(2);
    r.window = integer(a[8]); r.sinks = integer(a[9]);
    r.scale = a[10] == Py_None ? float(1.0 / std::sqrt(double(s.d))) : float(PyFloat_AsDouble(a[10]));
    if (PyErr_Occurred()) { PyErr_Clear(); return none(); }
    int64_t t = 0;
    if (a[11] != Py_None && (r.t_q != 1 || length % s.block + 1 == s.block || !new_rows(a[11], a[12], tensor(a[5]), device, r.k_new, r.v_new, t) || t != 1)) return none();
    if (r.window < 0 || r.sinks < 0 || r.t_q > length + t) return none();
    at::Tensor out, ws;
    if (a[13] == Py_None) {
        out = empty(q.sizes(), q.scalar_type(), device);
    } else {
        if (!is_tensor(a[13])) return none();
        out = tensor(a[13]);
        if (!here(out, device) || out.sizes() != q.sizes() || out.scalar_type() != q.scalar_type() || !out.is_contiguous() || reinterpret_cast<uintptr_t>(out.data_ptr()) % 16) return none();
    }
    r.out = out.data_ptr();
    // without room for the scratch that the call would like: Python takes it from here, with less
    r.workspace_bytes = tq_blocks_attend_workspace(&r);
    if (r.workspace_bytes) {
        try {
            ws = empty({int64_t(r.workspace_bytes)}, at::kByte, device);
        } catch (const c10::OutOfMemoryError&) {
            return none();
        }
        r.workspace = ws.data_ptr();
    }
    int rc;
    {
        Release gil;
        rc = tq_blocks_attend(&r, stream_of(device));
    }
    if (rc) return status(rc);
    if (a[13] != Py_None) {
        Py_INCREF(a[13]);
        return a[13];
    }
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

#define FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(codec_quantize), FAST(codec_dequantize), FAST(append), FAST(buffers), FAST(storage), FAST(quantize), FAST(fetch), FAST(rotary), FAST(blocks_write), FAST(blocks_read), FAST(blocks_attend),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", "Native host path; see csrc/host.cpp.", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__host() {
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "built_for", TQ_BUILT_FOR)) Py_CLEAR(m);       // (the loader compares it with what is running)
    return m;
}
