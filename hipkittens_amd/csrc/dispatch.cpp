// The dispatchers' argument checks and launches (GEMMs; the operators of training)
// for ordinary arguments, as a CPython module (`_dispatch`).
//
// A launch takes the runtime about 3 us; the same checks in Python, a call through ctypes and the attribute reads for it
// took 3 (FP8, BF16) to 6 us (MXFP4 with a workspace: six tensors) on top, which is what a GEMM of a few microseconds
// then costs. Per call, host, us, in Python / here: MXFP4 6 x 704 x 1536 8.4 (with a workspace 9.9) / 3.7 (3.9), FP8 6.8 / 3.6,
// BF16 6.2 / 3.5.
//
// Every function returns the library's status, or None where an argument is not what it knows (another type or device, a
// shape that does not fit, a subclass or a wrapper of a transform): the Python dispatcher then runs its own checks, which
// accept or refuse the call with their messages. No call is refused here. The module is not a condition either: where it is
// absent or built for another torch or Python (build_tag), every call is left to the Python dispatchers.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>
#include <limits>

#include "../../include/hk355.h"

namespace {

// the library's entry points, by address (it is loaded by _lib.py)
struct Entries {
    decltype(&hk_fp8_gemm) fp8;
    decltype(&hk_fp8_gemm_ws) fp8_ws;
    decltype(&hk_bf16_gemm) bf16;
    decltype(&hk_bf16_gemm_ws) bf16_ws;
    decltype(&hk_mxfp4_gemm) mxfp4;
    decltype(&hk_mxfp4_gemm_ws) mxfp4_ws;
    decltype(&hk_mxfp4_gemm_pitched) mxfp4_pitched;
    decltype(&hk_mxfp4_quantize_rows) mxfp4_quantize;
    decltype(&hk_moe_permute) permute;
    decltype(&hk_moe_permute_backward) permute_backward;
    decltype(&hk_moe_unpermute_backward) unpermute_backward;
    decltype(&hk_moe_grouped_gemm) grouped;
    decltype(&hk_moe_grouped_gemm_dgrad) grouped_dgrad;
    decltype(&hk_moe_grouped_gemm_wgrad) grouped_wgrad;
    decltype(&hk_linear_cross_entropy) head_loss;
    decltype(&hk_linear_cross_entropy_backward) head_gradients;
    decltype(&hk_gated_gemm) gated;
    decltype(&hk_gated_gemm_dgrad) gated_dgrad;
    decltype(&hk_bf16_gemm_dgrad) dense_dgrad;
    decltype(&hk_bf16_gemm_wgrad) dense_wgrad;
    decltype(&hk_embedding) embedding;
    decltype(&hk_embedding_backward) embedding_backward;
    decltype(&hk_grad_norm) grad_norm;
    decltype(&hk_grad_clip) grad_clip;
};
Entries entries{};
PyTypeObject* parameter_type = nullptr;

struct Operand {
    void* data;
    int64_t outer, rows, cols;   // cols of a vector: its length; outer: matrices of a stack
    int device;
};

using Types = std::initializer_list<at::ScalarType>;

// A plain contiguous GPU tensor of `ndim` dimensions (1 to 3) and one of `types`, nothing around its memory.
bool operand(PyObject* o, Types types, int ndim, Operand& out) {
    if (Py_TYPE(o) != reinterpret_cast<PyTypeObject*>(THPVariableClass) && Py_TYPE(o) != parameter_type) return false;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || !t.unsafeGetTensorImpl()->has_storage()) return false;
    using c10::DispatchKey;
    constexpr c10::DispatchKeySet wrapped({DispatchKey::Python, DispatchKey::PythonTLSSnapshot, DispatchKey::Functionalize,
                                           DispatchKey::FuncTorchBatched, DispatchKey::FuncTorchGradWrapper,
                                           DispatchKey::Negative, DispatchKey::Conjugate, DispatchKey::ZeroTensor});
    if (t.key_set().has_any(wrapped) || t.dim() != ndim || !t.is_contiguous()) return false;
    const at::ScalarType type = t.scalar_type();
    bool known = false;
    for (const at::ScalarType s : types) known = known || s == type;
    if (!known) return false;
    const auto sizes = t.sizes();
    out.outer = ndim == 3 ? sizes[0] : 1;
    out.rows = ndim >= 2 ? sizes[ndim - 2] : 1;
    out.cols = sizes[ndim - 1];
    out.device = t.device().index();
    constexpr int64_t kMax = std::numeric_limits<int>::max();
    if (out.outer > kMax || out.rows > kMax || (ndim >= 2 && out.cols > kMax / 2)) return false;
    out.data = t.data_ptr();
    return true;
}
bool number(PyObject* o, float& out) {
    if (!PyFloat_CheckExact(o)) return false;
    out = static_cast<float>(PyFloat_AS_DOUBLE(o));
    return true;
}
void* stream_of(int device) { return c10::hip::getCurrentHIPStream(static_cast<c10::DeviceIndex>(device)).stream(); }

// The call with the interpreter's lock released (a full queue makes a launch wait).
template <typename F>
PyObject* launch(F&& f) {
    int status;
    Py_BEGIN_ALLOW_THREADS;
    status = f();
    Py_END_ALLOW_THREADS;
    return PyLong_FromLong(status);
}
// A C++ exception must not cross into the interpreter: the call is left to the Python dispatcher.
template <typename F>
PyObject* guarded(F&& f) {
    try {
        return f();
    } catch (...) {
        Py_RETURN_NONE;
    }
}

constexpr Types kFp8{at::kFloat8_e4m3fn, at::kByte}, kBf16{at::kBFloat16}, kByte{at::kByte},
    kFp4{at::kByte, at::ScalarType::Float4_e2m1fn_x2}, kE8m0{at::kByte, at::ScalarType::Float8_e8m0fnu};

// (A, B, C, scale_a, scale_b, workspace or None)
PyObject* fp8_gemm(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        Operand a, b, c, ws{};
        float sa, sb;
        if (n != 6 || !operand(args[0], kFp8, 2, a) || !operand(args[1], kFp8, 2, b) || !operand(args[2], kBf16, 2, c) ||
            !number(args[3], sa) || !number(args[4], sb) || (args[5] != Py_None && !operand(args[5], kByte, 1, ws)) ||
            a.cols != b.cols || c.rows != a.rows || c.cols != b.rows || a.device != b.device || a.device != c.device)
            Py_RETURN_NONE;
        const int M = (int)a.rows, N = (int)b.rows, K = (int)a.cols;
        void* s = stream_of(a.device);
        if (args[5] != Py_None)
            return launch([&] { return entries.fp8_ws(a.data, b.data, c.data, M, N, K, sa, sb, ws.data, (size_t)ws.cols, s); });
        return launch([&] { return entries.fp8(a.data, b.data, c.data, M, N, K, sa, sb, s); });
    });
}

// (A, B, C, workspace or None)
PyObject* bf16_gemm(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        Operand a, b, c, ws{};
        if (n != 4 || !operand(args[0], kBf16, 2, a) || !operand(args[1], kBf16, 2, b) || !operand(args[2], kBf16, 2, c) ||
            (args[3] != Py_None && !operand(args[3], kByte, 1, ws)) || a.cols != b.cols || c.rows != a.rows ||
            c.cols != b.rows || a.device != b.device || a.device != c.device)
            Py_RETURN_NONE;
        const int M = (int)a.rows, N = (int)b.rows, K = (int)a.cols;
        void* s = stream_of(a.device);
        if (args[3] != Py_None)
            return launch([&] { return entries.bf16_ws(a.data, b.data, c.data, M, N, K, ws.data, (size_t)ws.cols, s); });
        return launch([&] { return entries.bf16(a.data, b.data, c.data, M, N, K, s); });
    });
}

// (A, A_scales, B, B_scales, C, workspace or None)
PyObject* mxfp4_gemm(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        Operand a, as, b, bs, c, ws{};
        if (n != 6 || !operand(args[0], kFp4, 2, a) || !operand(args[1], kE8m0, 2, as) || !operand(args[2], kFp4, 2, b) ||
            !operand(args[3], kE8m0, 2, bs) || !operand(args[4], kBf16, 2, c) ||
            (args[5] != Py_None && (!operand(args[5], kByte, 1, ws) || ws.device != a.device)))
            Py_RETURN_NONE;
        const int64_t K = 2 * a.cols;
        if (b.cols != a.cols || K % 32 != 0 || as.rows != a.rows || as.cols < K / 32 || bs.rows != b.rows ||
            bs.cols < K / 32 || c.rows != a.rows || c.cols != b.rows || as.device != a.device || b.device != a.device ||
            bs.device != a.device || c.device != a.device)
            Py_RETURN_NONE;
        const int M = (int)a.rows, N = (int)b.rows, pa = (int)as.cols, pb = (int)bs.cols, k = (int)K;
        void* s = stream_of(a.device);
        if (args[5] != Py_None)
            return launch([&] {
                return entries.mxfp4_ws(a.data, as.data, pa, b.data, bs.data, pb, c.data, M, N, k, ws.data, (size_t)ws.cols, s);
            });
        if (pa != k / 32 || pb != k / 32)
            return launch([&] { return entries.mxfp4_pitched(a.data, as.data, pa, b.data, bs.data, pb, c.data, M, N, k, s); });
        return launch([&] { return entries.mxfp4(a.data, as.data, b.data, bs.data, c.data, M, N, k, s); });
    });
}

// (x, packed, scales)
PyObject* mxfp4_quantize_rows(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        Operand x, p, sc;
        if (n != 3 || !operand(args[0], kBf16, 2, x) || !operand(args[1], kFp4, 2, p) || !operand(args[2], kE8m0, 2, sc) ||
            p.rows != x.rows || p.cols != x.cols / 2 || sc.rows != x.rows || p.device != x.device || sc.device != x.device)
            Py_RETURN_NONE;
        void* s = stream_of(x.device);
        return launch([&] {
            return entries.mxfp4_quantize(x.data, (int)x.rows, (int)x.cols, p.data, sc.data, (int)sc.cols, s);
        });
    });
}

constexpr Types kF32{at::kFloat}, kI32{at::kInt};
// The training entry points ask the runtime about the current device (compute units, LDS limits): calls for another one are
// left to Python, which makes it the current one.
bool current(int device) { return device == static_cast<int>(c10::hip::current_device()); }
// rows [T k, H] and slot_to_pos [T k] of tokens [T, H]
bool routed_rows(const Operand& tokens, const Operand& rows, const Operand& pos) {
    return tokens.rows > 0 && rows.rows > 0 && rows.rows % tokens.rows == 0 && rows.cols == tokens.cols && pos.cols == rows.rows &&
           rows.device == tokens.device && pos.device == tokens.device && current(tokens.device);
}

// (x, slot_to_pos, xp)
PyObject* moe_permute(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        Operand x, pos, xp;
        if (n != 3 || !operand(args[0], kBf16, 2, x) || !operand(args[1], kI32, 1, pos) || !operand(args[2], kBf16, 2, xp) ||
            !routed_rows(x, xp, pos))
            Py_RETURN_NONE;
        void* s = stream_of(x.device);
        return launch([&] {
            return entries.permute(x.data, (const int32_t*)pos.data, (int)x.rows, (int)(xp.rows / x.rows), (int)x.cols, xp.data, s);
        });
    });
}

// (dxp, slot_to_pos, dx, add or None)
PyObject* moe_permute_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        Operand dxp, pos, dx, add{};
        if (n != 4 || !operand(args[0], kBf16, 2, dxp) || !operand(args[1], kI32, 1, pos) || !operand(args[2], kBf16, 2, dx) ||
            !routed_rows(dx, dxp, pos) ||
            (args[3] != Py_None && (!operand(args[3], kBf16, 2, add) || add.rows != dx.rows || add.cols != dx.cols || add.device != dx.device)))
            Py_RETURN_NONE;
        void* s = stream_of(dx.device);
        return launch([&] {
            return entries.permute_backward(dxp.data, (const int32_t*)pos.data, (int)dx.rows, (int)(dxp.rows / dx.rows), (int)dx.cols,
                                            args[3] != Py_None ? add.data : nullptr, dx.data, s);
        });
    });
}

// (dy, o, weights, slot_to_pos, do, dweights)
PyObject* moe_unpermute_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        Operand dy, o, w, pos, d_o, dw;
        if (n != 6 || !operand(args[0], kBf16, 2, dy) || !operand(args[1], kBf16, 2, o) || !operand(args[2], kF32, 2, w) ||
            !operand(args[3], kI32, 1, pos) || !operand(args[4], kBf16, 2, d_o) || !operand(args[5], kF32, 2, dw) ||
            !routed_rows(dy, o, pos) || d_o.rows != o.rows || d_o.cols != o.cols || w.rows != dy.rows || w.rows * w.cols != o.rows ||
            dw.rows != w.rows || dw.cols != w.cols || w.device != dy.device || d_o.device != dy.device || dw.device != dy.device)
            Py_RETURN_NONE;
        void* s = stream_of(dy.device);
        return launch([&] {
            return entries.unpermute_backward(dy.data, o.data, (const float*)w.data, (const int32_t*)pos.data, (int)dy.rows, (int)w.cols,
                                              (int)dy.cols, d_o.data, (float*)dw.data, s);
        });
    });
}

// rows_n [R, N], rows_k [R, K], w [E, N, K], offsets [E + 1]
bool grouped_shapes(const Operand& rows_n, const Operand& rows_k, const Operand& w, const Operand& offsets) {
    return rows_n.rows == rows_k.rows && rows_n.cols == w.rows && rows_k.cols == w.cols && offsets.cols == w.outer + 1 &&
           rows_k.device == rows_n.device && w.device == rows_n.device && offsets.device == rows_n.device && current(rows_n.device);
}
// (x, w, expert_offsets, y) and (dy, w, expert_offsets, dx)
template <bool DGRAD>
PyObject* grouped(PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        Operand in, w, offsets, out;
        if (n != 4 || !operand(args[0], kBf16, 2, in) || !operand(args[1], kBf16, 3, w) || !operand(args[2], kI32, 1, offsets) ||
            !operand(args[3], kBf16, 2, out) || !grouped_shapes(DGRAD ? in : out, DGRAD ? out : in, w, offsets))
            Py_RETURN_NONE;
        void* s = stream_of(in.device);
        return launch([&] {
            return (DGRAD ? entries.grouped_dgrad : entries.grouped)(in.data, w.data, (const int32_t*)offsets.data, out.data, (int)in.rows,
                                                                     (int)w.outer, (int)w.rows, (int)w.cols, s);
        });
    });
}
PyObject* moe_grouped_gemm(PyObject*, PyObject* const* args, Py_ssize_t n) { return grouped<false>(args, n); }
PyObject* moe_grouped_gemm_dgrad(PyObject*, PyObject* const* args, Py_ssize_t n) { return grouped<true>(args, n); }
// (dy, x, expert_offsets, dw)
PyObject* moe_grouped_gemm_wgrad(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        Operand dy, x, offsets, dw;
        if (n != 4 || !operand(args[0], kBf16, 2, dy) || !operand(args[1], kBf16, 2, x) || !operand(args[2], kI32, 1, offsets)) Py_RETURN_NONE;
        const bool fp32 = operand(args[3], kF32, 3, dw);
        if ((!fp32 && !operand(args[3], kBf16, 3, dw)) || !grouped_shapes(dy, x, dw, offsets)) Py_RETURN_NONE;
        void* s = stream_of(dy.device);
        return launch([&] {
            return entries.grouped_wgrad(dy.data, x.data, (const int32_t*)offsets.data, dw.data, fp32 ? 1 : 0, (int)dy.rows, (int)dw.outer,
                                         (int)dw.rows, (int)dw.cols, s);
        });
    });
}

struct Head {
    Operand x, w, labels, ws;
    int label_type;
};
// x [M, K], w [V, K], labels [M], workspace
bool head(PyObject* x, PyObject* w, PyObject* labels, PyObject* ws, Head& h) {
    if (!operand(x, kBf16, 2, h.x) || !operand(w, kBf16, 2, h.w) || !operand(ws, kByte, 1, h.ws)) return false;
    h.label_type = operand(labels, {at::kLong}, 1, h.labels) ? 1 : 0;
    if (!h.label_type && !operand(labels, kI32, 1, h.labels)) return false;
    return h.w.cols == h.x.cols && h.labels.cols == h.x.rows && h.w.device == h.x.device && h.labels.device == h.x.device &&
           h.ws.device == h.x.device && current(h.x.device);
}
bool head_rows(PyObject* o, const Head& h, Operand& out) {
    return operand(o, kF32, 1, out) && out.cols == h.x.rows && out.device == h.x.device;
}

// (x, w, labels, loss, lse, workspace)
PyObject* linear_cross_entropy(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        Head h;
        Operand loss, lse;
        if (n != 6 || !head(args[0], args[1], args[2], args[5], h) || !head_rows(args[3], h, loss) || !head_rows(args[4], h, lse)) Py_RETURN_NONE;
        void* s = stream_of(h.x.device);
        return launch([&] {
            return entries.head_loss(h.x.data, h.w.data, h.labels.data, h.label_type, (float*)loss.data, (float*)lse.data, (int)h.x.rows,
                                     (int)h.w.rows, (int)h.x.cols, h.ws.data, (size_t)h.ws.cols, s);
        });
    });
}

// (x, w, labels, lse, dloss, dx or None, dw or None, workspace)
PyObject* linear_cross_entropy_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        Head h;
        Operand lse, dloss, dx{}, dw{};
        if (n != 8 || !head(args[0], args[1], args[2], args[7], h) || !head_rows(args[3], h, lse) || !head_rows(args[4], h, dloss) ||
            (args[5] == Py_None && args[6] == Py_None) ||
            (args[5] != Py_None && (!operand(args[5], kBf16, 2, dx) || dx.rows != h.x.rows || dx.cols != h.x.cols || dx.device != h.x.device)))
            Py_RETURN_NONE;
        bool fp32 = false;
        if (args[6] != Py_None) {
            fp32 = operand(args[6], kF32, 2, dw);
            if ((!fp32 && !operand(args[6], kBf16, 2, dw)) || dw.rows != h.w.rows || dw.cols != h.w.cols || dw.device != h.x.device) Py_RETURN_NONE;
        }
        void* s = stream_of(h.x.device);
        return launch([&] {
            return entries.head_gradients(h.x.data, h.w.data, h.labels.data, h.label_type, (const float*)lse.data, (const float*)dloss.data,
                                          args[5] != Py_None ? dx.data : nullptr, args[6] != Py_None ? dw.data : nullptr, fp32 ? 1 : 0,
                                          (int)h.x.rows, (int)h.w.rows, (int)h.x.cols, h.ws.data, (size_t)h.ws.cols, s);
        });
    });
}

struct Gated {
    Operand wide, w, gate_up{}, h{}, offsets{};
    int E, interleaved, act;
    float alpha, limit;
};
// rows [R, wide], w ([E,] .., ..), gate_up [R, 2 I] or None, h [R, I] or None, expert_offsets [E + 1] or None, interleaved, activation, alpha, limit
bool gated(PyObject* wide, PyObject* w, PyObject* gate_up, PyObject* h, PyObject* const* rest, Gated& g) {
    const bool experts = rest[0] != Py_None;
    if (!operand(wide, kBf16, 2, g.wide) || !operand(w, kBf16, experts ? 3 : 2, g.w) || (gate_up != Py_None && !operand(gate_up, kBf16, 2, g.gate_up)) ||
        (h != Py_None && !operand(h, kBf16, 2, g.h)) || (experts && !operand(rest[0], kI32, 1, g.offsets)) || !PyBool_Check(rest[1]) ||
        !PyLong_CheckExact(rest[2]) || !number(rest[3], g.alpha) || !number(rest[4], g.limit))
        return false;
    g.interleaved = rest[1] == Py_True;
    g.act = (int)PyLong_AsLong(rest[2]);
    g.E = (int)g.w.outer;
    for (const Operand* t : {&g.w, &g.gate_up, &g.h, &g.offsets})
        if (t->data && t->device != g.wide.device) return false;
    return (!g.gate_up.data || (g.gate_up.rows == g.wide.rows && g.gate_up.cols % 2 == 0)) && (!g.h.data || g.h.rows == g.wide.rows) &&
           (!experts || g.offsets.cols == g.w.outer + 1) && current(g.wide.device);
}
// (x, w13, h, gate_up or None, expert_offsets or None, interleaved, activation, alpha, limit)
PyObject* gated_gemm(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        Gated g;
        if (n != 9 || args[2] == Py_None || !gated(args[0], args[1], args[3], args[2], args + 4, g) || g.w.cols != g.wide.cols ||
            g.w.rows != 2 * g.h.cols || (g.gate_up.data && g.gate_up.cols != g.w.rows))
            Py_RETURN_NONE;
        void* s = stream_of(g.wide.device);
        return launch([&] {
            return entries.gated(g.wide.data, g.w.data, (const int32_t*)g.offsets.data, g.h.data, g.gate_up.data, (int)g.wide.rows, g.E, (int)g.h.cols,
                                 (int)g.wide.cols, g.interleaved, g.act, g.alpha, g.limit, s);
        });
    });
}
// (dy, w2, gate_up, dgate_up, h or None, expert_offsets or None, interleaved, activation, alpha, limit)
PyObject* gated_gemm_dgrad(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        Gated g;
        Operand d;
        if (n != 10 || args[2] == Py_None || !gated(args[0], args[1], args[2], args[4], args + 5, g) || !operand(args[3], kBf16, 2, d) ||
            g.w.rows != g.wide.cols || g.gate_up.cols != 2 * g.w.cols || (g.h.data && g.h.cols != g.w.cols) || d.rows != g.wide.rows ||
            d.cols != g.gate_up.cols || d.device != g.wide.device)
            Py_RETURN_NONE;
        void* s = stream_of(g.wide.device);
        return launch([&] {
            return entries.gated_dgrad(g.wide.data, g.w.data, (const int32_t*)g.offsets.data, g.gate_up.data, d.data, g.h.data, (int)g.wide.rows, g.E,
                                       (int)g.wide.cols, (int)g.w.cols, g.interleaved, g.act, g.alpha, g.limit, s);
        });
    });
}
// (dy, w, dx)
PyObject* bf16_gemm_dgrad(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        Operand dy, w, dx;
        if (n != 3 || !operand(args[0], kBf16, 2, dy) || !operand(args[1], kBf16, 2, w) || !operand(args[2], kBf16, 2, dx) || w.rows != dy.cols ||
            dx.rows != dy.rows || dx.cols != w.cols || w.device != dy.device || dx.device != dy.device || !current(dy.device))
            Py_RETURN_NONE;
        void* s = stream_of(dy.device);
        return launch([&] { return entries.dense_dgrad(dy.data, w.data, dx.data, (int)dy.rows, (int)dy.cols, (int)w.cols, s); });
    });
}
// (dy, x, dw)
PyObject* bf16_gemm_wgrad(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        Operand dy, x, dw;
        if (n != 3 || !operand(args[0], kBf16, 2, dy) || !operand(args[1], kBf16, 2, x)) Py_RETURN_NONE;
        const bool fp32 = operand(args[2], kF32, 2, dw);
        if ((!fp32 && !operand(args[2], kBf16, 2, dw)) || x.rows != dy.rows || dw.rows != dy.cols || dw.cols != x.cols || x.device != dy.device ||
            dw.device != dy.device || !current(dy.device))
            Py_RETURN_NONE;
        void* s = stream_of(dy.device);
        return launch([&] { return entries.dense_wgrad(dy.data, x.data, dw.data, fp32 ? 1 : 0, (int)dy.rows, (int)dy.cols, (int)x.cols, s); });
    });
}

struct Embedding {
    Operand ids, rows, table;
    int id_type, table_type;
    float scale;
};
// ids [T], rows [T, H], table [V, H]
bool embedding_operands(PyObject* ids, PyObject* rows, PyObject* table, PyObject* scale, Embedding& e) {
    e.id_type = operand(ids, {at::kLong}, 1, e.ids) ? 1 : 0;
    if (!e.id_type && !operand(ids, kI32, 1, e.ids)) return false;
    e.table_type = operand(table, kF32, 2, e.table) ? 1 : 0;
    if ((!e.table_type && !operand(table, kBf16, 2, e.table)) || !operand(rows, kBf16, 2, e.rows) || !number(scale, e.scale)) return false;
    return e.rows.rows == e.ids.cols && e.rows.cols == e.table.cols && e.rows.device == e.ids.device && e.table.device == e.ids.device &&
           current(e.ids.device);
}
// (ids, table, out, scale)
PyObject* embedding(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        Embedding e;
        if (n != 4 || !embedding_operands(args[0], args[2], args[1], args[3], e)) Py_RETURN_NONE;
        void* s = stream_of(e.ids.device);
        return launch([&] {
            return entries.embedding(e.ids.data, e.id_type, e.table.data, e.table_type, e.rows.data, (int)e.rows.rows, (int)e.table.rows,
                                     (int)e.table.cols, e.scale, s);
        });
    });
}
// (ids, dout, dtable, workspace, scale, add or None)
PyObject* embedding_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        Embedding e;
        Operand ws, add{};
        if (n != 6 || !embedding_operands(args[0], args[1], args[2], args[4], e) || !operand(args[3], kByte, 1, ws) || ws.device != e.ids.device ||
            (args[5] != Py_None && ((e.table_type ? !operand(args[5], kF32, 2, add) : !operand(args[5], kBf16, 2, add)) || add.rows != e.table.rows ||
                                    add.cols != e.table.cols || add.device != e.ids.device)))
            Py_RETURN_NONE;
        void* s = stream_of(e.ids.device);
        return launch([&] {
            return entries.embedding_backward(e.ids.data, e.id_type, e.rows.data, add.data, e.table.data, e.table_type, (int)e.rows.rows,
                                              (int)e.table.rows, (int)e.table.cols, e.scale, ws.data, (size_t)ws.cols, s);
        });
    });
}

struct GradList {
    Operand list, norm;
    int n;
    int64_t chunks;
};
// a GradTensors' list, n and chunks, and norm [1]
bool grad_list(PyObject* const* args, PyObject* norm, GradList& g) {
    if (!operand(args[0], kByte, 1, g.list) || !PyLong_CheckExact(args[1]) || !PyLong_CheckExact(args[2]) || !operand(norm, kF32, 1, g.norm)) return false;
    g.n = (int)PyLong_AsLong(args[1]);
    g.chunks = PyLong_AsLongLong(args[2]);
    return g.norm.cols == 1 && g.norm.device == g.list.device && current(g.list.device);
}
// (list, n, chunks, norm, workspace)
PyObject* grad_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        GradList g;
        Operand ws;
        if (n != 5 || !grad_list(args, args[3], g) || !operand(args[4], kByte, 1, ws) || ws.device != g.list.device) Py_RETURN_NONE;
        void* s = stream_of(g.list.device);
        return launch([&] { return entries.grad_norm(g.list.data, g.n, g.chunks, (float*)g.norm.data, ws.data, (size_t)ws.cols, s); });
    });
}
// (list, n, chunks, norm, max_norm)
PyObject* grad_clip(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        GradList g;
        float max_norm;
        if (n != 5 || !grad_list(args, args[3], g) || !number(args[4], max_norm)) Py_RETURN_NONE;
        void* s = stream_of(g.list.device);
        return launch([&] { return entries.grad_clip(g.list.data, g.n, g.chunks, (const float*)g.norm.data, max_norm, s); });
    });
}

// The library's functions by address, in the order of Entries.
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
    constexpr int kCount = sizeof(Entries) / sizeof(void*);
    void* p[kCount];
    if (n != kCount) return PyErr_Format(PyExc_TypeError, "bind: %d addresses", kCount);
    for (int i = 0; i < kCount; ++i) {
        p[i] = PyLong_AsVoidPtr(args[i]);
        if (!p[i]) return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_ValueError, "bind: null address");
    }
    static_assert(sizeof(Entries) == sizeof(p));
    std::memcpy(&entries, p, sizeof(p));
    Py_RETURN_NONE;
}

#define HK_METHOD(NAME) {#NAME, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(NAME)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {HK_METHOD(bind), HK_METHOD(fp8_gemm), HK_METHOD(bf16_gemm), HK_METHOD(mxfp4_gemm),
                         HK_METHOD(mxfp4_quantize_rows), HK_METHOD(moe_permute), HK_METHOD(moe_permute_backward),
                         HK_METHOD(moe_unpermute_backward), HK_METHOD(moe_grouped_gemm), HK_METHOD(moe_grouped_gemm_dgrad),
                         HK_METHOD(moe_grouped_gemm_wgrad), HK_METHOD(linear_cross_entropy),
                         HK_METHOD(linear_cross_entropy_backward), HK_METHOD(gated_gemm), HK_METHOD(gated_gemm_dgrad),
                         HK_METHOD(bf16_gemm_dgrad), HK_METHOD(bf16_gemm_wgrad), HK_METHOD(embedding), HK_METHOD(embedding_backward),
                         HK_METHOD(grad_norm), HK_METHOD(grad_clip), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_dispatch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__dispatch(void) {
    PyObject* nn = PyImport_ImportModule("torch.nn");
    if (!nn) return nullptr;
    PyObject* parameter = PyObject_GetAttrString(nn, "Parameter");
    Py_DECREF(nn);
    if (!parameter) return nullptr;
    parameter_type = reinterpret_cast<PyTypeObject*>(parameter);   // (kept for the life of the process)
    PyObject* module = PyModule_Create(&module_def);
    if (module && PyModule_AddStringConstant(module, "build_tag", HK_BUILD_TAG) < 0) Py_CLEAR(module);
    return module;
}
