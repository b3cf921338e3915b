// The calls a decode step makes most — quantise the activations, multiply them with packed weights — without the Python around
// them: argument checks, output allocation and the launch through the C ABI in one native function each.  What bounds the
// smallest calls is the host: one token through a quantiser and a 4096 -> 12288 linear is 14 us of GPU work; through the Python of
// flh_b200/_CUDA.py (checks, views, torch.empty, ctypes) it takes 35 us, so 17 (16 tokens through 11008 -> 4096: 42 and 21).
//
// Every function takes the plain case only and returns None for anything else — another type, layout or device than the
// current one, a tensor subclass, a transform, mode or trace that has to see the operations — and the caller then goes the
// way in Python, which has the error messages and the general shapes.  Nothing is kept between calls.
//
// Allocations and launches run without the interpreter's lock: an allocation may free blocks and synchronise, and a launch waits
// while the stream's queue is full, for as long as the GPU takes; other Python threads run meanwhile, among them the one that
// what is queued may be waiting for.
#include <Python.h>
#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <cmath>

#include "../../include/flh_b200.h"

namespace {

// operations that something other than this process's kernels has to see
bool observed() {
    return at::impl::torch_function_mode_enabled() || c10::impl::TorchDispatchModeTLS::any_modes_set() || torch::jit::tracer::isTracing();
}
// a contiguous (or, with `strides`, any strided) CUDA tensor on `device` (the current one, which is asked for only once a tensor is known to be a CUDA tensor: there may
// be no driver) with memory of its own kind and nothing wrapped around it
bool plain(const at::Tensor &t, c10::DeviceIndex device, bool strides = false) {
    if (!t.is_cuda() || t.device().index() != device || t.layout() != at::kStrided || (!strides && !t.is_contiguous()) || t.is_neg() || t.is_conj()) return false;
    const c10::DispatchKeySet ks = t.key_set();
    return !ks.has_any(c10::DispatchKeySet({c10::DispatchKey::Python, c10::DispatchKey::Functionalize, c10::DispatchKey::FuncTorchBatched,
                                            c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Batched, c10::DispatchKey::ZeroTensor}));
}
const at::Tensor *tensor(PyObject *o) { return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }

// the interpreter's lock given up for a scope, taken back also where an exception leaves it
struct Unlocked {
    PyThreadState *state = PyEval_SaveThread();
    Unlocked() = default;
    Unlocked(const Unlocked &) = delete;
    ~Unlocked() { PyEval_RestoreThread(state); }
};

PyObject *failed(const char *what, int rc) {
    PyErr_Format(PyExc_RuntimeError, "%s failed (status %d): %s", what, rc, flh_b200_last_error());
    return nullptr;
}
at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor &like) {
    return at::empty(sizes, at::TensorOptions().dtype(type).device(like.device()));
}
// the sizes of x with the last one replaced
c10::SmallVector<int64_t, 6> with_last(const at::Tensor &x, int64_t last) {
    c10::SmallVector<int64_t, 6> s(x.sizes().begin(), x.sizes().end());
    s.back() = last;
    return s;
}

// act_quant_group(x, group_size, hadamard) -> (q, scale)
PyObject *act_quant_group(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const at::Tensor *x = n == 3 ? tensor(args[0]) : nullptr;
    const long gs = x ? PyLong_AsLong(args[1]) : 0;
    const int had = x ? PyObject_IsTrue(args[2]) : 0;
    if (PyErr_Occurred()) { PyErr_Clear(); Py_RETURN_NONE; }
    if (!x || !x->is_cuda() || observed() || (gs != 32 && gs != 64 && gs != 128) || x->dim() < 1 || x->scalar_type() != at::kHalf) Py_RETURN_NONE;
    const c10::DeviceIndex dev = c10::cuda::current_device();
    const int64_t K = x->size(-1);
    if (!plain(*x, dev) || x->numel() == 0 || K % gs) Py_RETURN_NONE;
    const at::Tensor in = *x;
    const void *in_p = in.data_ptr();
    at::Tensor q, s;
    int rc;
    // torch divides a CUDA tensor by a number by multiplying with the number's reciprocal, rounded to binary32
    const float factor = had ? 1.0f / (float)std::sqrt((double)gs) : 1.0f;
    {
        const Unlocked unlocked;
        q = empty(with_last(in, K / 2), at::kByte, in);
        s = empty(with_last(in, K / gs), at::kHalf, in);
        rc = flh_b200_quant_group_sym_scaled_i4(in_p, in.numel() / gs, (int)gs, had, factor, static_cast<uint8_t *>(q.data_ptr()), s.data_ptr(),
                                                c10::cuda::getCurrentCUDAStream(dev).stream());
    }
    if (rc) return failed("quant_group_sym_i4", rc);
    return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(q)), THPVariable_Wrap(std::move(s)));
    END_HANDLE_TH_ERRORS
}

// act_quant_token(x, hadamard, clip, kfac, sign table or None) -> (q, scale, zero)
PyObject *act_quant_token(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const at::Tensor *x = n == 5 ? tensor(args[0]) : nullptr;
    const at::Tensor *bits = x ? tensor(args[4]) : nullptr;
    const int had = x ? PyObject_IsTrue(args[1]) : 0;
    const double clip = x ? PyFloat_AsDouble(args[2]) : 0;
    const long kfac = x ? PyLong_AsLong(args[3]) : 0;
    if (PyErr_Occurred()) { PyErr_Clear(); Py_RETURN_NONE; }
    if (!x || !x->is_cuda() || (!bits && args[4] != Py_None) || observed() || x->dim() < 1) Py_RETURN_NONE;
    if (x->scalar_type() != at::kHalf && x->scalar_type() != at::kBFloat16) Py_RETURN_NONE;
    const c10::DeviceIndex dev = c10::cuda::current_device();
    if (!plain(*x, dev) || x->numel() == 0) Py_RETURN_NONE;
    const at::Tensor in = *x, table = bits ? *bits : at::Tensor();
    const void *in_p = in.data_ptr();
    const uint32_t *table_p = bits ? static_cast<const uint32_t *>(table.data_ptr()) : nullptr;
    const int64_t K = in.size(-1);
    at::Tensor q, s, z;
    int rc;
    {
        const Unlocked unlocked;
        const auto one = with_last(in, 1);
        q = empty(with_last(in, K / 2), at::kByte, in);
        s = empty(one, at::kHalf, in);
        z = empty(one, at::kHalf, in);
        rc = flh_b200_quant_token_asym_i4(in_p, in.scalar_type() == at::kBFloat16 ? FLH_B200_BF16 : FLH_B200_F16, in.numel() / K, K, K, had ? 1 : 0,
                                          (int)kfac, table_p, (float)clip, static_cast<uint8_t *>(q.data_ptr()), s.data_ptr(), z.data_ptr(),
                                          c10::cuda::getCurrentCUDAStream(dev).stream());
    }
    if (rc) return failed("quant_token_asym_i4", rc);
    return Py_BuildValue("(NNN)", THPVariable_Wrap(std::move(q)), THPVariable_Wrap(std::move(s)), THPVariable_Wrap(std::move(z)));
    END_HANDLE_TH_ERRORS
}

// gemm(x, w, a_scale, a_zero, w_scale, rowsum, bias, bfloat16, algo, workspace) -> y: algo and workspace as the plan of
// flh_b200/_CUDA.py names them, the workspace a tensor, the bytes of scratch that this call alone uses, or None.
// x [.., K / 2], w flat or [N, K / 2].
PyObject *gemm(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 10) Py_RETURN_NONE;
    const at::Tensor *t[7];
    for (int i = 0; i < 7; ++i) {
        t[i] = tensor(args[i]);
        if (!t[i] && (args[i] != Py_None || i < 3 || i == 4)) Py_RETURN_NONE;
    }
    const at::Tensor *ws = tensor(args[9]);
    const long scratch = PyLong_Check(args[9]) ? PyLong_AsLong(args[9]) : 0;
    const int bf16 = PyObject_IsTrue(args[7]);
    const long algo = PyLong_AsLong(args[8]);
    if (PyErr_Occurred()) { PyErr_Clear(); Py_RETURN_NONE; }
    if ((!ws && !PyLong_Check(args[9]) && args[9] != Py_None) || observed()) Py_RETURN_NONE;
    const at::Tensor &x = *t[0], &w = *t[1], &sa = *t[2], &sb = *t[4];
    if (!x.is_cuda()) Py_RETURN_NONE;
    const c10::DeviceIndex dev = c10::cuda::current_device();
    for (int i = 0; i < 7; ++i)
        if (t[i] && !plain(*t[i], dev)) Py_RETURN_NONE;
    if (x.dim() < 1 || sb.dim() != 2 || x.numel() == 0 || sb.numel() == 0) Py_RETURN_NONE;
    const int64_t K = 2 * x.size(-1), M = x.numel() / x.size(-1), N = sb.size(0);
    if (sa.numel() == 0 || sa.numel() % M || w.numel() != N * (K / 2)) Py_RETURN_NONE;
    const int64_t ga = sa.numel() / M, gb = sb.size(1);
    if (K % ga || K % gb || x.scalar_type() != at::kByte || w.scalar_type() != at::kByte || sa.scalar_type() != at::kHalf ||
        sb.scalar_type() != at::kHalf || (t[3] && (t[3]->scalar_type() != at::kHalf || t[3]->numel() != sa.numel())) ||
        (t[5] && t[5]->scalar_type() != at::kInt) || (t[6] && (t[6]->scalar_type() != at::kHalf || t[6]->numel() != N)))
        Py_RETURN_NONE;
    at::Tensor held[8], y, own;                                  // the operands and the workspace stay alive while the lock is given up
    void *ptr[8] = {};
    for (int i = 0; i < 7; ++i)
        if (t[i]) { held[i] = *t[i]; ptr[i] = t[i]->data_ptr(); }
    size_t ws_bytes = 0;
    if (ws) { held[7] = *ws; ptr[7] = ws->data_ptr(); ws_bytes = (size_t)ws->numel(); }
    int rc;
    bool fits = true;
    {
        const Unlocked unlocked;
        y = empty(with_last(held[0], N), bf16 ? at::kBFloat16 : at::kHalf, held[0]);
        if (scratch > 0) {
            try {
                own = empty({(int64_t)scratch}, at::kByte, held[0]);     // freed in stream order when the call returns
                ptr[7] = own.data_ptr();
                ws_bytes = (size_t)scratch;
            } catch (const c10::OutOfMemoryError &) {
                fits = false;                                    // AUTO has a kernel that needs none
            }
        }
        rc = !fits ? 0 : flh_b200_gemm_i4_dequant(
            static_cast<const uint8_t *>(ptr[0]), static_cast<const uint8_t *>(ptr[1]), ptr[2], ptr[3], ptr[4], static_cast<const int32_t *>(ptr[5]),
            ptr[6], y.data_ptr(), M, N, K, K / ga, K / gb, bf16 ? FLH_B200_BF16 : FLH_B200_F16, (int)algo, ptr[7], ws_bytes,
            c10::cuda::getCurrentCUDAStream(dev).stream());
    }
    if (!fits) Py_RETURN_NONE;
    if (rc) return failed("gemm_i4_dequant", rc);
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// square(x) -> x * x in binary32, for values that no derivative is taken of
PyObject *square(PyObject *, PyObject *x_) {
    HANDLE_TH_ERRORS
    const at::Tensor *x = tensor(x_);
    if (!x || !x->is_cuda() || observed() || (x->scalar_type() != at::kHalf && x->scalar_type() != at::kBFloat16)) Py_RETURN_NONE;
    const c10::DeviceIndex dev = c10::cuda::current_device();
    if (!plain(*x, dev) || x->numel() % 8 || reinterpret_cast<uintptr_t>(x->data_ptr()) % 16) Py_RETURN_NONE;
    if ((c10::GradMode::is_enabled() && x->requires_grad()) || x->_fw_grad(0).defined()) Py_RETURN_NONE;
    const at::Tensor in = *x;
    const void *in_p = in.data_ptr();
    at::Tensor y;
    int rc;
    {
        const Unlocked unlocked;
        y = empty(in.sizes(), at::kFloat, in);
        rc = flh_b200_square_f32(in_p, in.scalar_type() == at::kBFloat16 ? FLH_B200_BF16 : FLH_B200_F16, in.numel(), y.data_ptr(),
                                 c10::cuda::getCurrentCUDAStream(dev).stream());
    }
    if (rc) return failed("square_f32", rc);
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// ---- a KV cache that is drafted into and evicted from -----------------------------------------
bool is_cache(const at::Tensor &t) { return t.dim() == 4 && (t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16); }
int dtype_of(const at::Tensor &t) { return t.scalar_type() == at::kBFloat16 ? FLH_B200_BF16 : FLH_B200_F16; }
bool ints(const at::Tensor &t, at::IntArrayRef sizes) { return t.scalar_type() == at::kInt && t.sizes() == sizes; }

// tree_attention(q, k, v, lengths, tree or None, weights or None, scale or None, counted or None) -> out
PyObject *tree_attention(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 8) Py_RETURN_NONE;
    const at::Tensor *t[7];
    for (int i = 0; i < 7; ++i) {
        PyObject *arg = args[i < 6 ? i : 7];
        t[i] = tensor(arg);
        if (!t[i] && (arg != Py_None || i < 4)) Py_RETURN_NONE;
    }
    const double given = args[6] == Py_None ? 0 : PyFloat_AsDouble(args[6]);
    if (PyErr_Occurred()) { PyErr_Clear(); Py_RETURN_NONE; }
    const at::Tensor &q = *t[0], &k = *t[1], &v = *t[2];
    if (!q.is_cuda() || observed() || q.dim() != 4 || !is_cache(k) || v.sizes() != k.sizes() || v.scalar_type() != k.scalar_type() || q.scalar_type() != k.scalar_type()) Py_RETURN_NONE;
    const c10::DeviceIndex dev = c10::cuda::current_device();
    for (int i = 0; i < 7; ++i)
        if (t[i] && !plain(*t[i], dev, i == 0)) Py_RETURN_NONE;
    const int64_t B = k.size(0), nkv = k.size(1), T = k.size(2), D = k.size(3), S = q.size(1), nh = q.size(2);
    if (q.size(0) != B || q.size(3) != D || B == 0 || S == 0 || S > FLH_B200_TREE_MAX_TOKENS || nkv == 0 || nh == 0 || nh % nkv || T == 0 || q.stride(3) != 1 || !ints(*t[3], {B}) ||
        B * nh * S >= 1L << 31)
        Py_RETURN_NONE;
    long st[3];
    for (int i = 0; i < 3; ++i) {
        st[i] = q.size(i) > 1 ? q.stride(i) : 0;
        if (st[i] % 8) Py_RETURN_NONE;
    }
    if (t[4] && (t[4]->scalar_type() != at::kLong || (t[4]->sizes() != at::IntArrayRef({S}) && t[4]->sizes() != at::IntArrayRef({B, S})))) Py_RETURN_NONE;
    if (t[5] && (t[5]->scalar_type() != at::kFloat || t[5]->sizes() != at::IntArrayRef({B, nkv, T}))) Py_RETURN_NONE;
    if (t[6] && (!t[5] || !ints(*t[6], {B}))) Py_RETURN_NONE;
    const float scale = args[6] == Py_None ? (float)(1.0 / std::sqrt((double)D)) : (float)given;
    const long tree_stride = t[4] && t[4]->dim() == 2 ? S : 0;
    at::Tensor held[7], out, ws;
    void *ptr[7] = {};
    for (int i = 0; i < 7; ++i)
        if (t[i]) { held[i] = *t[i]; ptr[i] = t[i]->data_ptr(); }
    const size_t need = flh_b200_tree_attention_workspace_bytes((int)B, (int)S, (int)nh, (int)nkv, (int)D, T, ptr[5] != nullptr);
    if (!need) Py_RETURN_NONE;
    int rc;
    {
        const Unlocked unlocked;
        out = empty({B, S, nh, D}, held[0].scalar_type(), held[0]);
        ws = empty({(int64_t)need}, at::kByte, held[0]);                // of this call alone, freed in stream order when it returns
        rc = flh_b200_tree_attention_counted(ptr[0], st[0], st[1], st[2], dtype_of(held[0]), ptr[1], ptr[2], static_cast<const int32_t *>(ptr[3]), static_cast<const int64_t *>(ptr[4]),
                                     tree_stride, scale, out.data_ptr(), static_cast<float *>(ptr[5]), static_cast<const int32_t *>(ptr[6]), (int)B, (int)S, (int)nh, (int)nkv, (int)D, T, ws.data_ptr(), need,
                                     c10::cuda::getCurrentCUDAStream(dev).stream());
    }
    if (rc) return failed("tree_attention", rc);
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// rope_kv_at(qkv, cos, sin, positions, lengths, k_cache, v_cache, nh) -> q
PyObject *rope_kv_at(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 8) Py_RETURN_NONE;
    const at::Tensor *t[7];
    for (int i = 0; i < 7; ++i)
        if (!(t[i] = tensor(args[i]))) Py_RETURN_NONE;
    const long nh = PyLong_AsLong(args[7]);
    if (PyErr_Occurred()) { PyErr_Clear(); Py_RETURN_NONE; }
    const at::Tensor &qkv = *t[0], &cos = *t[1], &sin = *t[2], &pos = *t[3], &k = *t[5], &v = *t[6];
    if (!qkv.is_cuda() || observed() || !is_cache(k) || v.sizes() != k.sizes() || v.scalar_type() != k.scalar_type() || qkv.scalar_type() != k.scalar_type()) Py_RETURN_NONE;
    const c10::DeviceIndex dev = c10::cuda::current_device();
    for (int i = 0; i < 7; ++i)
        if (!plain(*t[i], dev)) Py_RETURN_NONE;
    const int64_t B = k.size(0), nkv = k.size(1), T = k.size(2), D = k.size(3);
    if (pos.dim() != 2 || B == 0 || nh <= 0 || nh >= 1L << 24) Py_RETURN_NONE;
    const int64_t S = pos.size(1);
    if (S == 0 || !ints(pos, {B, S}) || !ints(*t[4], {B}) || qkv.sizes() != at::IntArrayRef({B * S, (nh + 2 * nkv) * D}) || cos.scalar_type() != at::kFloat ||
        sin.scalar_type() != at::kFloat || cos.dim() != 2 || cos.size(1) * 2 != D || sin.sizes() != cos.sizes())
        Py_RETURN_NONE;
    at::Tensor held[7], q;
    void *ptr[7];
    for (int i = 0; i < 7; ++i) { held[i] = *t[i]; ptr[i] = t[i]->data_ptr(); }
    const long P = cos.size(0);
    int rc;
    {
        const Unlocked unlocked;
        q = empty({B, S, nh, D}, held[0].scalar_type(), held[0]);
        rc = flh_b200_rope_kv_at(ptr[0], dtype_of(held[0]), static_cast<const float *>(ptr[1]), static_cast<const float *>(ptr[2]), P, static_cast<const int32_t *>(ptr[3]),
                                 static_cast<const int32_t *>(ptr[4]), q.data_ptr(), ptr[5], ptr[6], (int)B, (int)S, (int)nh, (int)nkv, (int)D, T,
                                 c10::cuda::getCurrentCUDAStream(dev).stream());
    }
    if (rc) return failed("rope_kv_at", rc);
    return THPVariable_Wrap(std::move(q));
    END_HANDLE_TH_ERRORS
}

// The caches of all layers: lists of plain tensors that are alike, weights a list or None.  Up to 384 tensors: what makes the first of a
// list plain is compared with the others' (their dispatch keys, types, devices and sizes are the same), 70 -> 25 ns each; references
// are taken to copies of the lists.
struct Layers {
    PyObject *kept[3] = {};
    void *ptr[3][FLH_B200_CACHE_MAX_LAYERS];
    at::Tensor first;
    int layers = 0;
    bool weights = false;
    Layers() = default;
    Layers(const Layers &) = delete;
    ~Layers() { for (PyObject *o : kept) Py_XDECREF(o); }
    bool take(PyObject *k, PyObject *v, PyObject *w, c10::DeviceIndex dev) {
        PyObject *lists[3] = {k, v, w};
        weights = w != Py_None;
        for (int i = 0; i < (weights ? 3 : 2); ++i) {
            if (!PyList_CheckExact(lists[i])) return false;
            if (!(kept[i] = PyList_AsTuple(lists[i]))) { PyErr_Clear(); return false; }
            const Py_ssize_t n = PyTuple_GET_SIZE(kept[i]);
            if (i == 0) {
                if (n < 1 || n > FLH_B200_CACHE_MAX_LAYERS) return false;
                layers = (int)n;
            }
            if (n != layers) return false;
            const at::Tensor *head = tensor(PyTuple_GET_ITEM(kept[i], 0));
            if (!head || !plain(*head, dev)) return false;
            if (i == 0) {
                if (!is_cache(*head)) return false;
                first = *head;
            }
            if (i < 2 ? head->sizes() != first.sizes() || head->scalar_type() != first.scalar_type() : head->scalar_type() != at::kFloat || head->sizes() != first.sizes().slice(0, 3))
                return false;
            const c10::TensorImpl *h = head->unsafeGetTensorImpl();
            const c10::DispatchKeySet keys = h->key_set();
            for (int j = 0; j < layers; ++j) {
                const at::Tensor *t = tensor(PyTuple_GET_ITEM(kept[i], j));
                if (!t) return false;
                const c10::TensorImpl *o = t->unsafeGetTensorImpl();
                if (j && (!(o->key_set() == keys) || o->dtype() != h->dtype() || o->device() != h->device() || o->sizes() != h->sizes() || !o->is_contiguous())) return false;
                ptr[i][j] = t->data_ptr();
            }
        }
        return true;
    }
};

// cache_accept(k list, v list, weights list or None, lengths, path, accepted, drafted) -> now
PyObject *cache_accept(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 7) Py_RETURN_NONE;
    const at::Tensor *t[3];
    for (int i = 0; i < 3; ++i)
        if (!(t[i] = tensor(args[3 + i])) || !t[i]->is_cuda()) Py_RETURN_NONE;
    const long drafted = PyLong_AsLong(args[6]);
    if (PyErr_Occurred()) { PyErr_Clear(); Py_RETURN_NONE; }
    if (observed() || drafted < 1 || drafted > FLH_B200_TREE_MAX_TOKENS) Py_RETURN_NONE;
    const c10::DeviceIndex dev = c10::cuda::current_device();
    Layers c;
    if (!plain(*t[0], dev) || !plain(*t[1], dev) || !plain(*t[2], dev) || !c.take(args[0], args[1], args[2], dev)) Py_RETURN_NONE;
    const at::Tensor lengths = *t[0], path = *t[1], accepted = *t[2], &k = c.first;
    const int64_t B = k.size(0), nkv = k.size(1), T = k.size(2), D = k.size(3);
    if (B == 0 || path.dim() != 2 || path.size(1) > drafted || !ints(lengths, {B}) || !ints(path, {B, path.size(1)}) || !ints(accepted, {B})) Py_RETURN_NONE;
    void *len_p = lengths.data_ptr(), *path_p = path.data_ptr(), *acc_p = accepted.data_ptr();
    at::Tensor now;
    int rc;
    {
        const Unlocked unlocked;
        now = empty({B}, at::kInt, lengths);
        rc = flh_b200_cache_accept(c.ptr[0], c.ptr[1], c.weights ? reinterpret_cast<float *const *>(c.ptr[2]) : nullptr, c.layers, dtype_of(k), static_cast<const int32_t *>(len_p),
                                   static_cast<const int32_t *>(path_p), static_cast<const int32_t *>(acc_p), static_cast<int32_t *>(now.data_ptr()), (int)B, (int)nkv, (int)D,
                                   T, (int)path.size(1), (int)drafted, c10::cuda::getCurrentCUDAStream(dev).stream());
    }
    if (rc) return failed("cache_accept", rc);
    return THPVariable_Wrap(std::move(now));
    END_HANDLE_TH_ERRORS
}

// cache_evict(k list, v list, weights list, lengths, keep, recent) -> (kept, left, now)
PyObject *cache_evict(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 6) Py_RETURN_NONE;
    const at::Tensor *len = tensor(args[3]);
    if (!len || !len->is_cuda()) Py_RETURN_NONE;
    const long keep = PyLong_AsLong(args[4]), recent = PyLong_AsLong(args[5]);
    if (PyErr_Occurred()) { PyErr_Clear(); Py_RETURN_NONE; }
    if (observed() || args[2] == Py_None) Py_RETURN_NONE;
    const c10::DeviceIndex dev = c10::cuda::current_device();
    Layers c;
    if (!plain(*len, dev) || !c.take(args[0], args[1], args[2], dev)) Py_RETURN_NONE;
    const at::Tensor lengths = *len, &k = c.first;
    const int64_t B = k.size(0), nkv = k.size(1), T = k.size(2), D = k.size(3);
    if (B == 0 || !ints(lengths, {B}) || keep < 1 || keep > T || recent < 0 || recent > keep) Py_RETURN_NONE;
    void *len_p = lengths.data_ptr();
    at::Tensor kept, left, now;
    int rc;
    {
        const Unlocked unlocked;
        kept = empty({c.layers, B, nkv, keep}, at::kInt, lengths);
        left = empty({c.layers, B, nkv, T}, at::kFloat, lengths);
        now = empty({B}, at::kInt, lengths);
        rc = flh_b200_cache_evict(c.ptr[0], c.ptr[1], reinterpret_cast<const float *const *>(c.ptr[2]), c.layers, dtype_of(k), static_cast<const int32_t *>(len_p), (int)keep,
                                  (int)recent, static_cast<int32_t *>(kept.data_ptr()), static_cast<float *>(left.data_ptr()), static_cast<int32_t *>(now.data_ptr()), (int)B,
                                  (int)nkv, (int)D, T, c10::cuda::getCurrentCUDAStream(dev).stream());
    }
    if (rc) return failed("cache_evict", rc);
    return Py_BuildValue("(NNN)", THPVariable_Wrap(std::move(kept)), THPVariable_Wrap(std::move(left)), THPVariable_Wrap(std::move(now)));
    END_HANDLE_TH_ERRORS
}

#define FASTCALL(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {
    FASTCALL(tree_attention), FASTCALL(rope_kv_at), FASTCALL(cache_accept), FASTCALL(cache_evict),
    {"square", square, METH_O, nullptr},
    {"act_quant_group", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(act_quant_group)), METH_FASTCALL, nullptr},
    {"act_quant_token", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(act_quant_token)), METH_FASTCALL, nullptr},
    {"gemm", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(gemm)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// torch_version: what the tensors' layout was compiled against; flh_b200/_CUDA.py uses the module under that version only
PyMODINIT_FUNC PyInit__host(void) {
    PyObject *m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "torch_version", FLH_TORCH) < 0) { Py_DECREF(m); return nullptr; }
    return m;
}
