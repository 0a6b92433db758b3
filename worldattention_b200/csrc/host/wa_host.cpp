// Native host side of the per-forward entry points.
//
// An HSA forward is three or four launches of 5..100 us, and a layer makes half a dozen such calls: with the checks,
// the descriptors and the workspace look-up done in Python through ctypes a call took 60..80 us to enqueue, more than
// the small shapes take to run.  Here a call is one C function: it reads the tensors' sizes and strides itself, takes
// its output from PyTorch's caching allocator, keeps the workspace of each stream, and calls the C ABI of libwa_b200.so.
// The functions of that library are handed over by address (`bind`), so this module does not care which file they
// come from.
#include <torch/extension.h>

#include <ATen/core/CachingHostAllocator.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <list>
#include <string>
#include <unordered_map>
#include <unordered_set>
#include <vector>

#include "../../../include/worldattention_b200.h"

namespace {

using at::Tensor;

// ---- the C ABI, by address ---------------------------------------------------------------------
decltype(&wa_last_error) f_last_error;
decltype(&wa_hsa_workspace_bytes) f_workspace_bytes;
decltype(&wa_hsa_forward) f_forward;
decltype(&wa_hsa_status) f_status;
decltype(&wa_qk_norm_rope) f_rope;
decltype(&wa_qk_norm_rope_at) f_rope_at;
decltype(&wa_kv_append_workspace_bytes) f_append_bytes;
decltype(&wa_kv_append_compress) f_append;
decltype(&wa_ln_modulate) f_ln;
decltype(&wa_gated_residual) f_residual;
decltype(&wa_axial_rope) f_axial;
decltype(&wa_hkv_move_pages) f_move_pages;
decltype(&wa_selected_workspace_bytes) f_selected_bytes;
decltype(&wa_selected_forward) f_selected_forward;
decltype(&wa_selected_backward) f_selected_backward;
PyObject *py_out_of_memory = nullptr;                                 // torch.OutOfMemoryError
PyObject *py_status_word = nullptr, *py_raise_if_failed = nullptr;   // _lib.status_word(index) -> address, _lib.raise_if_failed(index)

constexpr int MAX_DEVICES = 64;
volatile int *status_words[MAX_DEVICES] = {nullptr};

struct PyFailure {};   // a Python exception is set

[[noreturn]] void fail(PyObject *type, const std::string &msg) {
    if (PyGILState_Check()) {
        PyErr_SetString(type, msg.c_str());
    } else {                                // a thread of the autograd engine (its Python thread state outlives this scope)
        pybind11::gil_scoped_acquire gil;
        PyErr_SetString(type, msg.c_str());
    }
    throw PyFailure();
}

void check(int rc) {
    if (rc == 0) return;
    const std::string msg = f_last_error();
    if (rc == WA_ERR_ARG || rc == WA_ERR_ALIGN || rc == WA_ERR_WORKSPACE) fail(PyExc_ValueError, msg);
    if (rc == WA_ERR_UNSUPPORTED) fail(PyExc_NotImplementedError, msg);
    fail(PyExc_RuntimeError, "CUDA error " + std::to_string(rc) + ": " + msg);
}

// ---- arguments ---------------------------------------------------------------------------------
const Tensor *tensor_or_null(PyObject *o, const char *name) {
    if (o == Py_None) return nullptr;
    if (!THPVariable_Check(o)) fail(PyExc_TypeError, std::string(name) + " must be a tensor");
    return &THPVariable_Unpack(o);
}
const Tensor &tensor(PyObject *o, const char *name) {
    const Tensor *t = tensor_or_null(o, name);
    if (!t) fail(PyExc_TypeError, std::string(name) + " must be a tensor");
    return *t;
}
long long integer(PyObject *o) {
    if (!PyLong_Check(o)) {
        PyObject *as_int = PyNumber_Long(o);
        if (!as_int) throw PyFailure();
        const long long v = PyLong_AsLongLong(as_int);
        Py_DECREF(as_int);
        if (v == -1 && PyErr_Occurred()) throw PyFailure();
        return v;
    }
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw PyFailure();
    return v;
}
double real(PyObject *o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw PyFailure();
    return v;
}
void expect_args(Py_ssize_t got, Py_ssize_t want) {
    if (got != want) fail(PyExc_TypeError, "expected " + std::to_string(want) + " arguments, got " + std::to_string(got));
}

std::string shape_of(const Tensor &t) {
    std::string s = "(";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + (t.dim() == 1 ? ",)" : ")");
}

void require_cuda(const Tensor &t, c10::Device &dev, bool &seen) {
    if (!t.is_cuda())
        fail(PyExc_RuntimeError, "worldattention_b200 runs on CUDA tensors only (there is no CPU path); got a tensor on " + t.device().str());
    if (!seen) {
        dev = t.device();
        seen = true;
    } else if (t.device() != dev) {
        fail(PyExc_ValueError, "tensors live on different devices: " + dev.str() + " and " + t.device().str());
    }
}

int dtype_code(at::ScalarType t) {
    if (t == at::kFloat) return WA_F32;
    if (t == at::kBFloat16) return WA_BF16;
    fail(PyExc_ValueError, std::string("worldattention_b200 kernels take float32 or bfloat16 tensors, got ") +
                               (t == at::kHalf ? "torch.float16" : t == at::kDouble ? "torch.float64" : c10::toString(t)));
}

// `[B, L, H, D]` descriptor; `keep` holds a re-laid-out copy for the duration of the call where one is needed
wa_tensor4 view4(const Tensor &t, Tensor &keep) {
    if (t.dim() != 4) fail(PyExc_ValueError, "expected a [B, L, H, D] tensor, got shape " + shape_of(t));
    const Tensor *x = &t;
    if (t.stride(3) != 1 && t.size(3) != 1) {
        keep = t.contiguous();
        x = &keep;
    }
    return wa_tensor4{x->data_ptr(), dtype_code(x->scalar_type()), 0, x->stride(0), x->stride(1), x->stride(2)};
}

// a parameter as the kernels take it: on the device, contiguous, optionally in another tensor's dtype
const Tensor &plain(const Tensor &t, c10::Device dev, Tensor &keep, at::ScalarType dtype) {
    if (t.device() == dev && t.is_contiguous() && t.scalar_type() == dtype) return t;
    keep = t.detach().to(dev, dtype).contiguous();
    return keep;
}
const Tensor &plain(const Tensor &t, c10::Device dev, Tensor &keep) { return plain(t, dev, keep, t.scalar_type()); }

volatile int *status_word(int dev) {
    if (dev < 0 || dev >= MAX_DEVICES) fail(PyExc_RuntimeError, "device index out of range");
    if (!status_words[dev]) {
        PyObject *r = PyObject_CallFunction(py_status_word, "i", dev);
        if (!r) throw PyFailure();
        status_words[dev] = reinterpret_cast<volatile int *>(PyLong_AsVoidPtr(r));
        Py_DECREF(r);
        if (PyErr_Occurred()) throw PyFailure();
    }
    return status_words[dev];
}
void raise_if_failed(int dev) {
    if (*status_word(dev) == 0) return;
    pybind11::gil_scoped_acquire gil;       // (a gradient's call comes from a thread of the autograd engine)
    PyObject *r = PyObject_CallFunction(py_raise_if_failed, "i", dev);
    if (!r) throw PyFailure();
    Py_DECREF(r);
}

// ---- workspaces: one growing buffer per (kind, device, stream), the least recently used dropped beyond a bound ----
// A buffer is only handed out and its launches only enqueued while the interpreter lock is held, so two threads on one
// stream cannot interleave the launches that share it.  A dropped buffer goes back to the caching allocator, which
// recycles it in the order of the stream it was taken on.  A call that is being captured into a graph takes a buffer of
// its own (from the graph's memory pool): the graph outlives any bookkeeping here.
struct Slot {
    int kind, dev;
    cudaStream_t stream;
    Tensor buf;
};
std::list<Slot> &slots = *new std::list<Slot>;   // never destroyed: at exit the CUDA context may be gone before static objects
constexpr size_t MAX_SLOTS = 32;

Tensor workspace(int kind, c10::Device dev, cudaStream_t stream, size_t bytes, bool zeroed) {
    const auto opt = at::TensorOptions().dtype(at::kByte).device(dev);
    auto fresh = [&](size_t n) { return zeroed ? at::zeros({(int64_t)n}, opt) : at::empty({(int64_t)n}, opt); };
    if (at::cuda::currentStreamCaptureStatusMayInitCtx() != at::cuda::CaptureStatus::None) return fresh(bytes);
    for (auto it = slots.begin(); it != slots.end(); ++it)
        if (it->kind == kind && it->dev == dev.index() && it->stream == stream) {
            if (it != slots.begin()) slots.splice(slots.begin(), slots, it);
            if ((size_t)it->buf.numel() < bytes) {
                it->buf = Tensor();
                it->buf = fresh(bytes);
            }
            return it->buf;
        }
    if (slots.size() >= MAX_SLOTS) slots.pop_back();
    slots.push_front(Slot{kind, dev.index(), stream, fresh(std::max<size_t>(bytes, 1 << 20))});
    return slots.front().buf;
}

// ---- hsa_attention (wan/modules/hsa/attention.py:153-259) ---------------------------------------
// q, k, v, k_coarse|None, v_coarse|None, k_proj, v_proj, gate_w|None, gate_b|None, topk|None, block, tau_min, tau_max,
// segment, flags, k_pooled|None, k_pooled_valid, want_routing, check_status
//   -> out, or (out, index, num, thresholds, used_tuned) with want_routing
PyObject *hsa_forward(PyObject *const *a, Py_ssize_t n) {
    expect_args(n, 19);
    const Tensor &q = tensor(a[0], "q"), &k = tensor(a[1], "k"), &v0 = tensor(a[2], "v");
    const Tensor *kc = tensor_or_null(a[3], "k_coarse"), *vc = tensor_or_null(a[4], "v_coarse");
    const Tensor *gw = tensor_or_null(a[7], "gate weight"), *gb = tensor_or_null(a[8], "gate bias"), *topk = tensor_or_null(a[9], "topk_per_head");
    const Tensor *pooled = tensor_or_null(a[15], "k_pooled_cache");
    const bool want_routing = a[17] == Py_True, check_status = a[18] == Py_True;

    if (q.dim() != 4 || k.dim() != 4 || v0.dim() != 4) fail(PyExc_ValueError, "q, k and v must be [B, L, H, D] tensors");
    const int64_t B = q.size(0), Lq = q.size(1), H = q.size(2), D = q.size(3), Lkv = k.size(1);
    if (Lq <= 0 || Lkv <= 0) fail(PyExc_ValueError, "q_len and kv_len must be positive");
    c10::Device dev(c10::kCUDA, 0);
    bool seen = false;
    for (const Tensor *t : {&q, &k, &v0, kc, vc})
        if (t) require_cuda(*t, dev, seen);
    raise_if_failed(dev.index());
    c10::cuda::CUDAGuard guard(dev);
    cudaStream_t stream = at::cuda::getCurrentCUDAStream(dev.index()).stream();

    Tensor keep[12];
    wa_hsa_params p{};
    const long long block = integer(a[10]);
    if (block <= 0 || block > INT_MAX) fail(PyExc_ValueError, "block_size must be positive, got " + std::to_string(block));   // divided by below
    p.B = (int)B; p.H = (int)H; p.D = (int)D; p.Lq = (int)Lq; p.Lkv = (int)Lkv;
    p.block_size = (int)block;
    p.tau_min = real(a[11]);
    p.tau_max = real(a[12]);
    p.flags = (int)integer(a[14]);
    p.status_mirror = const_cast<int *>(status_word(dev.index()));
    const Tensor *v = &v0;
    if (v0.scalar_type() != k.scalar_type()) {
        keep[0] = v0.to(k.scalar_type());
        v = &keep[0];
    }
    p.q = view4(q, keep[1]);
    p.k = view4(k, keep[2]);
    p.v = view4(*v, keep[3]);
    if (pooled) {
        const int64_t blocks = (Lkv + block - 1) / block;
        if (pooled->scalar_type() != at::kFloat || pooled->sizes() != at::IntArrayRef({B, H, blocks, D}) || !pooled->is_contiguous() ||
            pooled->device() != dev)
            fail(PyExc_ValueError, "expected k_pooled_cache: contiguous float32 [" + std::to_string(B) + ", " + std::to_string(H) + ", " +
                                       std::to_string(blocks) + ", " + std::to_string(D) + "] on " + dev.str());
        const long long valid = integer(a[16]);
        if (valid < 0 || valid > blocks)
            fail(PyExc_ValueError, "k_pooled_valid must be in [0, " + std::to_string(blocks) + "], got " + std::to_string(valid));
        p.k_pooled = pooled->data_ptr<float>();
        p.k_pooled_valid = (int)valid;
    }
    if (kc) {
        if (kc->dim() != 4 || kc->size(0) != B || kc->size(2) != H || kc->size(3) != D)
            fail(PyExc_ValueError, "expected k_coarse shaped [B, Lc, " + std::to_string(H) + ", " + std::to_string(D) + "], got " + shape_of(*kc));
        if (vc->sizes() != kc->sizes()) fail(PyExc_ValueError, "v_coarse must have the same shape as k_coarse");
        if (kc->scalar_type() != vc->scalar_type()) {
            keep[4] = kc->to(vc->scalar_type());
            kc = &keep[4];
        }
        p.Lc = (int)kc->size(1);
        p.k_coarse = view4(*kc, keep[5]);
        p.v_coarse = view4(*vc, keep[6]);
    } else {
        const Tensor &kp = tensor(a[5], "k_proj_mat"), &vp = tensor(a[6], "v_proj_mat");
        if (kp.sizes() != vp.sizes())
            fail(PyExc_ValueError, "k_proj_mat and v_proj_mat must have the same shape, got " + shape_of(kp) + " and " + shape_of(vp));
        const long long asked = integer(a[13]), seg = asked > 0 ? asked : Lkv;
        if (std::min<long long>(seg, Lkv) > kp.size(1))
            fail(PyExc_ValueError, "segment length " + std::to_string(std::min<long long>(seg, Lkv)) + " exceeds projection length " +
                                       std::to_string(kp.size(1)) + "; increase proj_segment_len");
        const Tensor &pk = plain(kp, dev, keep[4]);
        const Tensor &pv = plain(vp, dev, keep[5], pk.scalar_type());
        p.proj_segment_len = (int)seg;
        p.proj_rank = (int)pk.size(0);
        p.proj_cols = (int)pk.size(1);
        p.proj_dtype = dtype_code(pk.scalar_type());
        p.k_proj = pk.data_ptr();
        p.v_proj = pv.data_ptr();
    }
    if (gw) {
        const Tensor &w = plain(*gw, dev, keep[7]);
        p.gate_dtype = dtype_code(w.scalar_type());
        p.gate_w = w.data_ptr();
        if (gb) p.gate_b = plain(*gb, dev, keep[8], w.scalar_type()).data_ptr();
    }
    if (topk) {
        const Tensor &counts = plain(*topk, dev, keep[9], at::kInt);
        if (counts.numel() != H) fail(PyExc_ValueError, "topk_per_head must have " + std::to_string(H) + " entries");
        p.topk_per_head = counts.data_ptr<int32_t>();
    }
    Tensor out = at::empty({B, Lq, H, D}, q.options().requires_grad(false));
    p.out = wa_tensor4{out.data_ptr(), dtype_code(out.scalar_type()), 0, Lq * H * D, H * D, D};
    Tensor index, num, thresholds;
    if (want_routing) {
        const int64_t nq = (Lq + block - 1) / block, nkv = (Lkv + block - 1) / block;
        const auto opt = at::TensorOptions().device(dev).dtype(at::kInt);
        index = at::empty({B, H, nq, nkv}, opt);
        num = at::empty({B, H, nq}, opt);
        thresholds = at::empty({H}, opt.dtype(at::kFloat));
        p.index_out = index.data_ptr<int32_t>();
        p.num_out = num.data_ptr<int32_t>();
        p.thresholds_out = thresholds.data_ptr<float>();
    }
    // A call that waits for its own status lets other threads run meanwhile, so its workspace is nobody else's.
    const size_t ws_bytes = f_workspace_bytes(&p);
    const Tensor ws = check_status ? at::empty({(int64_t)ws_bytes}, at::TensorOptions().dtype(at::kByte).device(dev))
                                   : workspace(0, dev, stream, ws_bytes, false);
    p.workspace = ws.data_ptr();
    p.workspace_bytes = (size_t)ws.numel();
    int used = 0;
    check(f_forward(&p, &used, stream));
    if (check_status && used) {
        int status = 0, rc = 0;
        Py_BEGIN_ALLOW_THREADS          // waits for the stream: other threads may be what it waits for
        rc = f_status(&p, &status, stream);
        Py_END_ALLOW_THREADS
        check(rc);
        if (status) {
            *status_word(dev.index()) = 0;
            fail(PyExc_RuntimeError, "tcgen05 HSA kernel gave up at wait site " + std::to_string(status) + "; its output is invalid");
        }
    }
    if (!want_routing) return THPVariable_Wrap(std::move(out));
    return Py_BuildValue("(NNNNO)", THPVariable_Wrap(out), THPVariable_Wrap(index), THPVariable_Wrap(num), THPVariable_Wrap(thresholds),
                         used ? Py_True : Py_False);
}

// ---- run_forward: address of a wa_hsa_params (workspace unset), device index -> used_tuned, or None ----------------
// For callers that fill the parameters themselves (partial outputs of a key shard): the stream's kept workspace and the
// launches, under the interpreter lock as above.  None: the call asked for the tcgen05 kernel, which does not cover it.
PyObject *run_forward(PyObject *const *a, Py_ssize_t n) {
    expect_args(n, 2);
    wa_hsa_params *p = reinterpret_cast<wa_hsa_params *>(PyLong_AsVoidPtr(a[0]));
    if (PyErr_Occurred()) throw PyFailure();
    if (!p) fail(PyExc_ValueError, "null parameters");
    const c10::Device dev(c10::kCUDA, (c10::DeviceIndex)integer(a[1]));
    c10::cuda::CUDAGuard guard(dev);
    cudaStream_t stream = at::cuda::getCurrentCUDAStream(dev.index()).stream();
    const Tensor ws = workspace(0, dev, stream, f_workspace_bytes(p), false);
    p->workspace = ws.data_ptr();
    p->workspace_bytes = (size_t)ws.numel();
    int used = 0;
    const int rc = f_forward(p, &used, stream);
    if (rc == WA_ERR_UNSUPPORTED && (p->flags & WA_HSA_REQUIRE_TUNED)) Py_RETURN_NONE;
    check(rc);
    return PyBool_FromLong(used);
}

// ---- qk_norm_rope: x [B, L, H, D], weight|None, eps, table|None, start_frame (int or int32 device tensor), grid_h, grid_w -> out ----
PyObject *qk_norm_rope(PyObject *const *a, Py_ssize_t n) {
    expect_args(n, 7);
    const Tensor &x = tensor(a[0], "x");
    c10::Device dev(c10::kCUDA, 0);
    bool seen = false;
    require_cuda(x, dev, seen);
    c10::cuda::CUDAGuard guard(dev);
    cudaStream_t stream = at::cuda::getCurrentCUDAStream(dev.index()).stream();
    Tensor keep[2];
    const wa_tensor4 xv = view4(x, keep[0]);
    Tensor out = at::empty(x.sizes(), x.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous));
    const int64_t L = x.size(1), H = x.size(2), D = x.size(3);
    const wa_tensor4 ov{out.data_ptr(), xv.dtype, 0, L * H * D, H * D, D};
    const Tensor *weight = tensor_or_null(a[1], "norm_weight"), *table = tensor_or_null(a[3], "table");
    const void *wp = nullptr;
    int wdt = 0;
    if (weight) {
        const Tensor &w = plain(*weight, dev, keep[1]);
        wp = w.data_ptr();
        wdt = dtype_code(w.scalar_type());
    }
    const double *freqs = table ? table->data_ptr<double>() : nullptr;
    const int rows = table ? (int)table->size(0) : 0, gh = (int)integer(a[5]), gw = (int)integer(a[6]);
    const float eps = (float)real(a[2]);
    if (THPVariable_Check(a[4])) {
        const Tensor &at_frame = THPVariable_Unpack(a[4]);
        if (at_frame.scalar_type() != at::kInt || at_frame.numel() != 1 || at_frame.device() != dev)
            fail(PyExc_ValueError, "a device-resident start_frame must be one int32 on the tensors' device");
        check(f_rope_at(&xv, &ov, (int)x.size(0), (int)L, (int)H, (int)D, wp, wdt, eps, freqs, rows, at_frame.data_ptr<int32_t>(), gh, gw, stream));
    } else {
        check(f_rope(&xv, &ov, (int)x.size(0), (int)L, (int)H, (int)D, wp, wdt, eps, freqs, rows, (int)integer(a[4]), gh, gw, stream));
    }
    return THPVariable_Wrap(std::move(out));
}

// ---- append_kv: k_new, v_new, k_cache, v_cache, k_coarse, v_coarse, position, segment, k_proj, v_proj, block -> bool ----
// False: the fused kernel does not cover the shape or the layout (nothing was launched).
PyObject *append_kv(PyObject *const *a, Py_ssize_t n) {
    expect_args(n, 11);
    static const char *names[6] = {"k_new", "v_new", "k_cache", "v_cache", "k_coarse", "v_coarse"};
    c10::Device dev(c10::kCUDA, 0);
    bool seen = false;
    Tensor keep[8];
    wa_tensor4 t[6];
    for (int i = 0; i < 6; ++i) require_cuda(tensor(a[i], names[i]), dev, seen);
    const Tensor &k_new = THPVariable_Unpack(a[0]);
    if (k_new.dim() != 4) fail(PyExc_ValueError, "expected [B, L, H, D] tensors");
    const long long position = integer(a[6]), seg = integer(a[7]), block = integer(a[10]);
    if (seg <= 0 || position % seg)
        fail(PyExc_ValueError, "rows are appended at segment boundaries, got position=" + std::to_string(position) + ", segment_len=" + std::to_string(seg));
    if (position + k_new.size(1) > THPVariable_Unpack(a[2]).size(1)) fail(PyExc_ValueError, "the rows do not fit the cache");
    if (seg > INT_MAX || block <= 0 || block > INT_MAX) fail(PyExc_ValueError, "segment_len and block_size must be positive");
    // what the kernels write, addressed from here on: rows in both caches, `rank` slots per whole segment in both tiers
    const int64_t rank_rows = tensor(a[8], "k_proj_mat").dim() == 2 ? THPVariable_Unpack(a[8]).size(0) : 0;
    const int64_t n_new = k_new.size(1), whole = n_new / seg, tail = n_new % seg;
    const int64_t stride = std::min<int64_t>(rank_rows, (seg + block - 1) / block);
    const int64_t slots = (position / seg + whole) * stride + std::min<int64_t>(rank_rows, (tail + block - 1) / block);
    for (int i = 1; i < 6; ++i) {
        const Tensor &x = THPVariable_Unpack(a[i]);
        const int64_t rows = i == 1 ? n_new : i < 4 ? position + n_new : slots;
        if (x.dim() != 4 || x.size(0) < k_new.size(0) || x.size(1) < rows || x.size(2) < k_new.size(2) || x.size(3) < k_new.size(3))
            fail(PyExc_ValueError, std::string(names[i]) + " of shape " + shape_of(x) + " does not hold the rows of k_new " + shape_of(k_new) +
                                       " (" + std::to_string(rows) + " of them are needed)");
    }
    for (int i = 2; i < 6; ++i) {      // written in place: a re-laid-out copy would take the rows
        const Tensor &dst = THPVariable_Unpack(a[i]);
        if (dst.dim() == 4 && dst.stride(3) != 1 && dst.size(3) != 1) Py_RETURN_FALSE;
    }
    for (int i = 0; i < 6; ++i) t[i] = view4(THPVariable_Unpack(a[i]), keep[i]);
    c10::cuda::CUDAGuard guard(dev);
    cudaStream_t stream = at::cuda::getCurrentCUDAStream(dev.index()).stream();
    const Tensor &pk = plain(tensor(a[8], "k_proj_mat"), dev, keep[6]);
    const Tensor &pv = plain(tensor(a[9], "v_proj_mat"), dev, keep[7], pk.scalar_type());
    const int B = (int)k_new.size(0), N = (int)k_new.size(1), H = (int)k_new.size(2), D = (int)k_new.size(3), rank = (int)pk.size(0);
    auto call = [&](void *ws, size_t bytes) {
        return f_append(&t[0], &t[1], &t[2], &t[3], &t[4], &t[5], B, N, (int)position, H, D, (int)seg, (int)block, pk.data_ptr(), pv.data_ptr(),
                        dtype_code(pk.scalar_type()), rank, (int)pk.size(1), ws, bytes, stream);
    };
    int rc = call(nullptr, 0);                                     // the tensor-core stream needs no workspace
    if (rc == WA_ERR_WORKSPACE) {
        const Tensor ws = workspace(1, dev, stream, f_append_bytes(B, N, H, D, (int)seg, (int)block, rank), true);   // zeroed once; every call leaves the counters zeroed
        rc = call(ws.data_ptr(), (size_t)ws.numel());
    }
    if (rc == WA_ERR_UNSUPPORTED) Py_RETURN_FALSE;
    check(rc);
    Py_RETURN_TRUE;
}

// ---- the element-wise steps of a block (causal_dit.py) ------------------------------------------
// `[B, F, 1, C]` or `[B, F, C]` modulation view -> (pointer, elements between consecutive frames); it must step uniformly
// over (b, f) and hold a vector for every `tokens` of the `rows` rows: the kernels take the vector of row / tokens
const void *frame_vectors(const Tensor *e, int64_t rows, int64_t tokens, int64_t dim, Tensor &keep, long long &stride) {
    if (!e) return nullptr;
    const Tensor *t = e;
    if (e->dim() < 3 || e->size(-1) < dim) fail(PyExc_ValueError, "expected a [B, F, 1, C] or [B, F, C] modulation, got shape " + shape_of(*e));
    const int64_t b = e->size(0), f = e->size(1);
    if (tokens > 0 && (rows + tokens - 1) / tokens > b * f)
        fail(PyExc_ValueError, std::to_string(rows) + " rows of " + std::to_string(tokens) + " tokens per frame need more than the modulation's " +
                                   std::to_string(b * f) + " frames");
    if (e->stride(-1) != 1 || (b > 1 && e->stride(0) != f * e->stride(1))) {
        keep = e->contiguous();
        t = &keep;
    }
    stride = t->stride(1);
    return t->data_ptr();
}

const Tensor &rows_bf16(const Tensor &t, Tensor &keep) {
    if (t.scalar_type() != at::kBFloat16) fail(PyExc_NotImplementedError, "the fused block glue is bf16 only");
    if (t.is_contiguous()) return t;
    keep = t.contiguous();
    return keep;
}

// x, eps, weight|None, bias|None, scale|None, shift|None, tokens_per_frame -> out
PyObject *ln_modulate(PyObject *const *a, Py_ssize_t n) {
    expect_args(n, 7);
    c10::Device dev(c10::kCUDA, 0);
    bool seen = false;
    require_cuda(tensor(a[0], "x"), dev, seen);
    Tensor keep[3];
    const Tensor &x = rows_bf16(THPVariable_Unpack(a[0]), keep[0]);
    c10::cuda::CUDAGuard guard(dev);
    cudaStream_t stream = at::cuda::getCurrentCUDAStream(dev.index()).stream();
    Tensor out = at::empty(x.sizes(), x.options().requires_grad(false));
    const int64_t c = x.size(-1);
    const Tensor *w = tensor_or_null(a[2], "weight"), *b = tensor_or_null(a[3], "bias");
    const Tensor *scale = tensor_or_null(a[4], "scale"), *shift = tensor_or_null(a[5], "shift");
    long long ss = 0, hs = 0;
    const int64_t rows = c ? x.numel() / c : 0, tokens = (int)integer(a[6]);
    const void *sp = frame_vectors(scale, rows, tokens, c, keep[1], ss), *hp = frame_vectors(shift, rows, tokens, c, keep[2], hs);
    if (sp && hp && ss != hs) fail(PyExc_ValueError, "scale and shift must share a layout");
    check(f_ln(x.data_ptr(), out.data_ptr(), rows, (int)c, (float)real(a[1]), w ? w->data_ptr() : nullptr, b ? b->data_ptr() : nullptr,
               sp, hp, ss ? ss : hs, (int)tokens, stream));
    return THPVariable_Wrap(std::move(out));
}

// x, y, gate|None, tokens_per_frame -> out
PyObject *gated_residual(PyObject *const *a, Py_ssize_t n) {
    expect_args(n, 4);
    c10::Device dev(c10::kCUDA, 0);
    bool seen = false;
    require_cuda(tensor(a[0], "x"), dev, seen);
    Tensor keep[3];
    const Tensor &x = rows_bf16(THPVariable_Unpack(a[0]), keep[0]), &y = rows_bf16(tensor(a[1], "y"), keep[1]);
    c10::cuda::CUDAGuard guard(dev);
    cudaStream_t stream = at::cuda::getCurrentCUDAStream(dev.index()).stream();
    Tensor out = at::empty(x.sizes(), x.options().requires_grad(false));
    const int64_t c = x.size(-1);
    long long gs = 0;
    const int64_t rows = c ? x.numel() / c : 0, tokens = (int)integer(a[3]);
    const void *gp = frame_vectors(tensor_or_null(a[2], "gate"), rows, tokens, c, keep[2], gs);
    check(f_residual(x.data_ptr(), y.data_ptr(), out.data_ptr(), rows, (int)c, gp, gs, (int)tokens, stream));
    return THPVariable_Wrap(std::move(out));
}

// A sequence's elements, for the time of a call
struct Sequence {
    PyObject *o;
    Sequence(PyObject *seq, const char *what) : o(PySequence_Fast(seq, what)) {
        if (!o) throw PyFailure();
    }
    ~Sequence() { Py_DECREF(o); }
    Sequence(const Sequence &) = delete;
    Py_ssize_t size() const { return PySequence_Fast_GET_SIZE(o); }
    PyObject *operator[](Py_ssize_t i) const { return PySequence_Fast_GET_ITEM(o, i); }
};
int small_integer(PyObject *o, const char *what) {
    const long long v = integer(o);
    if (v < INT_MIN || v > INT_MAX) fail(PyExc_ValueError, std::string(what) + " must fit 32 bits");
    return (int)v;
}

// Tangents of forward-mode derivatives are not carried: a call that has one is refused, where it would be lost without a word.
void refuse_tangents(at::TensorList xs) {
    for (const Tensor &x : xs)
        if (torch::autograd::impl::get_autograd_meta(x) && x._fw_grad(/*level=*/0).defined()) fail(PyExc_NotImplementedError, "forward-mode derivatives are not offered: a tensor of the call has a tangent");
}

// ---- attention over selected blocks (hsa/selected.py): q [B, Lq, H, D], k, v [B, Lkv, Hkv, D], index [B, H, Nq, S], num [B, H, Nq], block, block_sizes|None,
// lists as block_sparse_attention takes them (hsa/block_sparse_torch.py) ----
struct SelectedCall {
    wa_selected_params p{};
    Tensor keep[9];
    c10::Device dev{c10::kCUDA, 0};
    bool nothing = false;              // no query or no key: no launch

    SelectedCall(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &index, const Tensor &num, int block, const Tensor *sizes, bool as_listed) {
        bool seen = false;
        for (const Tensor *t : {&q, &k, &v, &index, &num}) require_cuda(*t, dev, seen);
        if (sizes) require_cuda(*sizes, dev, seen);
        if (q.dim() != 4 || k.dim() != 4 || v.dim() != 4) fail(PyExc_ValueError, "q, k and v must be [B, L, H, D] tensors");
        const int64_t B = q.size(0), Lq = q.size(1), H = q.size(2), D = q.size(3), Lkv = k.size(1), Hkv = k.size(2);
        for (const int64_t x : {B, Lq, H, D, Lkv, Hkv})
            if (x > INT_MAX) fail(PyExc_NotImplementedError, "sizes must fit 32 bits");
        if (k.sizes() != v.sizes() || k.size(0) != B || k.size(3) != D)
            fail(PyExc_ValueError, "k and v must be [B, Lkv, Hkv, D] with q's B and D, got q " + shape_of(q) + ", k " + shape_of(k) + ", v " + shape_of(v));
        if (k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type()) fail(PyExc_ValueError, "q, k and v must have one dtype");
        dtype_code(q.scalar_type());
        if (H == 0 || Hkv == 0 || H % Hkv) fail(PyExc_ValueError, std::to_string(H) + " query heads do not divide among " + std::to_string(Hkv) + " key heads");
        if (block <= 0) fail(PyExc_ValueError, "block_size must be positive, got " + std::to_string(block));
        const int64_t nq = (Lq + block - 1) / block, nkv = (Lkv + block - 1) / block;
        if (index.dim() != 4 || index.size(0) != B || index.size(1) != H || index.size(2) != nq || num.dim() != 3 || num.size(0) != B || num.size(1) != H || num.size(2) != nq)
            fail(PyExc_ValueError, "index must be [B, H, Nq, ids] and num [B, H, Nq] with Nq = " + std::to_string(nq) + " query blocks, got " + shape_of(index) + " and " + shape_of(num));
        if (index.scalar_type() != at::kInt || num.scalar_type() != at::kInt) fail(PyExc_ValueError, "index and num must be int32");
        if (sizes && (sizes->dim() != 1 || (as_listed ? sizes->size(0) < nkv : sizes->size(0) != nkv) || sizes->scalar_type() != at::kInt))
            fail(PyExc_ValueError, "block_sizes must be int32 [" + std::to_string(nkv) + "], got shape " + shape_of(*sizes));
        nothing = B == 0 || Lq == 0 || Lkv == 0 || D == 0 || index.size(3) == 0;
        p.as_listed = as_listed;
        p.B = (int)B; p.H = (int)H; p.Hkv = (int)Hkv; p.D = (int)D; p.Lq = (int)Lq; p.Lkv = (int)Lkv; p.block_size = block;
        if (index.size(3) > INT_MAX) fail(PyExc_NotImplementedError, "sizes must fit 32 bits");
        p.index_stride = (int)index.size(3);
        if (nothing) return;
        p.q = view4(q, keep[0]); p.k = view4(k, keep[1]); p.v = view4(v, keep[2]);
        keep[3] = index.contiguous(); keep[4] = num.contiguous();
        p.index = keep[3].data_ptr<int32_t>(); p.num = keep[4].data_ptr<int32_t>();
        if (sizes) {
            keep[5] = sizes->contiguous();
            p.block_sizes = keep[5].data_ptr<int32_t>();
        }
        p.status_mirror = const_cast<int32_t *>(reinterpret_cast<volatile int32_t *>(status_word(dev.index())));
    }
    // the workspace lives in the caching allocator for the time of the call: recycled in the stream's order, a graph's own while one is captured
    Tensor workspace_for(bool backward) {
        const size_t bytes = f_selected_bytes(&p, backward);
        if (bytes == 0) check(backward ? f_selected_backward(&p, nullptr) : f_selected_forward(&p, nullptr));      // says why
        Tensor ws = at::empty({(int64_t)bytes}, at::TensorOptions().dtype(at::kByte).device(dev));
        p.workspace = ws.data_ptr();
        p.workspace_bytes = bytes;
        return ws;
    }
};
wa_tensor4 result4(const Tensor &t) { return wa_tensor4{t.data_ptr(), dtype_code(t.scalar_type()), 0, t.stride(0), t.stride(1), t.stride(2)}; }

// -> out [B, Lq, H, D], lse float32 [B, H, Lq]
std::pair<Tensor, Tensor> selected_run(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &index, const Tensor &num, int block, const Tensor *sizes,
                                       bool as_listed) {
    SelectedCall c(q, k, v, index, num, block, sizes, as_listed);
    raise_if_failed(c.dev.index());
    c10::cuda::CUDAGuard guard(c.dev);
    const auto options = q.options().requires_grad(false);
    // (as listed: [B, H, Lq, D] in memory, as that call's results lie without gradients)
    const int64_t B = c.p.B, H = c.p.H, L = c.p.Lq, D = c.p.D;
    Tensor out = as_listed ? at::empty_strided({B, L, H, D}, {H * L * D, D, L * D, 1}, options) : at::empty(q.sizes(), options.memory_format(at::MemoryFormat::Contiguous));
    if (c.nothing) return {out.zero_(), at::full({B, H, L}, -INFINITY, options.dtype(at::kFloat))};
    Tensor lse = at::empty({B, H, L}, options.dtype(at::kFloat).memory_format(at::MemoryFormat::Contiguous));
    c.p.out = result4(out);
    c.p.lse = lse.data_ptr<float>();
    const Tensor ws = c.workspace_for(false);
    check(f_selected_forward(&c.p, at::cuda::getCurrentCUDAStream(c.dev.index()).stream()));
    return {out, lse};
}

// -> dq, dk, dv
std::vector<Tensor> selected_gradients(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &index, const Tensor &num, int block, const Tensor *sizes,
                                       bool as_listed, const Tensor &out, const Tensor &lse, const Tensor &dout) {
    SelectedCall c(q, k, v, index, num, block, sizes, as_listed);
    raise_if_failed(c.dev.index());
    bool seen = true;
    for (const Tensor *t : {&out, &lse, &dout}) require_cuda(*t, c.dev, seen);
    c10::cuda::CUDAGuard guard(c.dev);
    if (out.sizes() != q.sizes() || dout.sizes() != q.sizes() || out.scalar_type() != q.scalar_type() || dout.scalar_type() != q.scalar_type())
        fail(PyExc_ValueError, "out and dout must have q's shape and dtype");
    std::vector<Tensor> grad(3);
    for (int i = 0; i < 3; ++i) {
        const Tensor &x = i == 0 ? q : k;
        const auto options = x.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous);
        grad[i] = c.nothing ? at::zeros(x.sizes(), x.options().requires_grad(false)) : at::empty(x.sizes(), options);
    }
    if (c.nothing) return grad;
    if (lse.scalar_type() != at::kFloat || lse.numel() != (int64_t)c.p.B * c.p.H * c.p.Lq) fail(PyExc_ValueError, "lse must be float32 [B, H, Lq]");
    // (a gradient without memory of its own, or of odd strides, is laid out: the tensor-core kernels read 16 bytes at a time)
    const bool odd = dout.scalar_type() == at::kBFloat16 && (dout.stride(0) % 8 || dout.stride(1) % 8 || dout.stride(2) % 8 || dout.stride(1) <= 0 || dout.stride(2) <= 0);
    const Tensor laid = odd ? dout.contiguous() : dout;
    c.p.out = view4(out, c.keep[6]);
    c.p.dout = view4(laid, c.keep[7]);
    c.keep[8] = lse.contiguous();
    c.p.lse = c.keep[8].data_ptr<float>();
    c.p.dq = result4(grad[0]); c.p.dk = result4(grad[1]); c.p.dv = result4(grad[2]);
    const Tensor ws = c.workspace_for(true);
    check(f_selected_backward(&c.p, at::cuda::getCurrentCUDAStream(c.dev.index()).stream()));
    return grad;
}

// Autograd nodes live here because a Python one costs a step 60 us: its backward takes the interpreter lock on the engine's thread.
[[noreturn]] void rethrow_on_engine() {       // what `fail` left on this thread, as an exception that the engine carries to the caller
    pybind11::gil_scoped_acquire gil;
    python_error e;
    e.persist();
    throw std::move(e);
}

// A captured backward pass ends at its leaves.  A leaf that an eager graph still leads to keeps that graph's stream; where that is the default
// stream, the engine makes it wait for the captured one, which is no legal step of a capture and ends the process.  So such a call is
// refused while that can still be an exception: at once where a leaf is an input, or one seen through views and other nodes of one input, and in the
// backward pass, before a gradient leaves this node, for every leaf that the pass will reach from here.
bool capturing() { return at::cuda::currentStreamCaptureStatusMayInitCtx() != at::cuda::CaptureStatus::None; }
void refuse_eager_leaf(torch::autograd::Node &node) {
    const auto stream = node.stream();
    if (stream && stream->device_type() == c10::kCUDA && *stream == at::cuda::getDefaultCUDAStream(stream->device_index()).unwrap())
        fail(PyExc_RuntimeError, "a training step cannot be captured while an eager graph of the same leaves, made on the default stream, is alive: drop its "
                                 "results first, or make it on a side stream");
}
void refuse_captured_over_eager(at::TensorList xs) {
    if (!capturing()) return;
    for (const Tensor &x : xs) {
        if (!x.requires_grad()) continue;
        std::shared_ptr<torch::autograd::Node> node = x.grad_fn() ? x.grad_fn() : torch::autograd::impl::try_get_grad_accumulator(x);
        while (node && node->num_outputs() == 1) node = node->next_edge(0).function;
        if (node && node->num_outputs() == 0) refuse_eager_leaf(*node);
    }
}
void refuse_captured_backward_over_eager() {
    if (!capturing()) return;
    const auto *tasks = torch::autograd::get_current_graph_task_exec_info();      // empty: everything is executed
    std::unordered_set<const torch::autograd::Node *> seen;
    std::vector<std::shared_ptr<torch::autograd::Node>> todo{torch::autograd::get_current_node()};
    while (!todo.empty()) {
        const auto node = todo.back();
        todo.pop_back();
        if (!node || !seen.insert(node.get()).second) continue;
        if (seen.size() > 1 && tasks && !tasks->empty()) {
            const auto task = tasks->find(node.get());
            if (task == tasks->end() || !task->second.should_execute()) continue;
            if (!task->second.needed_ && node->num_outputs() != 0) continue;      // its gradient is wanted, and none behind it
        }
        if (node->num_outputs() == 0) refuse_eager_leaf(*node);
        for (const auto &edge : node->next_edges()) todo.push_back(edge.function);
    }
}

struct SelectedNode : torch::autograd::Function<SelectedNode> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &index,
                                                  const Tensor &num, int64_t block, const std::optional<Tensor> &sizes, bool as_listed) {
        auto [out, lse] = selected_run(q, k, v, index, num, (int)block, sizes ? &*sizes : nullptr, as_listed);
        ctx->save_for_backward({q, k, v, index, num, sizes ? *sizes : Tensor(), out, lse});
        ctx->saved_data["block"] = block;
        ctx->saved_data["as_listed"] = as_listed;
        ctx->mark_non_differentiable({lse});
        ctx->set_materialize_grads(false);
        return {out, lse};
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, const torch::autograd::variable_list &grads) {
        torch::autograd::variable_list result(8);
        if (!grads[0].defined()) return result;
        const auto s = ctx->get_saved_variables();
        torch::autograd::variable_list three;
        try {
            refuse_captured_backward_over_eager();
            at::NoGradGuard no_grad;
            three = selected_gradients(s[0], s[1], s[2], s[3], s[4], (int)ctx->saved_data["block"].toInt(), s[5].defined() ? &s[5] : nullptr,
                                       ctx->saved_data["as_listed"].toBool(), s[6], s[7], grads[0].detach());
        } catch (const PyFailure &) {
            rethrow_on_engine();
        }
        if (at::GradMode::is_enabled()) {     // (create_graph: these gradients have no gradient)
            for (Tensor &t : three) t.requires_grad_();
            const auto error = std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice a function that was marked with @once_differentiable", 3);
            three = (*error)(std::move(three));
        }
        for (int i = 0; i < 3; ++i)
            if (ctx->needs_input_grad(i)) result[i] = three[i];
        return result;
    }
};

// q, k, v, index, num, block, block_sizes|None, as listed -> (out, lse), with a graph where gradients are asked for
PyObject *selected_attention(PyObject *const *a, Py_ssize_t n) {
    expect_args(n, 8);
    const Tensor &q = tensor(a[0], "q"), &k = tensor(a[1], "k"), &v = tensor(a[2], "v"), &index = tensor(a[3], "index"), &num = tensor(a[4], "num");
    const int block = small_integer(a[5], "block_size");
    const Tensor *sizes = tensor_or_null(a[6], "block_sizes");
    const bool as_listed = a[7] == Py_True;
    refuse_tangents({q, k, v});
    Tensor out, lse;
    if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad())) {
        if (!as_listed) refuse_captured_over_eager({q, k, v});      // (a forward pass alone was captured before that call carried gradients)
        auto both = SelectedNode::apply(q, k, v, index, num, (int64_t)block, sizes ? std::optional<Tensor>(*sizes) : std::nullopt, as_listed);
        out = std::move(both[0]);
        lse = std::move(both[1]);
    } else {
        std::tie(out, lse) = selected_run(q, k, v, index, num, block, sizes, as_listed);
    }
    PyObject *pair = PyTuple_New(2);
    if (!pair) throw PyFailure();
    PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(std::move(out)));
    PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(std::move(lse)));
    return pair;
}

// ---- axial_rope(tensors, positions int32 [L, A] or [B, L, A], table float32 [rows, pairs, 2], pairs of each axis, interleaved) -> list of tensors ----
std::vector<Tensor> axial_run(at::TensorList xs, const Tensor &pos0, const Tensor &table0, const std::vector<int64_t> &axes, bool interleaved, bool inverse) {
    constexpr size_t MOST = 4;
    if (xs.size() < 1 || xs.size() > MOST) fail(PyExc_ValueError, "expected one to four tensors, got " + std::to_string(xs.size()));
    c10::Device dev(c10::kCUDA, 0);
    bool seen = false;
    for (const Tensor &x : xs) require_cuda(x, dev, seen);
    require_cuda(pos0, dev, seen);
    require_cuda(table0, dev, seen);
    const Tensor &x0 = xs[0];
    if (x0.dim() != 4) fail(PyExc_ValueError, "expected [B, L, H, D] tensors, got shape " + shape_of(x0));
    const int64_t B = x0.size(0), L = x0.size(1), D = x0.size(3), A = (int64_t)axes.size();
    if (B > INT_MAX || L > INT_MAX || D > INT_MAX) fail(PyExc_NotImplementedError, "sizes must fit 32 bits");
    int pairs[8];
    if (A < 1 || A > 8) fail(PyExc_ValueError, "expected one to eight axes, got " + std::to_string(A));
    int64_t sum = 0;
    for (int64_t i = 0; i < A; ++i) sum += pairs[i] = (int)axes[i];
    if (table0.dim() != 3 || table0.size(2) != 2 || table0.size(0) < 1 || table0.scalar_type() != at::kFloat)
        fail(PyExc_ValueError, "table must be float32 [rows, pairs, 2], got shape " + shape_of(table0));
    if (table0.size(1) != sum || 2 * sum > D)
        fail(PyExc_ValueError, "the axes turn " + std::to_string(sum) + " pairs, the table has " + std::to_string(table0.size(1)) + " and a head " + std::to_string(D / 2));
    const bool shared = pos0.dim() == 2;
    if (pos0.scalar_type() != at::kInt || (!shared && pos0.dim() != 3) || pos0.size(-1) != A || pos0.size(-2) != L || (!shared && pos0.size(0) != B))
        fail(PyExc_ValueError, "positions must be int32 [L, axes] or [B, L, axes] for tensors of shape " + shape_of(x0) + ", got shape " + shape_of(pos0));
    c10::cuda::CUDAGuard guard(dev);
    cudaStream_t stream = at::cuda::getCurrentCUDAStream(dev.index()).stream();
    const Tensor pos = pos0.stride(-1) == 1 || A == 1 ? pos0 : pos0.contiguous(), table = table0.contiguous();
    wa_tensor4 in[MOST], out[MOST];
    int32_t heads[MOST];
    Tensor keep[MOST];
    std::vector<Tensor> result(xs.size());
    for (size_t t = 0; t < xs.size(); ++t) {
        const Tensor &x = xs[t];
        if (x.dim() != 4 || x.size(0) != B || x.size(1) != L || x.size(3) != D || x.scalar_type() != x0.scalar_type())
            fail(PyExc_ValueError, "the tensors must share batch, length, head_dim and dtype, got shapes " + shape_of(x0) + " and " + shape_of(x));
        if (x.size(2) > INT_MAX) fail(PyExc_NotImplementedError, "sizes must fit 32 bits");
        in[t] = view4(x, keep[t]);
        result[t] = at::empty(x.sizes(), x.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous));
        out[t] = result4(result[t]);
        heads[t] = (int32_t)x.size(2);
    }
    check(f_axial(in, out, heads, (int)xs.size(), (int)B, (int)L, (int)D, pos.data_ptr<int32_t>(), shared ? 0 : pos.stride(0), pos.stride(-2), pairs, (int)A,
                  table.data_ptr<float>(), (int)std::min<int64_t>(table.size(0), INT_MAX), interleaved, inverse, stream));
    return result;
}

std::vector<Tensor> axial_turn(const std::vector<Tensor> &xs, const Tensor &pos, const Tensor &table, const std::vector<int64_t> &axes, bool interleaved, bool inverse);

struct AxialNode : torch::autograd::Function<AxialNode> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext *ctx, const Tensor &pos, const Tensor &table, std::vector<int64_t> axes,
                                                  bool interleaved, bool inverse, at::TensorList xs) {
        ctx->save_for_backward({pos, table});
        ctx->saved_data["axes"] = axes;
        ctx->saved_data["interleaved"] = interleaved;
        ctx->saved_data["inverse"] = inverse;
        ctx->set_materialize_grads(false);
        return axial_run(xs, pos, table, axes, interleaved, inverse);
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, const torch::autograd::variable_list &grads) {
        const auto s = ctx->get_saved_variables();
        torch::autograd::variable_list result(5 + grads.size());
        std::vector<Tensor> there;
        std::vector<size_t> at;
        for (size_t i = 0; i < grads.size(); ++i)
            if (grads[i].defined() && ctx->needs_input_grad(2 + i)) {      // (counts tensors: positions, table, then these)
                there.push_back(grads[i]);
                at.push_back(5 + i);
            }
        if (there.empty()) return result;
        try {
            refuse_captured_backward_over_eager();
            const auto turned = axial_turn(there, s[0], s[1], ctx->saved_data["axes"].toIntVector(), ctx->saved_data["interleaved"].toBool(), !ctx->saved_data["inverse"].toBool());
            for (size_t i = 0; i < at.size(); ++i) result[at[i]] = turned[i];
        } catch (const PyFailure &) {
            rethrow_on_engine();
        }
        return result;
    }
};

std::vector<Tensor> axial_turn(const std::vector<Tensor> &xs, const Tensor &pos, const Tensor &table, const std::vector<int64_t> &axes, bool interleaved, bool inverse) {
    refuse_tangents(xs);
    refuse_tangents(table);
    if (at::GradMode::is_enabled() && table.requires_grad()) fail(PyExc_ValueError, "the table has no gradient: it must not require one");
    if (at::GradMode::is_enabled() && std::any_of(xs.begin(), xs.end(), [](const Tensor &x) { return x.requires_grad(); })) {
        refuse_captured_over_eager(xs);
        return AxialNode::apply(pos, table, axes, interleaved, inverse, at::TensorList(xs));
    }
    return axial_run(xs, pos, table, axes, interleaved, inverse);
}

PyObject *axial_rope(PyObject *const *a, Py_ssize_t n) {
    expect_args(n, 5);
    const Sequence given(a[0], "expected a tensor or a tuple of tensors"), pairs(a[3], "axes must be a sequence of integers");
    std::vector<Tensor> xs;
    for (Py_ssize_t t = 0; t < given.size(); ++t) xs.push_back(tensor(given[t], "every element"));
    std::vector<int64_t> axes;
    for (Py_ssize_t i = 0; i < pairs.size(); ++i) axes.push_back(small_integer(pairs[i], "axes"));
    std::vector<Tensor> result = axial_turn(xs, tensor(a[1], "positions"), tensor(a[2], "table"), axes, a[4] == Py_True, false);
    PyObject *list = PyList_New((Py_ssize_t)result.size());
    if (!list) throw PyFailure();
    for (size_t t = 0; t < result.size(); ++t) PyList_SET_ITEM(list, (Py_ssize_t)t, THPVariable_Wrap(std::move(result[t])));
    return list;
}

// ---- move_pages(tensors [B, tokens, ...], destination pages, source pages or None, tokens of a page: one or one per tensor) ----
PyObject *move_pages(PyObject *const *a, Py_ssize_t n) {
    expect_args(n, 4);
    const Sequence xs(a[0], "expected a sequence of tensors"), to(a[1], "destination must be a sequence of page numbers"),
        from(a[2], "source must be a sequence of page numbers or None");
    if (to.size() != from.size())
        fail(PyExc_ValueError, "destination and source must be equally long, got " + std::to_string(to.size()) + " and " + std::to_string(from.size()));
    const bool one = PyIndex_Check(a[3]);
    std::vector<int32_t> dst(to.size()), src(from.size());
    for (Py_ssize_t i = 0; i < to.size(); ++i) {
        dst[i] = small_integer(to[i], "page numbers");
        src[i] = from[i] == Py_None ? -1 : small_integer(from[i], "page numbers");
        if (dst[i] < 0 || (src[i] < 0 && from[i] != Py_None)) fail(PyExc_ValueError, "page numbers must not be negative");
    }
    std::vector<wa_page_tensor> tensors(xs.size());
    std::vector<int> lengths;
    if (one) {
        lengths.assign(xs.size(), small_integer(a[3], "page_tokens"));
    } else {
        const Sequence each(a[3], "page_tokens must be an integer or a sequence of integers");
        if (each.size() != xs.size()) fail(PyExc_ValueError, "page_tokens must name a length for each tensor");
        for (Py_ssize_t t = 0; t < each.size(); ++t) lengths.push_back(small_integer(each[t], "page_tokens"));
    }
    c10::Device dev(c10::kCUDA, 0);
    bool seen = false;
    for (Py_ssize_t t = 0; t < xs.size(); ++t) {
        const Tensor &x = tensor(xs[t], "every element");
        require_cuda(x, dev, seen);
        if (x.dim() < 2) fail(PyExc_ValueError, "expected [B, tokens, ...] tensors, got shape " + shape_of(x));
        if (lengths[t] <= 0) fail(PyExc_ValueError, "page_tokens must be positive");
        refuse_tangents(x);
        if (x.requires_grad() && at::GradMode::is_enabled())
            fail(PyExc_RuntimeError, "pages are moved in place: a tensor that requires a gradient cannot be moved with gradients enabled");
        int64_t row = 1;
        for (int64_t d = x.dim() - 1; d >= 2; --d) {
            if (x.size(d) != 1 && x.stride(d) != row) fail(PyExc_ValueError, "the axes behind the tokens must be contiguous");
            row *= x.size(d);
        }
        if (x.size(0) > INT_MAX) fail(PyExc_NotImplementedError, "sizes must fit 32 bits");
        const int64_t size = x.element_size();
        tensors[t] = wa_page_tensor{x.numel() ? x.data_ptr() : nullptr, x.stride(0) * size, x.stride(1) * size, x.size(1), row * size, (int32_t)x.size(0), lengths[t]};
    }
    if (xs.size() == 0) Py_RETURN_NONE;
    c10::cuda::CUDAGuard guard(dev);
    cudaStream_t stream = at::cuda::getCurrentCUDAStream(dev.index()).stream();
    check(f_move_pages(tensors.data(), (int)tensors.size(), dst.data(), src.data(), (int)dst.size(), stream));
    for (Py_ssize_t t = 0; t < xs.size(); ++t) {        // what autograd saved of them before is no longer there
        const Tensor &x = THPVariable_Unpack(xs[t]);
        if (!x.is_inference()) x.unsafeGetTensorImpl()->bump_version();
    }
    Py_RETURN_NONE;
}

// ---- tensor_table(tensors) -> bytes: twelve int64 per tensor -------------------------------------
// address, device index (-1: host), scalar type, dimensions, the first four sizes, the first four strides.  A prompt switch looks
// at some hundred tensors; asked for one attribute at a time from Python that took longer than the copies.
PyObject *tensor_table(PyObject *const *a, Py_ssize_t n) {
    expect_args(n, 1);
    PyObject *seq = PySequence_Fast(a[0], "expected a sequence of tensors");
    if (!seq) throw PyFailure();
    const Py_ssize_t count = PySequence_Fast_GET_SIZE(seq);
    PyObject *out = PyBytes_FromStringAndSize(nullptr, count * 12 * (Py_ssize_t)sizeof(int64_t));
    if (!out) {
        Py_DECREF(seq);
        throw PyFailure();
    }
    int64_t *row = reinterpret_cast<int64_t *>(PyBytes_AS_STRING(out));
    try {
        for (Py_ssize_t i = 0; i < count; ++i, row += 12) {
            const Tensor &t = tensor(PySequence_Fast_GET_ITEM(seq, i), "every element");
            row[0] = reinterpret_cast<int64_t>(t.data_ptr());
            row[1] = t.is_cuda() ? t.device().index() : -1;
            row[2] = (int64_t)t.scalar_type();
            row[3] = t.dim();
            for (int d = 0; d < 4; ++d) {
                row[4 + d] = d < t.dim() ? t.size(d) : 1;
                row[8 + d] = d < t.dim() ? t.stride(d) : 0;
            }
        }
    } catch (...) {
        Py_DECREF(seq);
        Py_DECREF(out);
        throw;
    }
    Py_DECREF(seq);
    return out;
}

// ---- read_on_stream(tensors, stream_id, device_index) -> bool -------------------------------------
// Tells PyTorch's allocator of page-locked memory that the stream reads these host tensors, so that it keeps their memory from the
// next allocation until what the stream carries by then is done, whoever drops them and when: its own copies say so, a copy
// queued by this library does not.  False: some are page-locked by another hand, and only the caller can keep them.
PyObject *read_on_stream(PyObject *const *a, Py_ssize_t n) {
    expect_args(n, 3);
    const c10::Stream stream = c10::Stream::unpack3(integer(a[1]), (c10::DeviceIndex)integer(a[2]), c10::DeviceType::CUDA);
    PyObject *seq = PySequence_Fast(a[0], "expected a sequence of tensors");
    if (!seq) throw PyFailure();
    bool all = true;
    try {
        at::HostAllocator *allocator = at::getHostAllocator(at::kCUDA);
        for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(seq); ++i) {
            const Tensor &t = tensor(PySequence_Fast_GET_ITEM(seq, i), "every element");
            const c10::DataPtr &memory = t.storage().data_ptr();
            if (t.numel() && !allocator->record_event(memory.get(), memory.get_context(), stream) && t.is_pinned()) all = false;
        }
    } catch (...) {
        Py_DECREF(seq);
        throw;
    }
    Py_DECREF(seq);
    return PyBool_FromLong(all);
}

// ---- bind(addresses: dict name -> int, status_word, raise_if_failed) ----------------------------
PyObject *bind(PyObject *const *a, Py_ssize_t n) {
    expect_args(n, 3);
    auto get = [&](const char *name, auto &fn) {
        PyObject *o = PyDict_GetItemString(a[0], name);
        if (!o) fail(PyExc_KeyError, name);
        fn = reinterpret_cast<std::decay_t<decltype(fn)>>(PyLong_AsVoidPtr(o));
    };
    get("wa_last_error", f_last_error);
    get("wa_hsa_workspace_bytes", f_workspace_bytes);
    get("wa_hsa_forward", f_forward);
    get("wa_hsa_status", f_status);
    get("wa_qk_norm_rope", f_rope);
    get("wa_qk_norm_rope_at", f_rope_at);
    get("wa_kv_append_workspace_bytes", f_append_bytes);
    get("wa_kv_append_compress", f_append);
    get("wa_ln_modulate", f_ln);
    get("wa_gated_residual", f_residual);
    get("wa_axial_rope", f_axial);
    get("wa_hkv_move_pages", f_move_pages);
    get("wa_selected_workspace_bytes", f_selected_bytes);
    get("wa_selected_forward", f_selected_forward);
    get("wa_selected_backward", f_selected_backward);
    if (PyErr_Occurred()) throw PyFailure();
    PyObject *torch_module = PyImport_ImportModule("torch");
    py_out_of_memory = torch_module ? PyObject_GetAttrString(torch_module, "OutOfMemoryError") : nullptr;
    Py_XDECREF(torch_module);
    if (!py_out_of_memory) throw PyFailure();
    Py_INCREF(a[1]);
    Py_INCREF(a[2]);
    py_status_word = a[1];
    py_raise_if_failed = a[2];
    Py_RETURN_NONE;
}

template <PyObject *(*F)(PyObject *const *, Py_ssize_t)>
PyObject *entry(PyObject *, PyObject *const *args, Py_ssize_t n) {
    try {
        return F(args, n);
    } catch (const PyFailure &) {
        return nullptr;
    } catch (python_error &e) {
        e.restore();
        return nullptr;
    } catch (const c10::OutOfMemoryError &e) {
        PyErr_SetString(py_out_of_memory, e.what_without_backtrace());
        return nullptr;
    } catch (const c10::Error &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
        return nullptr;
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

#define WA_ENTRY(name) {#name, (PyCFunction)(void (*)(void))entry<name>, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {WA_ENTRY(bind), WA_ENTRY(hsa_forward), WA_ENTRY(run_forward), WA_ENTRY(qk_norm_rope), WA_ENTRY(append_kv), WA_ENTRY(ln_modulate),
                         WA_ENTRY(gated_residual), WA_ENTRY(axial_rope), WA_ENTRY(selected_attention), WA_ENTRY(move_pages), WA_ENTRY(tensor_table), WA_ENTRY(read_on_stream), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) { return PyModule_Create(&module); }
