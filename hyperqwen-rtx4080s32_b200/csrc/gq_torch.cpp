// Native call path of a packed run: the Python extension module `_gq_torch`.
//
// GGUFLinearMethod.apply is called once per linear layer and token step.  Going through the torch custom op and ctypes
// costs 46 us of host time per call on an idle GPU (boxing nine arguments, three of them lists of tensors, a Python
// kernel, two allocations from Python and a ctypes call with fifteen arguments), six times what the GPU needs for a small
// layer.  A Run keeps what does not change between calls — the packed buffer, the descriptor tables, the split per
// row count — and does the call's host work here: output and scratch from torch's caching allocator on the current
// stream, then the C ABI of include/gq_b200.h.
//
// forward() answers None for whatever is not the plain case (dtype, layout, device, autograd, torch modes, tracing, function
// transforms, a call of zero rows); the caller then takes the general path, which also states the errors.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/util/SmallVector.h>
#include <pybind11/pybind11.h>
#include <pybind11/stl.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/core/grad_mode.h>
#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <string>
#include <utility>
#include <vector>
#include "../../include/gq_b200.h"

namespace py = pybind11;

namespace {

const char *error_text(int rc) {
    switch (rc) {
        case GQ_ERR_TYPE: return "unsupported GGML type";
        case GQ_ERR_SHAPE: return "bad shape (K not a multiple of 256, negative size, or M over the limit)";
        case GQ_ERR_ARG: return "bad argument (null or misaligned pointer, inconsistent sizes)";
        case GQ_ERR_WORKSPACE: return "workspace too small";
        case GQ_ERR_CUDA: return "CUDA runtime error";
        case GQ_ERR_LIMIT: return "size beyond a fixed maximum";
        default: return "unknown error";
    }
}
PyObject *g_error = PyExc_RuntimeError;      // GqError of _lib.py, kept for the life of the process

void raise_if(int64_t rc, const char *what) {
    if (rc >= 0) return;
    std::string msg = std::string(what) + " failed (" + std::to_string(rc) + "): " + error_text((int)rc);
    if (rc == GQ_ERR_CUDA) msg += std::string(": ") + gq_last_cuda_error();
    PyErr_SetString(g_error, msg.c_str());
    throw py::error_already_set();
}

// what a call of the C ABI returned, kept until the GIL is held again
struct Status {
    int64_t rc = 0;
    const char *what = "";
    void check() const { raise_if(rc, what); }
};

// Whether nothing stands between a torch call and its kernel on this thread: no dispatch or function mode, no tracer, no
// function transform (vmap, jvp).  Each of them shows in the thread's own dispatch keys or as a function mode.
inline bool plain_thread() {
    const uint64_t keys = c10::impl::tls_local_dispatch_key_set().included_.raw_repr();
    return !(keys & ~c10::default_included_set.raw_repr()) && !at::impl::torch_function_mode_enabled();
}
// Whether a tensor is what its memory says: a dense CUDA tensor with no key beside the usual ones (negative view, zero tensor,
// a transform's or a mode's wrapper)
inline bool plain_tensor(const at::Tensor &t) {
    constexpr c10::DispatchKeySet usual({c10::DispatchKey::CUDA, c10::DispatchKey::AutogradCUDA, c10::DispatchKey::ADInplaceOrView,
                                         c10::DispatchKey::AutocastCUDA});
    return t.is_cuda() && !(t.key_set().raw_repr() & ~usual.raw_repr()) && !t.has_names();
}
inline bool plain_cuda(const at::Tensor &t, int device) { return plain_tensor(t) && t.get_device() == device && !t.requires_grad(); }

// Whether two sets of bf16 rows may share memory: `cols` columns each, rows and row strides of their own.  Rows of one stride that lie beside each
// other, as two column ranges of one buffer do, do not.
inline bool may_overlap(const void *a, int64_t rows_a, int64_t ld_a, const void *b, int64_t rows_b, int64_t ld_b, int64_t cols) {
    const int64_t pa = (int64_t)((uintptr_t)a / 2), pb = (int64_t)((uintptr_t)b / 2);
    if (pa + (rows_a - 1) * ld_a + cols <= pb || pb + (rows_b - 1) * ld_b + cols <= pa) return false;
    if (ld_a != ld_b) return true;
    const int64_t off = ((pb - pa) % ld_a + ld_a) % ld_a;
    return off < cols || ld_a - off < cols;
}

class Run {
  public:
    Run(at::Tensor packed, std::vector<at::Tensor> descs, std::vector<int64_t> splits, std::vector<int64_t> n_outs, std::vector<int64_t> types,
        int64_t nb, std::vector<int64_t> split_of_rows, int64_t decode_rows, int64_t pre_rows)
        : packed_(std::move(packed)), descs_(std::move(descs)), splits_(std::move(splits)), K_(nb * 256), decode_rows_(decode_rows),
          pre_rows_(pre_rows), device_(packed_.get_device()) {
        std::vector<int32_t> t32(types.begin(), types.end());
        raise_if(info_ = gq_run_info((int)t32.size(), t32.data()), "gq_run_info");
        const int order = t32.size() == n_outs.size() ? gq_run_order((int)t32.size(), t32.data(), n_outs.data()) : 0;      // a hint
        raise_if(order, "gq_run_order");
        info_ |= order;
        for (int64_t n : n_outs) n_total_ += n;
        one_ = index_of(1);
        for (int64_t s : split_of_rows) by_rows_.push_back(index_of(s));
        TORCH_CHECK((int64_t)by_rows_.size() > decode_rows_, "split_of_rows covers 0..decode_rows");
    }

    // x [..., K] -> [..., n_total]; None: not the plain case
    PyObject *forward(py::handle x) { return call(x, 0, nullptr, nullptr, nullptr, 0.0f); }
    PyObject *forward_silu_mul(py::handle x) { return call(x, 1, nullptr, nullptr, nullptr, 0.0f); }
    PyObject *forward_add_rms_norm(py::handle x, const at::Tensor &weight, c10::optional<at::Tensor> residual,
                                   c10::optional<at::Tensor> residual_out, double eps) {
        return call(x, 2, &weight, residual.has_value() ? &*residual : nullptr, residual_out.has_value() ? &*residual_out : nullptr, (float)eps);
    }

  private:
    // the table of a split, or of the largest below it that there is (split 1 always is)
    int index_of(int64_t split) const {
        int best = -1;
        for (size_t i = 0; i < splits_.size(); ++i)
            if (splits_[i] <= split && (best < 0 || splits_[i] > splits_[best])) best = (int)i;
        return best < 0 ? 0 : best;
    }
    static PyObject *none() { Py_RETURN_NONE; }

    PyObject *call(py::handle xh, int pre, const at::Tensor *weight, const at::Tensor *residual, const at::Tensor *residual_out, float eps) {
        if (!THPVariable_CheckExact(xh.ptr()) || !plain_thread()) return none();
        const at::Tensor x = THPVariable_Unpack(xh.ptr());      // a reference of its own: the GIL is released below
        const int64_t width = pre == 1 ? 2 * K_ : K_, nd = x.dim();
        if (nd < 1 || !plain_cuda(x, device_) || x.scalar_type() != at::kBFloat16 || x.size(-1) != width || x.stride(-1) != 1) return none();
        int64_t m = 1, ldx = width;
        if (nd == 2) { m = x.size(0); ldx = x.stride(0); if (m == 1 && ldx < width) ldx = width; }
        else { if (!x.is_contiguous()) return none(); for (int64_t i = 0; i + 1 < nd; ++i) m *= x.size(i); }
        if (m <= 0 || n_total_ == 0 || ldx < width) return none();
        if (pre) {
            if (pre == 2) {
                if (!plain_cuda(*weight, device_) || weight->scalar_type() != at::kBFloat16 || weight->numel() != K_ || !weight->is_contiguous()) return none();
                if ((residual == nullptr) != (residual_out == nullptr)) return none();
                if (residual) {
                    for (const at::Tensor *r : {residual, residual_out})
                        if (!plain_cuda(*r, device_) || r->scalar_type() != at::kBFloat16 || r->dim() != 2 || r->size(0) != m || r->size(1) != K_ ||
                            r->stride(1) != 1) return none();
                    if (residual->stride(0) != residual_out->stride(0)) return none();
                }
            }
        }
        const bool wide = m > decode_rows_, apart = pre && m > pre_rows_;       // apart: the op is a launch of its own
        if (apart && residual) {
            // the new residual may take the old one's place; where it shares other memory that the kernel reads, the general path reads all of it first
            const void *out = residual_out->data_ptr();
            const int64_t ld = residual_out->stride(0);
            if (ld < K_ || (out != residual->data_ptr() && may_overlap(out, m, ld, residual->data_ptr(), m, ld, K_)) ||
                may_overlap(out, m, ld, x.data_ptr(), m, ldx, K_) || may_overlap(out, m, ld, weight->data_ptr(), 1, K_, K_)) return none();
        }
        if (wide && !apart && ((ldx & 7) || (reinterpret_cast<uintptr_t>(x.data_ptr()) & 15))) return none();
        at::Tensor y;
        Status status;
        {
            // the allocator and a full launch queue can keep the caller waiting: other Python threads go on meanwhile
            py::gil_scoped_release unlocked;
            status = launch(x, m, ldx, pre, weight, residual, residual_out, eps, y);
        }
        status.check();
        return THPVariable_Wrap(std::move(y));
    }

    // the call itself, without the GIL: output and scratch, then the C ABI
    Status launch(const at::Tensor &x, int64_t m, int64_t ldx, int pre, const at::Tensor *weight, const at::Tensor *residual,
                  const at::Tensor *residual_out, float eps, at::Tensor &y) const {
        const bool wide = m > decode_rows_;
        const void *in = x.data_ptr();
        c10::DataPtr pre_out;
        c10::cuda::CUDAGuard guard((c10::DeviceIndex)device_);
        void *stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device_).stream();
        at::DimVector sizes(x.sizes().begin(), x.sizes().end());
        sizes.back() = n_total_;
        y = at::detail::empty_cuda(sizes, at::kBFloat16, x.device(), c10::nullopt);
        auto *alloc = c10::cuda::CUDACachingAllocator::get();
        if (pre && m > pre_rows_) {
            pre_out = alloc->allocate((size_t)(m * K_ * 2));
            const int rc = gq_pre_op(in, m, K_, ldx, pre, weight ? weight->data_ptr() : nullptr, residual ? residual->data_ptr() : nullptr,
                                     residual_out ? residual_out->data_ptr() : nullptr, residual ? residual->stride(0) : 0, eps, pre_out.get(), K_, stream);
            if (rc < 0) return {rc, "gq_pre_op"};
            in = pre_out.get(); ldx = K_; pre = 0;
        }
        if (wide) {
            const int64_t n_desc = descs_[one_].size(0), need = gq_prefill_workspace_bytes(m, K_, n_total_, n_desc);
            if (need < 0) return {need, "gq_prefill_workspace_bytes"};
            c10::DataPtr ws = alloc->allocate((size_t)need + 1024);
            const uintptr_t base = (reinterpret_cast<uintptr_t>(ws.get()) + 1023) & ~(uintptr_t)1023;
            return {gq_gemm_prefill(in, m, K_, ldx, packed_.data_ptr(), (const int32_t *)descs_[one_].data_ptr(), n_desc, info_, y.data_ptr(),
                                    n_total_, n_total_, (void *)base, need, stream), "gq_gemm_prefill"};
        }
        const int i = by_rows_[m];
        const int split = (int)splits_[i];
        const at::Tensor &d = descs_[i];
        const int64_t need = gq_workspace_bytes(m, K_, n_total_, split);
        if (need < 0) return {need, "gq_workspace_bytes"};
        c10::DataPtr ws = alloc->allocate((size_t)need);
        if (pre)
            return {gq_gemv_grouped_pre(x.data_ptr(), m, K_, ldx, pre, weight ? weight->data_ptr() : nullptr, residual ? residual->data_ptr() : nullptr,
                                        residual_out ? residual_out->data_ptr() : nullptr, residual ? residual->stride(0) : 0, eps, packed_.data_ptr(),
                                        (const int32_t *)d.data_ptr(), d.size(0), split, info_, y.data_ptr(), n_total_, n_total_, ws.get(), need, stream),
                    "gq_gemv_grouped_pre"};
        // 15: nobody reads this workspace's status word, so a small launch may do without the preparation kernel
        return {gq_gemv_grouped_phases(in, m, K_, ldx, packed_.data_ptr(), (const int32_t *)d.data_ptr(), d.size(0), split, info_,
                                       y.data_ptr(), n_total_, n_total_, ws.get(), need, stream, 15), "gq_gemv_grouped"};
    }

    at::Tensor packed_;
    std::vector<at::Tensor> descs_;
    std::vector<int64_t> splits_;
    std::vector<int> by_rows_;       // rows -> index into descs_
    int64_t K_, n_total_ = 0, decode_rows_, pre_rows_;
    int device_, info_ = 0, one_ = 0;
};

// The load-time calls, on arguments that ops.py has checked: device and stream of the tensor, then the C ABI.
void *stream_of(const at::Tensor &t) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)t.get_device()).stream(); }

void repack(const at::Tensor &raw, int64_t n_out, int64_t type, int64_t nb, const at::Tensor &out) {
    Status status;
    {
        py::gil_scoped_release unlocked;
        c10::cuda::CUDAGuard guard((c10::DeviceIndex)raw.get_device());
        status = {gq_repack((int)type, raw.data_ptr(), n_out, nb * 256, raw.stride(0), out.data_ptr(), stream_of(raw)), "gq_repack"};
    }
    status.check();
}
at::Tensor dequantize(const at::Tensor &tiles, int64_t n_out, int64_t k, int64_t type, bool bf16) {
    Status status;
    at::Tensor out;
    {
        py::gil_scoped_release unlocked;
        c10::cuda::CUDAGuard guard((c10::DeviceIndex)tiles.get_device());
        out = at::detail::empty_cuda({n_out, k}, bf16 ? at::kBFloat16 : at::kFloat, tiles.device(), c10::nullopt);
        status = {gq_dequant((int)type, tiles.data_ptr(), n_out, k, out.data_ptr(), bf16 ? 1 : 0, k, stream_of(tiles)), "gq_dequant"};
    }
    status.check();
    return out;
}
// waits for the caller's stream on the tensor's device; one that is being captured has nothing to wait for
void finish(const at::Tensor &t) {
    py::gil_scoped_release unlocked;
    c10::cuda::CUDAGuard guard((c10::DeviceIndex)t.get_device());
    if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None)
        c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)t.get_device()).synchronize();
}
void build_descs(const std::vector<int32_t> &types, const std::vector<int64_t> &n_outs, int64_t k, const std::vector<int32_t> &splits, const at::Tensor &out) {
    Status status;
    {
        py::gil_scoped_release unlocked;
        c10::cuda::CUDAGuard guard((c10::DeviceIndex)out.get_device());
        status = {gq_build_descs_device((int)types.size(), types.data(), n_outs.data(), k, (int)splits.size(), splits.data(), (int32_t *)out.data_ptr(),
                                        stream_of(out)), "gq_build_descs_device"};
    }
    status.check();
}

// rows `ids` of a raw table -> weights; None: not the plain case
PyObject *dequantize_rows(py::handle rawh, int64_t type, py::handle idsh, bool bf16) {
    if (!THPVariable_CheckExact(rawh.ptr()) || !THPVariable_CheckExact(idsh.ptr()) || !plain_thread()) Py_RETURN_NONE;
    const at::Tensor raw = THPVariable_Unpack(rawh.ptr()), ids = THPVariable_Unpack(idsh.ptr());
    const int B = gq_bytes_per_256((int)type);
    if (!plain_tensor(raw) || !plain_tensor(ids) || raw.scalar_type() != at::kByte || raw.dim() != 2 || raw.stride(1) != 1 || raw.stride(0) < raw.size(1) || raw.size(0) == 0 || B == 0 || raw.size(1) == 0 ||
        raw.size(1) % B || ids.get_device() != raw.get_device() || !ids.is_contiguous() || ids.numel() == 0 ||
        (ids.scalar_type() != at::kLong && ids.scalar_type() != at::kInt)) Py_RETURN_NONE;
    const int64_t K = raw.size(1) / B * 256;
    at::DimVector sizes(ids.sizes().begin(), ids.sizes().end());
    sizes.push_back(K);
    at::Tensor out;
    Status status;
    {
        py::gil_scoped_release unlocked;
        c10::cuda::CUDAGuard guard((c10::DeviceIndex)raw.get_device());
        out = at::detail::empty_cuda(sizes, bf16 ? at::kBFloat16 : at::kFloat, raw.device(), c10::nullopt);
        status = {gq_dequant_rows((int)type, raw.data_ptr(), raw.size(0), K, raw.stride(0), ids.data_ptr(), ids.scalar_type() == at::kLong ? 8 : 4,
                                  ids.numel(), out.data_ptr(), bf16 ? 1 : 0, K, stream_of(raw)), "gq_dequant_rows"};
    }
    status.check();
    return THPVariable_Wrap(std::move(out));
}

// ---- the operators beside the quantized layers ---------------------------------------------------------
// Arguments are checked here in full (shapes and types first, then devices and memory), then handed to the C ABI on the current stream of their device.  ops.py comes here directly on a
// plain thread only; inside a mode, a tracer or a transform it calls the registered op, which the dispatcher brings here.

[[noreturn]] void refuse(const char *op, const std::string &why) {
    PyErr_SetString(g_error, (std::string(op) + ": " + why).c_str());
    throw py::error_already_set();
}
std::string shape_of(const at::Tensor &t) {
    std::string s = "[";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + "] " + c10::toString(t.scalar_type());
}
// What all tensors of a call have in common: memory of one CUDA device that is what it says, and no gradient to keep
class Checked {
  public:
    explicit Checked(const char *op) : op_(op) {}
    void need(bool ok, const char *what) const { if (!ok) refuse(op_, what); }
    void shaped(const at::Tensor &t, at::ScalarType type, std::initializer_list<int64_t> sizes, const char *what) const {      // -1: any size
        bool ok = t.scalar_type() == type && t.dim() == (int64_t)sizes.size();
        int64_t i = 0;
        for (int64_t n : sizes) { ok = ok && (n < 0 || t.size(i) == n); ++i; }
        if (!ok) refuse(op_, std::string(what) + ", got " + shape_of(t));
    }
    void add(const at::Tensor &t) { if (count_ < 16) all_[count_++] = &t; }
    void devices() const {
        for (int i = 0; i < count_; ++i)
            if (all_[i]->_fw_grad(0).defined()) refuse(op_, "has no forward derivative: call it with the primals of its inputs");
        for (int i = 0; i < count_; ++i) {
            if (!all_[i]->is_cuda()) refuse(op_, "takes CUDA tensors (there is no CPU path)");
            if (!plain_tensor(*all_[i])) refuse(op_, "takes tensors that are what their memory says (no negative views, wrappers or transforms)");
            if (all_[i]->get_device() != all_[0]->get_device()) refuse(op_, "takes tensors of one device");
            if (all_[i]->requires_grad() && at::GradMode::is_enabled()) refuse(op_, "has no backward pass: call it under torch.no_grad(), or detach its inputs");
        }
    }
  private:
    const char *op_;
    const at::Tensor *all_[16];
    int count_ = 0;
};
inline bool on16(const at::Tensor &t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }
// elements from a tensor's first to behind its last
inline int64_t extent(const at::Tensor &t) {
    int64_t n = 1;
    for (int64_t i = 0; i < t.dim(); ++i) { if (t.size(i) == 0) return 0; n += (t.size(i) - 1) * t.stride(i); }
    return n;
}
using Dims = c10::SmallVector<std::pair<int64_t, int64_t>, 4>;          // stride, size
// A tensor's dimensions of more than one element, the longest stride first; false if two of its elements may be one (a stride shorter than what lies inside it)
bool nested(const at::Tensor &t, Dims &dims) {
    for (int64_t i = 0; i < t.dim(); ++i)
        if (t.size(i) > 1) dims.emplace_back(t.stride(i), t.size(i));
    std::sort(dims.rbegin(), dims.rend());
    int64_t inside = 1;
    for (size_t i = dims.size(); i-- > 0;) {
        if (dims[i].first < inside) return false;
        inside += (dims[i].second - 1) * dims[i].first;
    }
    return true;
}
bool own_memory(const at::Tensor &t) {
    Dims dims;
    return t.numel() == 0 || nested(t, dims);
}
// whether some difference of two indexes of these dimensions is `off` elements
bool apart_by(const Dims &dims, size_t i, int64_t off) {
    if (i == dims.size()) return off == 0;
    const int64_t down = off / dims[i].first - (off % dims[i].first < 0);
    for (int64_t d : {down, down + 1})           // what is left has to be less than a stride
        if (std::abs(d) < dims[i].second && apart_by(dims, i + 1, off - d * dims[i].first)) return true;
    return false;
}
// whether two caches of one shape share an element; exact where their strides are the same, else whether they start at one place
bool same_cells(const at::Tensor &u, const at::Tensor &v) {
    if (u.numel() == 0 || u.data_ptr() == v.data_ptr()) return u.numel() != 0;
    Dims du, dv;
    if (!nested(u, du) || !nested(v, dv) || du != dv) return false;
    return apart_by(du, 0, ((const char *)v.data_ptr() - (const char *)u.data_ptr()) / u.element_size());
}
// whether two tensors' ranges of memory meet; of rows with unit stride, whether the rows do
bool meet(const at::Tensor &u, const at::Tensor &v) {
    const char *a = (const char *)u.data_ptr(), *b = (const char *)v.data_ptr();
    const int64_t na = extent(u) * u.element_size(), nb = extent(v) * v.element_size();
    if (na == 0 || nb == 0 || a + na <= b || b + nb <= a) return false;
    if (u.dim() == 2 && v.dim() == 2 && u.scalar_type() == at::kBFloat16 && v.scalar_type() == at::kBFloat16 && u.size(1) == v.size(1) && u.size(0) > 1 && v.size(0) > 1 &&
        u.stride(0) >= u.size(1) && v.stride(0) >= v.size(1))
        return may_overlap(a, u.size(0), u.stride(0), b, v.size(0), v.stride(0), u.size(1));
    return true;
}
// rows that start at multiples of 16 bytes: the tensor itself, or a copy
at::Tensor rows16(const at::Tensor &t) {
    bool ok = t.stride(-1) == 1 && on16(t);
    for (int64_t i = 0; ok && i + 1 < t.dim(); ++i) ok = t.size(i) == 1 || (t.stride(i) % 8 == 0 && t.stride(i) >= t.size(-1));
    return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}
// elements between rows; one row has none, and any number will do
inline int64_t row_stride(const at::Tensor &t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
inline int id_bytes(const at::Tensor &t) { return t.scalar_type() == at::kLong ? 8 : 4; }
inline bool integers(const at::Tensor &t) { return t.scalar_type() == at::kLong || t.scalar_type() == at::kInt; }
// scratch of a call: from torch's allocator, on the current stream
c10::DataPtr scratch(int64_t bytes) { return bytes > 0 ? c10::cuda::CUDACachingAllocator::get()->allocate((size_t)bytes) : c10::DataPtr(); }

at::Tensor low_rank_add(const at::Tensor &base0, const at::Tensor &x0, const at::Tensor &a, const at::Tensor &b, const at::Tensor &scales, const at::Tensor &ids0,
                        const std::vector<int64_t> &n_outs, c10::optional<at::Tensor> out0) {
    Checked c("low_rank_add");
    gq_low_rank_args p{};
    c.need(!n_outs.empty() && n_outs.size() <= GQ_MAX_DEVICE_SHARDS, "n_outs names one to eight shards");
    int64_t n = 0;
    for (size_t s = 0; s < n_outs.size(); ++s) { c.need(n_outs[s] >= 0, "n_outs holds the columns of each shard"); n += p.n_outs[s] = n_outs[s]; }
    c.shaped(x0, at::kBFloat16, {-1, -1}, "x is bf16 [M, K]");
    const int64_t m = x0.size(0), k = x0.size(1), shards = (int64_t)n_outs.size();
    c.need(k > 0 && k % 256 == 0, "K is a multiple of 256");
    c.shaped(base0, at::kBFloat16, {m, n}, "base is bf16 [M, sum(n_outs)]");
    c.shaped(b, at::kBFloat16, {-1, n, -1}, "b is bf16 [adapters, sum(n_outs), rank]");
    const int64_t bank = b.size(0), rank = b.size(2);
    c.need(bank > 0 && rank > 0 && rank % 8 == 0 && rank <= GQ_MAX_RANK, "the rank is a multiple of 8 up to 128, of one adapter or more");
    c.shaped(a, at::kBFloat16, {bank, shards * rank, k}, "a is bf16 [adapters, shards * rank, K]");
    c.shaped(scales, at::kFloat, {bank, shards}, "scales is float32 [adapters, shards]");
    c.need(ids0.dim() == 1 && ids0.size(0) == m && integers(ids0), "ids is int32 or int64 [M]");
    c.need(a.is_contiguous() && b.is_contiguous() && scales.is_contiguous(), "a, b and scales are contiguous");
    if (out0.has_value()) {
        c.shaped(*out0, at::kBFloat16, {m, n}, "out is bf16 [M, sum(n_outs)]");
        c.need(m == 0 || n == 0 || (out0->stride(1) == 1 && (m == 1 || out0->stride(0) >= n)), "out has unit column stride and rows of their own");
    }
    for (const at::Tensor *t : {&x0, &base0, &a, &b, &scales, &ids0}) c.add(*t);
    if (out0.has_value()) c.add(*out0);
    c.devices();
    c.need(on16(a) && on16(b), "a and b start at multiples of 16 bytes");
    if (out0.has_value() && m > 0 && n > 0) {
        const bool in_place = out0->data_ptr() == base0.data_ptr() && base0.stride(1) == 1 && row_stride(*out0) == row_stride(base0);
        c.need(in_place || !meet(*out0, base0), "out is base itself or shares no memory with it");
        for (const at::Tensor *t : {&x0, &a, &b, &scales, &ids0}) c.need(!meet(*out0, *t), "out shares no memory with an input other than base");
    }
    Status status;
    at::Tensor out;
    {
        py::gil_scoped_release unlocked;
        c10::cuda::CUDAGuard guard((c10::DeviceIndex)x0.get_device());
        out = out0.has_value() ? *out0 : at::detail::empty_cuda({m, n}, at::kBFloat16, x0.device(), c10::nullopt);
        if (m > 0 && n > 0) {
            const at::Tensor x = rows16(x0), ids = ids0.contiguous(), base = base0.stride(1) == 1 && (m == 1 || base0.stride(0) >= n) ? base0 : base0.contiguous();
            p.base = base.data_ptr(); p.x = x.data_ptr(); p.a = a.data_ptr(); p.b = b.data_ptr(); p.scales = (const float *)scales.data_ptr();
            p.ids = ids.data_ptr(); p.out = out.data_ptr(); p.M = m; p.K = k; p.ld_base = row_stride(base); p.ldx = row_stride(x); p.ld_out = row_stride(out);
            p.n_shards = (int)shards; p.n_adapters = (int)bank; p.rank = (int)rank; p.ids_bytes = id_bytes(ids);
            p.workspace_bytes = gq_low_rank_workspace_bytes(&p);
            const c10::DataPtr ws = scratch(p.workspace_bytes);
            p.workspace = ws.get();
            status = p.workspace_bytes < 0 ? Status{p.workspace_bytes, "gq_low_rank_workspace_bytes"} : Status{gq_low_rank_add(&p, stream_of(x)), "gq_low_rank_add"};
        }
    }
    status.check();
    return out;
}

// the pages of a cache, [pages, rows, kv heads, head_dim] by strides
void take_pages(const Checked &c, const at::Tensor &t, int64_t kv_heads, int64_t dim, const char *what, int64_t (&strides)[3]) {
    c.shaped(t, at::kBFloat16, {-1, -1, kv_heads, dim}, what);
    c.need(t.size(1) > 0, "a page holds one row or more");
    c.need(t.numel() == 0 || t.stride(3) == 1, "the pages' head_dim has unit stride");
    for (int i = 0; i < 3; ++i) {
        c.need(t.size(i) <= 1 || (t.stride(i) % 8 == 0 && t.stride(i) >= dim), "the pages' rows and heads start at multiples of 16 bytes, each in memory of its own");
        strides[i] = t.size(i) > 1 ? t.stride(i) : 0;
    }
}

// Both forms: with a cache given (all of k_pages, v_pages, slots) keys and values go there and q comes back, without one q and k
py::object norm_heads(const at::Tensor &qkv0, const at::Tensor &positions0, const at::Tensor &inv_freq, int64_t n_heads, int64_t n_kv_heads, int64_t head_dim,
                        c10::optional<at::Tensor> q_norm, c10::optional<at::Tensor> k_norm, double eps, double amplitude, bool interleaved, bool gated,
                        c10::optional<at::Tensor> k_pages, c10::optional<at::Tensor> v_pages, c10::optional<at::Tensor> slots0) {
    const bool store = k_pages.has_value();
    Checked c(store ? "qk_norm_rope_store" : "qk_norm_rope");
    gq_head_norm_args p{};
    c.need(n_heads > 0 && n_kv_heads > 0 && n_heads <= 16384 && n_kv_heads <= 16384, "one or more heads of queries and of keys");
    c.need(head_dim >= 8 && head_dim % 8 == 0 && head_dim <= 512, "head_dim is a multiple of 8 up to 512");
    const int64_t width = (n_heads * (gated ? 2 : 1) + 2 * n_kv_heads) * head_dim;
    c.shaped(qkv0, at::kBFloat16, {-1, width}, "qkv is bf16 [T, all heads of q (each with its gate if gated), k and v]");
    const int64_t t = qkv0.size(0);
    c.need(positions0.dim() == 1 && positions0.size(0) == t && integers(positions0), "positions is int32 or int64 [T]");
    c.shaped(inv_freq, at::kDouble, {-1}, "inv_freq is float64 [rotary_dim / 2]");
    c.need(inv_freq.is_contiguous() && 2 * inv_freq.numel() <= head_dim, "inv_freq is contiguous, of at most head_dim / 2 values");
    for (auto *w : {&q_norm, &k_norm})
        if (w->has_value()) {
            c.shaped(**w, at::kBFloat16, {head_dim}, "a norm weight is bf16 [head_dim]");
            c.need((*w)->is_contiguous(), "a norm weight is contiguous");
        }
    if (store) {
        take_pages(c, *k_pages, n_kv_heads, head_dim, "k_pages is bf16 [pages, rows, kv heads, head_dim]", p.k_strides);
        take_pages(c, *v_pages, n_kv_heads, head_dim, "v_pages is bf16 [pages, rows, kv heads, head_dim]", p.v_strides);
        c.need(k_pages->size(0) == v_pages->size(0) && k_pages->size(1) == v_pages->size(1), "k_pages and v_pages hold the same pages");
        c.need(own_memory(*k_pages) && own_memory(*v_pages), "the pages' rows and heads each have memory of their own");
        c.need(!same_cells(*k_pages, *v_pages), "keys and values have pages of their own");
        c.need(slots0->dim() == 1 && slots0->size(0) == t && integers(*slots0), "slots is int32 or int64 [T]");
    }
    for (const at::Tensor *x : {&qkv0, &positions0, &inv_freq}) c.add(*x);
    for (auto *x : {&q_norm, &k_norm, &k_pages, &v_pages, &slots0})
        if (x->has_value()) c.add(**x);
    c.devices();
    if (store) {
        c.need(on16(*k_pages) && on16(*v_pages), "the pages start at multiples of 16 bytes");
        for (auto *pages : {&*k_pages, &*v_pages}) {
            for (const at::Tensor *x : std::initializer_list<const at::Tensor *>{&qkv0, &positions0, &inv_freq, &*slots0}) c.need(!meet(*pages, *x), "the pages share no memory with the other arguments");
            for (auto *w : {&q_norm, &k_norm})
                if (w->has_value()) c.need(!meet(*pages, **w), "the pages share no memory with the other arguments");
        }
    }
    Status status;
    at::Tensor q, k;
    {
        py::gil_scoped_release unlocked;
        c10::cuda::CUDAGuard guard((c10::DeviceIndex)qkv0.get_device());
        q = at::detail::empty_cuda({t, n_heads, head_dim}, at::kBFloat16, qkv0.device(), c10::nullopt);
        if (!store) k = at::detail::empty_cuda({t, n_kv_heads, head_dim}, at::kBFloat16, qkv0.device(), c10::nullopt);
        if (t > 0) {
            const at::Tensor qkv = rows16(qkv0), positions = positions0.contiguous(), slots = store ? slots0->contiguous() : at::Tensor();
            auto weight = [](const c10::optional<at::Tensor> &w) { return !w.has_value() ? at::Tensor() : on16(*w) ? *w : w->clone(); };
            const at::Tensor wq = weight(q_norm), wk = weight(k_norm);
            p.qkv = qkv.data_ptr(); p.positions = positions.data_ptr(); p.inv_freq = (const double *)inv_freq.data_ptr();
            p.q_norm = wq.defined() ? wq.data_ptr() : nullptr; p.k_norm = wk.defined() ? wk.data_ptr() : nullptr;
            p.q_out = q.data_ptr(); p.k_out = store ? nullptr : k.data_ptr();
            p.T = t; p.ld_qkv = row_stride(qkv);
            p.n_heads = (int)n_heads; p.n_kv_heads = (int)n_kv_heads; p.head_dim = (int)head_dim; p.rotary_dim = (int)(2 * inv_freq.numel());
            p.positions_bytes = id_bytes(positions); p.interleaved = interleaved; p.gated = gated; p.eps = (float)eps; p.amplitude = (float)amplitude;
            if (store) {
                p.k_pages = k_pages->data_ptr(); p.v_pages = v_pages->data_ptr(); p.slots = slots.data_ptr(); p.slots_bytes = id_bytes(slots);
                p.n_pages = k_pages->size(0); p.page_size = (int)k_pages->size(1);
            }
            status = {gq_head_norm_rope(&p, stream_of(qkv)), "gq_head_norm_rope"};
        }
    }
    status.check();
    return store ? py::cast(q) : py::object(py::make_tuple(q, k));
}

py::object qk_norm_rope(const at::Tensor &qkv, const at::Tensor &positions, const at::Tensor &inv_freq, int64_t n_heads, int64_t n_kv_heads, int64_t head_dim, c10::optional<at::Tensor> q_norm,
                        c10::optional<at::Tensor> k_norm, double eps, double amplitude, bool interleaved, bool gated) {
    return norm_heads(qkv, positions, inv_freq, n_heads, n_kv_heads, head_dim, q_norm, k_norm, eps, amplitude, interleaved, gated, c10::nullopt, c10::nullopt, c10::nullopt);
}
py::object qk_norm_rope_store(const at::Tensor &qkv, const at::Tensor &positions, const at::Tensor &inv_freq, int64_t n_heads, int64_t n_kv_heads, int64_t head_dim, c10::optional<at::Tensor> q_norm,
                              c10::optional<at::Tensor> k_norm, double eps, double amplitude, bool interleaved, bool gated, c10::optional<at::Tensor> k_pages, c10::optional<at::Tensor> v_pages,
                              c10::optional<at::Tensor> slots) {
    Checked("qk_norm_rope_store").need(k_pages.has_value() && v_pages.has_value() && slots.has_value(), "k_pages, v_pages and slots are all given");
    return norm_heads(qkv, positions, inv_freq, n_heads, n_kv_heads, head_dim, q_norm, k_norm, eps, amplitude, interleaved, gated, k_pages, v_pages, slots);
}

at::Tensor paged_attention(const at::Tensor &q0, const at::Tensor &k_pages, const at::Tensor &v_pages, const at::Tensor &table0, const at::Tensor &lens0,
                           c10::optional<at::Tensor> q_starts0, c10::optional<double> scale, c10::optional<at::Tensor> gate0, c10::optional<at::Tensor> out0) {
    Checked c("paged_attention");
    gq_attention_args p{};
    c.shaped(q0, at::kBFloat16, {-1, -1, -1}, "q is bf16 [T, heads, head_dim]");
    const int64_t t = q0.size(0), heads = q0.size(1), dim = q0.size(2);
    c.need(dim == 64 || dim == 128 || dim == 256, "head_dim is 64, 128 or 256");
    take_pages(c, k_pages, -1, dim, "k_pages is bf16 [pages, rows, kv heads, head_dim]", p.k_strides);
    const int64_t kv_heads = k_pages.size(2);
    take_pages(c, v_pages, kv_heads, dim, "v_pages is bf16 [pages, rows, kv heads, head_dim]", p.v_strides);
    c.need(k_pages.size(0) == v_pages.size(0) && k_pages.size(1) == v_pages.size(1), "k_pages and v_pages hold the same pages");
    c.need(heads > 0 && heads <= 65535 && kv_heads > 0 && heads % kv_heads == 0, "the query heads are a multiple of the key-value heads");
    c.shaped(table0, at::kInt, {-1, -1}, "page_table is int32 [sequences, pages of the longest]");
    const int64_t seqs = table0.size(0);
    c.shaped(lens0, at::kInt, {seqs}, "lens is int32 [sequences]");
    if (q_starts0.has_value()) c.shaped(*q_starts0, at::kInt, {seqs + 1}, "q_starts is int32 [sequences + 1]");
    else c.need(seqs ? t % seqs == 0 : t == 0, "without q_starts every sequence has the same number of tokens");
    for (auto *x : {&gate0, &out0})
        if (x->has_value()) {
            c.shaped(**x, at::kBFloat16, {t, heads, dim}, x == &gate0 ? "gate is bf16, of q's shape" : "out is bf16, of q's shape");
            c.need((*x)->numel() == 0 || (*x)->stride(2) == 1, "gate and out have unit stride along head_dim");
        }
    if (out0.has_value())
        c.need((t <= 1 || out0->stride(0) >= dim) && (heads <= 1 || out0->stride(1) >= dim) && own_memory(*out0), "out's rows and heads have memory of their own");
    for (const at::Tensor *x : {&q0, &k_pages, &v_pages, &table0, &lens0}) c.add(*x);
    for (auto *x : {&q_starts0, &gate0, &out0})
        if (x->has_value()) c.add(**x);
    c.devices();
    c.need(on16(k_pages) && on16(v_pages), "the pages start at multiples of 16 bytes");
    if (out0.has_value()) {
        for (const at::Tensor *x : {&q0, &k_pages, &v_pages, &table0, &lens0}) c.need(!meet(*out0, *x), "out shares no memory with an input");
        for (auto *x : {&q_starts0, &gate0})
            if (x->has_value()) c.need(!meet(*out0, **x), "out shares no memory with an input");
    }
    Status status;
    at::Tensor out;
    {
        py::gil_scoped_release unlocked;
        c10::cuda::CUDAGuard guard((c10::DeviceIndex)q0.get_device());
        if (out0.has_value()) out = *out0;
        else {
            out = at::detail::empty_cuda({t, heads, dim}, at::kBFloat16, q0.device(), c10::nullopt);
            if (q_starts0.has_value()) out.zero_();                 // rows behind the last sequence
        }
        if (t > 0 && seqs > 0) {
            const at::Tensor q = rows16(q0), lens = lens0.contiguous(), starts = q_starts0.has_value() ? q_starts0->contiguous() : at::Tensor();
            const at::Tensor table = table0.size(1) == 0 || (table0.stride(1) == 1 && (seqs == 1 || table0.stride(0) >= table0.size(1))) ? table0 : table0.contiguous();
            p.q = q.data_ptr(); p.k_pages = k_pages.data_ptr(); p.v_pages = v_pages.data_ptr(); p.page_table = (const int32_t *)table.data_ptr();
            p.lens = (const int32_t *)lens.data_ptr(); p.q_starts = starts.defined() ? (const int32_t *)starts.data_ptr() : nullptr; p.out = out.data_ptr();
            p.T = t; p.n_seqs = seqs; p.table_width = table.size(1); p.ld_table = row_stride(table); p.n_pages = k_pages.size(0); p.page_size = (int)k_pages.size(1);
            p.n_heads = (int)heads; p.n_kv_heads = (int)kv_heads; p.head_dim = (int)dim;
            p.scale = scale.has_value() ? (float)*scale : 1.0f / std::sqrt((float)dim);
            auto strides = [](const at::Tensor &x, int64_t (&s)[2]) { for (int i = 0; i < 2; ++i) s[i] = x.size(i) > 1 ? x.stride(i) : 0; };
            strides(q, p.q_strides); strides(out, p.out_strides);
            if (gate0.has_value()) { p.gate = gate0->data_ptr(); strides(*gate0, p.gate_strides); }
            p.workspace_bytes = gq_attention_workspace_bytes(&p);
            const c10::DataPtr ws = scratch(p.workspace_bytes);
            p.workspace = ws.get();
            status = p.workspace_bytes < 0 ? Status{p.workspace_bytes, "gq_attention_workspace_bytes"} : Status{gq_paged_attention(&p, stream_of(q)), "gq_paged_attention"};
        }
    }
    status.check();
    return out;
}

}  // namespace

PYBIND11_MODULE(_gq_torch, m) {
    m.def("set_error_type", [](py::object e) { g_error = e.release().ptr(); });
    m.def("repack", &repack);
    m.def("dequantize", &dequantize);
    m.def("build_descs", &build_descs);
    m.def("finish", &finish);
    m.def("dequantize_rows", [](py::handle raw, int64_t type, py::handle ids, bool bf16) {
        return py::reinterpret_steal<py::object>(dequantize_rows(raw, type, ids, bf16));
    });
    m.def("plain_thread", &plain_thread);
    m.def("low_rank_add", &low_rank_add);
    m.def("qk_norm_rope", &qk_norm_rope);
    m.def("qk_norm_rope_store", &qk_norm_rope_store);
    m.def("paged_attention", &paged_attention);
    py::class_<Run>(m, "Run")
        .def(py::init<at::Tensor, std::vector<at::Tensor>, std::vector<int64_t>, std::vector<int64_t>, std::vector<int64_t>, int64_t, std::vector<int64_t>,
                      int64_t, int64_t>())
        .def("forward", [](Run &r, py::handle x) { return py::reinterpret_steal<py::object>(r.forward(x)); })
        .def("forward_silu_mul", [](Run &r, py::handle x) { return py::reinterpret_steal<py::object>(r.forward_silu_mul(x)); })
        .def("forward_add_rms_norm", [](Run &r, py::handle x, const at::Tensor &w, c10::optional<at::Tensor> res, c10::optional<at::Tensor> out, double eps) {
            return py::reinterpret_steal<py::object>(r.forward_add_rms_norm(x, w, res, out, eps));
        });
}
