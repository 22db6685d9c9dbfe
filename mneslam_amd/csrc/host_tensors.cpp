// host_tensors.cpp -- the host side of optim.adamw_step: lists of torch tensors checked and written into the table of
// mne_adamw_step.  A list of several hundred small tensors is bound by this loop and not by the GPU: in python it costs 2.5 us a
// tensor (about thirty attribute reads), here 0.1 us.
#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <map>
#include <vector>

#include "mneslam_hip.h"

namespace {

typedef std::vector<at::Tensor> Tensors;
typedef int (*adamw_step_fn)(const int64_t*, int64_t, const mne_adamw_cfg_t*, const mne_clock_t*, void*);

int type_code(at::ScalarType t) {
    return t == at::kFloat ? MNE_T_F32 : t == at::kBFloat16 ? MNE_T_BF16 : t == at::kHalf ? MNE_T_F16 : -1;
}

// equal strides in every dimension that has more than one entry (the shapes are equal)
bool laid_out_alike(const at::Tensor& a, const at::Tensor& b) {
    for (int64_t d = 0; d < a.dim(); ++d)
        if (a.size(d) > 1 && a.stride(d) != b.stride(d)) return false;
    return true;
}

int adamw_step(uintptr_t fn, const Tensors& params, const Tensors& grads, const Tensors& exp_avgs, const Tensors& exp_avg_sqs,
               const c10::optional<Tensors>& scales, const c10::optional<std::vector<int64_t>>& ordinals, double lr, double beta1,
               double beta2, double eps, double weight_decay, int64_t step, int64_t seed, bool zero_grad, uintptr_t clock,
               uintptr_t stream, bool on_host) {
    const size_t n = params.size();
    const bool small = scales.has_value();
    if (grads.size() != n || exp_avgs.size() != n || exp_avg_sqs.size() != n || (small && scales->size() != n) ||
        (ordinals && ordinals->size() != n))
        throw py::value_error("adamw_step: lists of different lengths");
    if (!n) return 0;
    const at::Device dev = params[0].device();
    if (dev.type() != (on_host ? at::kCPU : at::kCUDA))
        throw py::value_error("adamw_step: tensors on " + dev.str() + ": the HIP kernels need them on the GPU");
    std::map<std::pair<int, int>, std::vector<int64_t>> tables;          // by the types of parameter and gradient
    std::vector<std::pair<int64_t, int64_t>> ranges;
    Tensors keep;
    c10::NoGradGuard no_grad;
    for (size_t i = 0; i < n; ++i) {
        const at::Tensor &p = params[i], &m = exp_avgs[i], &v = exp_avg_sqs[i];
        at::Tensor g = grads[i];
        for (const at::Tensor* t : {&p, (const at::Tensor*)&g, &m, &v, small ? &(*scales)[i] : &p}) {
            if (!t->defined() || t->layout() != at::kStrided) throw py::value_error("adamw_step: sparse or undefined tensors are not supported");
            if (t->device() != dev) throw py::value_error("adamw_step: tensors on " + dev.str() + " and on " + t->device().str());
        }
        const int pt = type_code(p.scalar_type()), gt = type_code(g.scalar_type());
        if (pt < 0 || gt < 0 || !(gt == pt || gt == MNE_T_F32 || pt == MNE_T_F32))
            throw py::type_error(std::string("adamw_step: parameter ") + c10::toString(p.scalar_type()) + " with gradient " +
                                 c10::toString(g.scalar_type()) + " is not supported");
        if (m.scalar_type() != (small ? at::kChar : at::kFloat) || v.scalar_type() != (small ? at::kByte : at::kFloat))
            throw py::type_error(small ? "adamw_step: 8-bit moments must be int8 and uint8" : "adamw_step: moments must be float32");
        if (g.sizes() != p.sizes() || m.sizes() != p.sizes() || v.sizes() != p.sizes())
            throw py::value_error("adamw_step: gradient and moments need their parameter's shape");
        const int64_t count = p.numel(), ordinal = ordinals ? (*ordinals)[i] : (int64_t)i;
        if (ordinal < 0 || ordinal > 0xFFFFFFFFll) throw py::value_error("adamw_step: ordinals are numbers of 32 bits");
        if (small) {
            const at::Tensor& s = (*scales)[i];
            if (s.scalar_type() != at::kFloat || s.dim() != 2 || s.size(0) != (count + 255) / 256 || s.size(1) != 2 || !s.is_contiguous())
                throw py::value_error("adamw_step: scales must be contiguous float32 [ceil(n / 256), 2]");
        }
        if (!count) continue;
        if (!p.is_non_overlapping_and_dense()) throw py::value_error("adamw_step: parameters must be dense");
        if (!laid_out_alike(m, p) || !laid_out_alike(v, p)) throw py::value_error("adamw_step: moments must be laid out like their parameter");
        if (!laid_out_alike(g, p)) {
            if (zero_grad) throw py::value_error("adamw_step: zero_grad needs gradients laid out like their parameters");
            g = at::empty_like(p, p.options().dtype(g.scalar_type())).copy_(g);
            keep.push_back(g);
        }
        const int64_t at = (int64_t)p.data_ptr();
        ranges.emplace_back(at, at + count * (int64_t)p.element_size());
        std::vector<int64_t>& table = tables[{pt, gt}];
        const int64_t row[7] = {at, (int64_t)g.data_ptr(), (int64_t)m.data_ptr(), (int64_t)v.data_ptr(),
                                small ? (int64_t)(*scales)[i].data_ptr() : 0, count, ordinal};
        table.insert(table.end(), row, row + 7);
    }
    std::sort(ranges.begin(), ranges.end());
    for (size_t i = 1; i < ranges.size(); ++i)
        if (ranges[i].first < ranges[i - 1].second) throw py::value_error("adamw_step: parameters overlap (the same one twice?)");
    for (const auto& t : tables) {
        mne_adamw_cfg_t cfg = {};
        cfg.lr = lr; cfg.beta1 = beta1; cfg.beta2 = beta2; cfg.eps = eps; cfg.weight_decay = weight_decay;
        cfg.step = (int32_t)step; cfg.state_bits = small ? 8 : 32; cfg.p_type = t.first.first; cfg.g_type = t.first.second;
        cfg.zero_grad = zero_grad; cfg.seed = (uint32_t)seed;
        const int rc = ((adamw_step_fn)fn)(t.second.data(), (int64_t)t.second.size() / 7, &cfg, (const mne_clock_t*)clock, (void*)stream);
        if (rc) return rc;
    }
    for (const at::Tensor& p : params)              // what autograd has saved of a parameter is out of date, as after p.add_()
        if (!p.is_inference()) p.unsafeGetTensorImpl()->bump_version();
    return 0;
}

}  // namespace

PYBIND11_MODULE(_host_tensors, m) {
    m.def("adamw_step", &adamw_step);
    m.attr("ABI_VERSION") = MNE_ABI_VERSION;
}
