// host_tensors.cpp -- the host side of optim.adamw_step and of routing: torch tensors checked and handed to the C ABI, and the autograd
// nodes of the row movements.  Calls that take a few microseconds on the GPU are bound by what runs before and between them: a list of
// several hundred tensors costs 2.5 us a tensor in python (about thirty attribute reads) and 0.25 us here, and a backward pass through two
// python nodes 140 us and 30 us.
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <map>
#include <unordered_set>
#include <vector>

#include "mneslam_hip.h"

namespace {

typedef std::vector<at::Tensor> Tensors;
using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

// The entry points of the library that the package has loaded (a table by value: a node of a graph keeps the one it was made with).
struct Library {
    decltype(&mne_last_error) last_error;
    decltype(&mne_adamw_step) adamw_step;
    decltype(&mne_adamw_moments) adamw_moments;
    decltype(&mne_expert_sort_workspace_bytes) sort_bytes;
    decltype(&mne_expert_sort) sort;
    decltype(&mne_expert_dispatch) dispatch;
    decltype(&mne_expert_combine) combine;
    decltype(&mne_expert_combine_backward) combine_backward;
    int64_t on_host;
};
Library g_lib;

void bind(const std::vector<uintptr_t>& addresses, bool on_host) {
    if (addresses.size() * sizeof(uintptr_t) + sizeof(int64_t) != sizeof(Library)) throw py::value_error("bind: wrong number of entry points");
    memcpy((void*)&g_lib, addresses.data(), addresses.size() * sizeof(uintptr_t));
    g_lib.on_host = on_host;
}

void check(int rc, const char* what) {
    if (rc) throw std::runtime_error(std::string("libmneslam_hip ") + what + " failed (" + std::to_string(rc) + "): " + g_lib.last_error());
}

// These calls are no operators of torch's dispatcher: a tracer sees the allocation of their results and not what fills it, so the program it
// makes would return memory that nothing wrote.  (Modes that only watch real operations, a counter for instance, are let through.)
void not_traced(const char* what) {
    using c10::impl::TorchDispatchModeKey;
    using c10::impl::TorchDispatchModeTLS;
    bool traced = torch::jit::tracer::isTracing() || c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch);
    if (TorchDispatchModeTLS::any_modes_set())
        for (const auto key : {TorchDispatchModeKey::PROXY, TorchDispatchModeKey::FAKE, TorchDispatchModeKey::FUNCTIONAL})
            traced = traced || TorchDispatchModeTLS::get_mode(key).has_value();
    if (traced) throw std::runtime_error(std::string(what) + ": this call cannot be traced (torch.jit.trace, make_fx, fake tensors)");
}
// ... and a tensor whose class brings its own operations is not the memory it holds.
void no_subclass(const char* what, const at::Tensor& t) {
    if (t.unsafeGetTensorImpl()->is_python_dispatch())
        throw py::type_error(std::string(what) + ": tensors of classes with operations of their own are not supported");
}

// All on one device that the library reaches (a kernel that is given an address of host memory would fault).
void one_device(const char* what, std::initializer_list<const at::Tensor*> tensors) {
    not_traced(what);
    const at::Device dev = (*tensors.begin())->device();
    for (const at::Tensor* t : tensors) {
        if (!t->defined()) continue;
        no_subclass(what, *t);
        if (t->layout() != at::kStrided) throw py::value_error(std::string(what) + ": sparse tensors are not supported");
        if (t->device() != dev) throw py::value_error(std::string(what) + ": tensors on " + dev.str() + " and on " + t->device().str());
    }
    if (dev.type() != (g_lib.on_host ? at::kCPU : at::kCUDA))
        throw py::value_error(std::string(what) + ": tensors on " + dev.str() + ": the HIP kernels need them on the GPU");
}

void* stream_of(const at::Device& dev) { return dev.is_cuda() ? (void*)c10::hip::getCurrentHIPStream(dev.index()).stream() : nullptr; }

int type_code(at::ScalarType t) {
    return t == at::kFloat ? MNE_T_F32 : t == at::kBFloat16 ? MNE_T_BF16 : t == at::kHalf ? MNE_T_F16 : -1;
}

// A tensor whose memory holds its values: one that is negated lazily (the imaginary part of a conjugate) is copied, and one of zeros that
// has no memory (forward-mode differentiation makes them) gets some.
at::Tensor in_memory(const at::Tensor& t) {
    if (t.defined() && t._is_zerotensor()) return t.clone();
    return t.defined() && t.is_neg() ? t.resolve_neg() : t;
}
bool written_in_memory(const at::Tensor& t) { return !t.is_neg() && !t._is_zerotensor(); }

// equal strides in every dimension that has more than one entry (the shapes are equal)
bool laid_out_alike(const at::Tensor& a, const at::Tensor& b) {
    for (int64_t d = 0; d < a.dim(); ++d)
        if (a.size(d) > 1 && a.stride(d) != b.stride(d)) return false;
    return true;
}

// A step that has been checked, ready to be launched.
struct AdamwStep {
    Tensors keep, clear;                                 // clear: gradients that are zeroed behind it
    at::Device dev = at::kCPU;
    std::map<std::pair<int, int>, std::vector<int64_t>> tables;          // by the types of parameter and gradient
    mne_adamw_cfg_t cfg = {};
    uintptr_t clock = 0;
};
// Memory that the steps write and read: from where to where, of which row, and the tensor (which the caller holds).
struct Range {
    int64_t from, to, owner;
    c10::TensorImpl* tensor;
};
struct Ranges {
    std::vector<Range> written, read;
    int64_t owners = 0;
};

// zero_grad: 1, by the step itself; 2, also of gradients laid out otherwise, behind it
AdamwStep adamw_prepare(Ranges& ranges, const Tensors& params, const Tensors& grads, const Tensors& exp_avgs, const Tensors& exp_avg_sqs,
                        const c10::optional<Tensors>& scales, const c10::optional<std::vector<int64_t>>& ordinals, double lr, double beta1,
                        double beta2, double eps, double weight_decay, int64_t step, int64_t seed, int64_t zero_grad, uintptr_t clock) {
    AdamwStep s;
    const size_t n = params.size();
    const bool small = scales.has_value();
    if (grads.size() != n || exp_avgs.size() != n || exp_avg_sqs.size() != n || (small && scales->size() != n) ||
        (ordinals && ordinals->size() != n))
        throw py::value_error("adamw_step: lists of different lengths");
    if (!n) return s;
    if (!params[0].defined()) throw py::value_error("adamw_step: undefined tensors");
    one_device("adamw_step", {&params[0]});
    const at::Device dev = params[0].device();
    c10::NoGradGuard no_grad;
    s.dev = dev; s.clock = clock;
    ranges.written.reserve(ranges.written.size() + 5 * n);
    ranges.read.reserve(ranges.read.size() + n);
    s.cfg.lr = lr; s.cfg.beta1 = beta1; s.cfg.beta2 = beta2; s.cfg.eps = eps; s.cfg.weight_decay = weight_decay;
    s.cfg.step = (int32_t)step; s.cfg.state_bits = small ? 8 : 32; s.cfg.zero_grad = zero_grad != 0; s.cfg.seed = (uint32_t)seed;
    for (size_t i = 0; i < n; ++i) {
        const at::Tensor &p = params[i], &m = exp_avgs[i], &v = exp_avg_sqs[i];
        at::Tensor g = grads[i];
        bool plain = true;                               // (all but a few are)
        for (const at::Tensor* t : {&p, (const at::Tensor*)&g, &m, &v, small ? &(*scales)[i] : &p}) {
            if (!t->defined() || t->layout() != at::kStrided) throw py::value_error("adamw_step: sparse or undefined tensors are not supported");
            no_subclass("adamw_step", *t);
            plain = plain && written_in_memory(*t);
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
        if (!plain) {
            for (const at::Tensor* t : {&p, &m, &v, small ? &(*scales)[i] : &p})
                if (!written_in_memory(*t)) throw py::value_error("adamw_step: what is written in place must not be a negated view or without memory");
            if (zero_grad) throw py::value_error("adamw_step: zero_grad cannot clear a negated view or zeros without memory");
            g = in_memory(g);
            s.keep.push_back(g);
        }
        const int64_t count = p.numel(), ordinal = ordinals ? (*ordinals)[i] : (int64_t)i;
        if (ordinal < 0 || ordinal > 0xFFFFFFFFll) throw py::value_error("adamw_step: ordinals are numbers of 32 bits");
        if (small) {
            const at::Tensor& t = (*scales)[i];
            if (t.scalar_type() != at::kFloat || t.dim() != 2 || t.size(0) != (count + 255) / 256 || t.size(1) != 2 || !t.is_contiguous() ||
                (count && (uintptr_t)t.data_ptr() % 8))
                throw py::value_error("adamw_step: scales must be contiguous float32 [ceil(n / 256), 2] at a multiple of 8 bytes");
        }
        if (!count) continue;
        if (!p.is_non_overlapping_and_dense()) throw py::value_error("adamw_step: parameters must be dense");
        if (!laid_out_alike(m, p) || !laid_out_alike(v, p)) throw py::value_error("adamw_step: moments must be laid out like their parameter");
        if (!laid_out_alike(g, p)) {
            if (zero_grad == 1) throw py::value_error("adamw_step: zero_grad needs gradients laid out like their parameters");
            if (zero_grad && at::has_internal_overlap(g) == at::MemOverlap::Yes)
                throw py::value_error("adamw_step: zero_grad cannot clear a gradient whose elements share memory");
            if (zero_grad) s.clear.push_back(g);
            g = at::empty_like(p, p.options().dtype(g.scalar_type())).copy_(g);
            s.keep.push_back(g);
        }
        std::vector<int64_t>& table = s.tables[{pt, gt}];
        const int64_t row[7] = {(int64_t)p.data_ptr(), (int64_t)g.data_ptr(), (int64_t)m.data_ptr(), (int64_t)v.data_ptr(),
                                small ? (int64_t)(*scales)[i].data_ptr() : 0, count, ordinal};
        const int64_t owner = ranges.owners++, wide = (int64_t)p.element_size(), state = small ? 1 : 4;
        ranges.written.push_back({row[0], row[0] + count * wide, owner, p.unsafeGetTensorImpl()});
        ranges.written.push_back({row[2], row[2] + count * state, owner, m.unsafeGetTensorImpl()});
        ranges.written.push_back({row[3], row[3] + count * state, owner, v.unsafeGetTensorImpl()});
        if (small) ranges.written.push_back({row[4], row[4] + (count + 255) / 256 * 8, owner, (*scales)[i].unsafeGetTensorImpl()});
        (zero_grad ? ranges.written : ranges.read).push_back({row[1], row[1] + count * (int64_t)g.element_size(), owner, g.unsafeGetTensorImpl()});
        table.insert(table.end(), row, row + 7);
    }
    if (clock) check(g_lib.adamw_step(nullptr, 0, &s.cfg, (const mne_clock_t*)clock, nullptr), "mne_adamw_step");        // (of no tensors: the clock alone)
    return s;
}

// What is written is nobody else's, and what is read (a gradient) is at most its own tensor's, element for element.
void adamw_apart(Ranges& ranges) {
    std::vector<Range>& w = ranges.written;
    std::sort(w.begin(), w.end(), [](const Range& a, const Range& b) { return a.from < b.from; });
    for (size_t i = 1; i < w.size(); ++i)
        if (w[i].from < w[i - 1].to) throw py::value_error("adamw_step: parameters or moments overlap (the same one twice?)");
    for (const Range& r : ranges.read) {
        auto at = std::upper_bound(w.begin(), w.end(), r.from, [](int64_t from, const Range& x) { return from < x.to; });
        for (; at != w.end() && at->from < r.to; ++at)
            if (at->owner != r.owner || at->from != r.from || at->to != r.to)
                throw py::value_error("adamw_step: a gradient overlaps what the step writes (parameters, moments)");
    }
}

// What autograd has saved of it is out of date, as after p.add_().
void adamw_changed(const Ranges& ranges) {
    for (const Range& r : ranges.written)
        if (!r.tensor->is_inference()) r.tensor->bump_version();
}

void adamw_launch(AdamwStep& s) {
    const c10::DeviceGuard guard(s.dev);
    c10::NoGradGuard no_grad;
    for (const auto& t : s.tables) {
        s.cfg.p_type = t.first.first;
        s.cfg.g_type = t.first.second;
        check(g_lib.adamw_step(t.second.data(), (int64_t)t.second.size() / 7, &s.cfg, (const mne_clock_t*)s.clock, stream_of(s.dev)), "mne_adamw_step");
    }
    for (const at::Tensor& g : s.clear) g.zero_();
}

void adamw_step(const Tensors& params, const Tensors& grads, const Tensors& exp_avgs, const Tensors& exp_avg_sqs,
                const c10::optional<Tensors>& scales, const c10::optional<std::vector<int64_t>>& ordinals, double lr, double beta1,
                double beta2, double eps, double weight_decay, int64_t step, int64_t seed, int64_t zero_grad, uintptr_t clock) {
    Ranges ranges;
    AdamwStep s = adamw_prepare(ranges, params, grads, exp_avgs, exp_avg_sqs, scales, ordinals, lr, beta1, beta2, eps, weight_decay, step, seed,
                                zero_grad, clock);
    adamw_apart(ranges);
    adamw_launch(s);
    adamw_changed(ranges);
}

// Several of them (an optimizer's groups): all are checked before the first is launched.
typedef std::tuple<Tensors, Tensors, Tensors, Tensors, c10::optional<Tensors>, c10::optional<std::vector<int64_t>>, double, double, double, double, double,
                   int64_t, int64_t, int64_t, uintptr_t> AdamwCall;
void adamw_steps(const std::vector<AdamwCall>& calls) {
    Ranges ranges;
    std::vector<AdamwStep> steps;
    for (const AdamwCall& call : calls)
        steps.push_back(std::apply([&](const auto&... args) { return adamw_prepare(ranges, args...); }, call));
    adamw_apart(ranges);
    for (AdamwStep& s : steps) adamw_launch(s);
    adamw_changed(ranges);
}

std::vector<at::Tensor> adamw_moments(const at::Tensor& given_m, const at::Tensor& given_v, const at::Tensor& given_scales) {
    one_device("adamw_moments", {&given_m, &given_v, &given_scales});
    c10::NoGradGuard no_grad;
    const at::Tensor m = in_memory(given_m), v = in_memory(given_v), scales = in_memory(given_scales);
    if (m.scalar_type() != at::kChar || v.scalar_type() != at::kByte) throw py::type_error("adamw_moments: the codes are int8 and uint8");
    if (m.sizes() != v.sizes() || !m.is_non_overlapping_and_dense() || !laid_out_alike(m, v))
        throw py::value_error("adamw_moments: the codes must be dense and laid out alike");
    const int64_t n = m.numel();
    if (scales.scalar_type() != at::kFloat || scales.dim() != 2 || scales.size(0) != (n + 255) / 256 || scales.size(1) != 2 || !scales.is_contiguous())
        throw py::value_error("adamw_moments: scales must be contiguous float32 [ceil(n / 256), 2]");
    const c10::DeviceGuard guard(m.device());
    at::Tensor a = at::empty_like(m, m.options().dtype(at::kFloat)), b = at::empty_like(a);
    check(g_lib.adamw_moments((const int8_t*)m.data_ptr(), (const uint8_t*)v.data_ptr(), (const float*)scales.data_ptr(), n,
                              (float*)a.data_ptr(), (float*)b.data_ptr(), stream_of(m.device())), "mne_adamw_moments");
    return {a, b};
}

// ---- routing ---------------------------------------------------------------------------------------------------------
// order [m], position [n, k], offsets [experts + 1]
std::vector<at::Tensor> expert_sort(const at::Tensor& given, int64_t experts) {
    one_device("expert_sort", {&given});
    if ((given.scalar_type() != at::kInt && given.scalar_type() != at::kLong) || (given.dim() != 1 && given.dim() != 2))
        throw py::type_error("expert_sort: ids must be int32 or int64 [N, K] or [N]");
    if (experts < 1 || experts > 4096) throw py::value_error("expert_sort: 1 to 4096 experts, got " + std::to_string(experts));
    const int64_t n = given.size(0), k = given.dim() == 2 ? given.size(1) : 1, m = n * k;
    if (k < 1) throw py::value_error("expert_sort: ids without a choice");
    if (m >= (1ll << 31) - 65536) throw py::value_error("expert_sort: too many choices for 32-bit rows");
    const c10::DeviceGuard guard(given.device());
    c10::NoGradGuard no_grad;
    const at::Tensor ids = in_memory(given).contiguous();
    const size_t bytes = g_lib.sort_bytes(m, (int)experts);
    // (tensors of their own: the workspace is free behind the call, and who writes into one of the plan's changes no other)
    const at::TensorOptions opts = ids.options().dtype(at::kInt);
    const at::Tensor order = at::empty({m}, opts), position = at::empty({n, k}, opts), offsets = at::empty({experts + 1}, opts);
    const at::Tensor workspace = bytes ? at::empty({(int64_t)bytes / 4}, opts) : at::Tensor();
    check(g_lib.sort(ids.data_ptr(), ids.scalar_type() == at::kLong, m, (int)experts, (int32_t*)order.data_ptr(), (int32_t*)position.data_ptr(),
                     (int32_t*)offsets.data_ptr(), bytes ? workspace.data_ptr() : nullptr, bytes, stream_of(ids.device())), "mne_expert_sort");
    return {order, position, offsets};
}

void check_rows(const at::Tensor& t, const char* what) {
    if (t.dim() != 2) throw py::value_error(std::string(what) + ": rows must be [rows, width]");
    if (type_code(t.scalar_type()) < 0)
        throw py::type_error(std::string(what) + ": " + c10::toString(t.scalar_type()) + " is not supported (float32, bfloat16, float16)");
}
// a row's elements next to each other (a copy where they are not)
at::Tensor rows(const at::Tensor& given, const char* what) {
    check_rows(given, what);
    const at::Tensor t = in_memory(given);
    return t.stride(1) == 1 || t.size(1) <= 1 ? t : t.contiguous();
}
at::Tensor weights32(const at::Tensor& t) { return t.defined() ? in_memory(t).to(at::kFloat).contiguous() : t; }
const int32_t* ints(const at::Tensor& t) { return (const int32_t*)t.data_ptr(); }
const int32_t* live_rows(const at::Tensor& offsets) { return ints(offsets) + offsets.size(0) - 1; }
const float* floats(const at::Tensor& t) { return t.defined() ? (const float*)t.data_ptr() : nullptr; }

at::Tensor dispatch(const Library& lib, const at::Tensor& given, const at::Tensor& position, const at::Tensor& offsets) {
    const at::Tensor x = rows(given, "expert_dispatch");
    const c10::DeviceGuard guard(x.device());
    const int64_t n = position.size(0), k = position.size(1), width = x.size(1);
    at::Tensor out = at::empty({n * k, width}, x.options());
    check(lib.dispatch(x.data_ptr(), x.stride(0), type_code(x.scalar_type()), n, (int)k, width, ints(position), live_rows(offsets), out.data_ptr(),
                       stream_of(x.device())), "mne_expert_dispatch");
    return out;
}

at::Tensor combine(const Library& lib, const at::Tensor& given, const at::Tensor& position, const at::Tensor& weights) {
    const at::Tensor y = rows(given, "expert_combine"), w = weights32(weights);
    const c10::DeviceGuard guard(y.device());
    const int64_t n = position.size(0), k = position.size(1), width = y.size(1);
    at::Tensor out = at::empty({n, width}, y.options());
    check(lib.combine(y.data_ptr(), y.stride(0), type_code(y.scalar_type()), n, (int)k, width, ints(position), floats(w), out.data_ptr(),
                      stream_of(y.device())), "mne_expert_combine");
    return out;
}

// A gradient of a gradient would come out as zero, unnoticed: refused.
void once(const char* what) {
    if (c10::GradMode::is_enabled()) throw std::runtime_error(std::string(what) + ": differentiable once (create_graph=True is not supported)");
}

// A backward pass that is being recorded must not lead on to the default stream, which cannot be recorded: the recording would be broken
// there in a way that ends the process.  It leads there if something upstream was built on that stream, also by a leaf alone that an
// eager graph still holds.
void recordable(const char* what, const at::Device& dev) {
    if (!dev.is_cuda() || c10::hip::getCurrentHIPStream(dev.index()).id() == 0) return;
    const c10::DeviceGuard guard(dev);
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    const std::shared_ptr<torch::autograd::Node> self = torch::autograd::get_current_node();
    std::vector<torch::autograd::Node*> open = {self.get()};
    std::unordered_set<torch::autograd::Node*> seen;
    while (!open.empty()) {
        torch::autograd::Node* node = open.back();
        open.pop_back();
        if (!node || !seen.insert(node).second) continue;
        const auto stream = node->stream();
        if (stream && stream->id() == 0)
            throw std::runtime_error(std::string(what) + ": this backward pass cannot be recorded, it leads to " + node->name() +
                                     " on the default stream (drop the eager graphs of the same leaves first)");
        for (const auto& edge : node->next_edges()) open.push_back(edge.function.get());
    }
}

Library library_of(AutogradContext* ctx) {
    Library lib;
    const std::string bytes = ctx->saved_data["library"].toStringRef();
    memcpy((void*)&lib, bytes.data(), sizeof(lib));
    return lib;
}

struct DispatchNode : torch::autograd::Function<DispatchNode> {
    static Variable forward(AutogradContext* ctx, const Variable& x, const Variable& position, const Variable& offsets) {
        ctx->save_for_backward({position});
        ctx->saved_data["library"] = std::string((const char*)&g_lib, sizeof(g_lib));
        return dispatch(g_lib, x, position, offsets);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once("expert_dispatch");
        not_traced("expert_dispatch");
        if (!grads[0].defined()) return {Variable(), Variable(), Variable()};
        recordable("expert_dispatch", grads[0].device());
        return {combine(library_of(ctx), grads[0], ctx->get_saved_variables()[0], at::Tensor()), Variable(), Variable()};
    }
};

struct CombineNode : torch::autograd::Function<CombineNode> {
    // (a node takes no undefined tensor: without weights, `weights` is any other; so is what is saved for `y` where the weights have no
    // gradient, which is all that its values are needed for)
    static Variable forward(AutogradContext* ctx, const Variable& y, const Variable& position, const Variable& offsets, const Variable& weights,
                            bool weighted) {
        ctx->save_for_backward({weighted && weights.requires_grad() ? y : position, position, offsets, weights});
        ctx->saved_data["library"] = std::string((const char*)&g_lib, sizeof(g_lib));
        ctx->saved_data["weighted"] = weighted;
        return combine(g_lib, y, position, weighted ? weights : at::Tensor());
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once("expert_combine");
        not_traced("expert_combine");
        if (!grads[0].defined()) return {Variable(), Variable(), Variable(), Variable(), Variable()};
        recordable("expert_combine", grads[0].device());
        const Library lib = library_of(ctx);
        const variable_list saved = ctx->get_saved_variables();
        const at::Tensor &position = saved[1], &offsets = saved[2];
        const at::Tensor weights = ctx->saved_data["weighted"].toBool() ? saved[3] : at::Tensor();
        const at::Tensor dout = rows(grads[0], "expert_combine"), w = weights32(weights);
        const c10::DeviceGuard guard(dout.device());
        const int64_t n = position.size(0), k = position.size(1), width = dout.size(1);
        const bool want_dw = weights.defined() && ctx->needs_input_grad(3), want_dy = ctx->needs_input_grad(0);
        const at::Tensor y = want_dw ? rows(saved[0], "expert_combine") : dout;          // (not read without dw)
        at::Tensor dy, dw;
        if (want_dy) dy = at::empty({n * k, width}, dout.options());
        if (want_dw) dw = width ? at::empty({n, k}, w.options()) : at::zeros({n, k}, w.options());
        check(lib.combine_backward(dout.data_ptr(), dout.stride(0), y.data_ptr(), y.stride(0), type_code(dout.scalar_type()), n, (int)k, width,
                                   ints(position), live_rows(offsets), floats(w), want_dy ? dy.data_ptr() : nullptr,
                                   want_dw ? (float*)dw.data_ptr() : nullptr, stream_of(dout.device())), "mne_expert_combine_backward");
        return {dy, Variable(), Variable(), want_dw ? dw.to(weights.scalar_type()) : dw, Variable()};
    }
};

void check_plan(const char* what, const at::Tensor& position, const at::Tensor& offsets) {
    if (position.scalar_type() != at::kInt || offsets.scalar_type() != at::kInt) throw py::type_error(std::string(what) + ": a plan's tensors are int32");
    if (position.dim() != 2 || position.size(1) < 1 || offsets.dim() != 1 || offsets.size(0) < 2 || !position.is_contiguous() || !offsets.is_contiguous())
        throw py::value_error(std::string(what) + ": not a plan of expert_sort");
    if (!written_in_memory(position) || !written_in_memory(offsets))
        throw py::value_error(std::string(what) + ": a plan's tensors must not be negated views or without memory");
}

at::Tensor expert_dispatch(const at::Tensor& x, const at::Tensor& position, const at::Tensor& offsets) {
    one_device("expert_dispatch", {&x, &position, &offsets});
    check_plan("expert_dispatch", position, offsets);
    if (x.dim() != 2 || x.size(0) != position.size(0))
        throw py::value_error("expert_dispatch: x must be [" + std::to_string(position.size(0)) + " tokens, width]");
    check_rows(x, "expert_dispatch");
    return DispatchNode::apply(x, position, offsets);
}

at::Tensor expert_combine(const at::Tensor& y, const at::Tensor& position, const at::Tensor& offsets, const c10::optional<at::Tensor>& weights) {
    const at::Tensor w = weights ? *weights : at::Tensor();
    one_device("expert_combine", {&y, &position, &offsets, &w});
    check_plan("expert_combine", position, offsets);
    if (y.dim() != 2 || y.size(0) != position.numel())
        throw py::value_error("expert_combine: y must be [" + std::to_string(position.numel()) + " rows, width]");
    if (w.defined()) {
        if (w.sizes() != position.sizes()) throw py::value_error("expert_combine: weights must be [tokens, choices]");
        if (type_code(w.scalar_type()) < 0) throw py::type_error("expert_combine: weights must be float32, bfloat16 or float16");
    }
    check_rows(y, "expert_combine");
    return CombineNode::apply(y, position, offsets, w.defined() ? w : position, w.defined());
}

}  // namespace

PYBIND11_MODULE(_host_tensors, m) {
    m.def("bind", &bind);
    m.def("adamw_step", &adamw_step);
    m.def("adamw_steps", &adamw_steps);
    m.def("adamw_moments", &adamw_moments);
    m.def("expert_sort", &expert_sort);
    m.def("expert_dispatch", &expert_dispatch);
    m.def("expert_combine", &expert_combine);
    m.attr("ABI_VERSION") = MNE_ABI_VERSION;
}
