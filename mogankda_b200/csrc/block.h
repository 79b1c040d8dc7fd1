// What the Python entry points of the operators around the layer share (block.cpp, mixer.cpp): the autograd node, rows and sequences as the kernels take them, checks.
#pragma once
#include "binding.h"

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/saved_variable.h>

#include <cmath>
#include <functional>
#include <memory>
#include <mutex>
#include <numeric>
#include <unordered_map>

using namespace mkda_host;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

namespace {

using Need = std::function<bool(int)>;
using Backward = std::function<variable_list(const variable_list& saved, const variable_list& grads, const Need& need)>;

// The node of a call: what it saves (inputs, then intermediates, an output among them where `output` says so) and the launches of its backward pass.
// Saved variables see in-place changes and a second backward pass, and saved-tensor hooks get all of them.
struct BlockBackward : public torch::autograd::Node {
    std::string what;
    at::Device dev = at::Device(at::kCUDA);
    std::vector<SavedVariable> vars;
    std::vector<bool> output;
    std::vector<std::vector<int64_t>> sizes;
    std::vector<at::ScalarType> types;
    std::vector<uint32_t> depends;             // per gradient: the inputs that it is a function of, besides the incoming gradients
    bool state_linear = false;                 // of the second output alone it is a function of none of them
    Backward run;
    bool released = false;

    std::string name() const override { return what + "Backward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        released = true;
        for (auto& v : vars) v.reset_data();
    }
    void save(const Tensor& t, bool is_output = false) {
        vars.emplace_back(t, is_output);
        output.push_back(is_output);
        sizes.push_back(t.defined() ? t.sizes().vec() : std::vector<int64_t>());
        types.push_back(t.defined() ? t.scalar_type() : at::kFloat);
    }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        TORCH_CHECK(!released, torch::autograd::ERR_BACKWARD_TWICE);
        variable_list saved;
        for (size_t i = 0; i < vars.size(); ++i) {
            saved.push_back(vars[i].unpack(output[i] ? getptr() : nullptr));
            const Tensor& t = saved.back();          // sizes and types decide what the kernels read
            TORCH_CHECK(!t.defined() || (t.sizes() == at::IntArrayRef(sizes[i]) && t.scalar_type() == types[i] && t.device() == dev), what,
                        ": a saved-tensor hook returned another tensor than was saved");
        }
        c10::cuda::CUDAGuard guard(dev);
        variable_list out;
        {
            at::AutoGradMode off(false);
            out = library_call([&] { return run(saved, grads, [&](int i) { return task_should_compute_output(i); }); });
        }
        for (size_t i = 0; i < out.size(); ++i)
            if (!task_should_compute_output(i)) out[i] = Tensor();
        refuse_second(*this, what, grads, state_linear && !grads[0].defined() ? std::vector<uint32_t>(out.size(), 0u) : depends, out);
        return out;
    }
};

std::shared_ptr<BlockBackward> new_node(const char* what, const at::Device& dev, const variable_list& inputs, std::vector<uint32_t> depends, Backward run) {
    auto node = std::shared_ptr<BlockBackward>(new BlockBackward(), torch::autograd::deleteNode);
    node->what = what;
    node->dev = dev;
    node->depends = std::move(depends);
    node->run = std::move(run);
    node->set_next_edges(torch::autograd::collect_next_edges(inputs));
    return node;
}

bool any_requires_grad(const variable_list& inputs) {
    if (!c10::GradMode::is_enabled()) return false;
    for (const Tensor& t : inputs)
        if (t.defined() && t.requires_grad()) return true;
    return false;
}

bool float_type(const Tensor& t) { return t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf; }
void check_rc(int rc, const char* what) {
    if (rc != MKDA_OK) throw LibraryError(std::string(what) + " failed (" + std::to_string(rc) + "): " + mkda_last_error());
}
const void* cptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* mptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
const float* fptr(const Tensor& t) { return static_cast<const float*>(cptr(t)); }
float* fmptr(const Tensor& t) { return static_cast<float*>(mptr(t)); }
// parameters and states of the scan: fp32, contiguous, 16-byte aligned
Tensor param(const Tensor& t) {
    if (!t.defined()) return t;
    return aligned(t.scalar_type() == at::kFloat ? t : t.to(at::kFloat));
}

// A tensor as rows of its last `inner` axes with one stride between them: a slice of the channels of a wider projection is read where it lies; other
// layouts are copied.
struct Rows { Tensor t; int64_t stride = 0; };
Rows rows_of(const Tensor& t, int inner = 1) {
    if (!t.defined()) return {};
    int64_t width = 1;
    bool dense = true;
    for (int64_t d = t.dim() - 1; d >= t.dim() - inner; --d) {
        if (t.size(d) != 1 && t.stride(d) != width) dense = false;
        width *= t.size(d);
    }
    int64_t stride = -1, span = -1;
    for (int64_t d = t.dim() - inner - 1; dense && d >= 0; --d) {
        if (t.size(d) == 1) continue;
        if (stride < 0) stride = t.stride(d);
        else if (t.stride(d) != span) dense = false;
        span = t.stride(d) * t.size(d);
    }
    if (!dense) return {t.contiguous(), width};
    return {t, stride < 0 ? width : stride};
}

// The sequences of a call.  table: int32, boundaries, first checkpoints and order of packed sequences, or undefined for the rows of a batch.
struct Sequences {
    MkdaSeqs s{};
    Tensor table;
    bool covers_all = true;
    int64_t checkpoints = 0, longest = 0, end = 0;         // end: behind the last sequence
};
bool get_sequences(PyObject* table, PyObject* dims, int64_t B, int64_t T, Sequences& q) {
    if (!tensor_arg(table, q.table)) return false;
    q.s.TT = (int)(B * T);
    q.s.T = (int)T;
    if (!q.table.defined()) {
        q.s.N = (int)B;
        q.s.has_empty = T == 0;
        q.checkpoints = B * ((T + MKDA_SCAN_CHECKPOINT - 1) / MKDA_SCAN_CHECKPOINT);
        q.longest = T;
        q.end = B * T;
        return true;
    }
    int all, empty;
    long long ck, longest, end;
    if (!PyArg_ParseTuple(dims, "iiiLLL", &q.s.N, &all, &empty, &ck, &longest, &end)) return false;
    q.covers_all = all;
    q.s.has_empty = empty;
    q.checkpoints = ck;
    q.longest = longest;
    q.end = end;
    const int* p = static_cast<const int*>(q.table.data_ptr());
    q.s.cu = p;
    q.s.ckpt_off = p + q.s.N + 1;
    q.s.order = p + 2 * q.s.N + 1;
    return true;
}
// The kernels of the current stream read the table: the allocator hears of it if it is another stream than the table's own, and a table that a stream capture records is
// kept for good, since the cache that holds it (index.py) may let go of it before the last replay.
void reads_table(const Sequences& q) {
    if (!q.table.defined()) return;
    const auto on = c10::cuda::getCurrentCUDAStream();
    if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) {
        c10::cuda::CUDACachingAllocator::recordStream(q.table.storage().data_ptr(), on);
        return;
    }
    static std::mutex lock;
    static auto* const kept = new std::unordered_map<const void*, Tensor>();      // never destroyed: CUDA may be gone by then
    std::lock_guard<std::mutex> hold(lock);
    kept->emplace(q.table.unsafeGetTensorImpl(), q.table);
}
Tensor out_like(const Tensor& x, bool covers_all) {          // contiguous; tokens outside every sequence are zero
    Tensor t = new_cuda(x.sizes(), x.scalar_type(), x.device());
    if (!covers_all) t.zero_();
    return t;
}
cudaStream_t stream() { return c10::cuda::getCurrentCUDAStream(); }
int sms() { return at::cuda::getCurrentDeviceProperties()->multiProcessorCount; }

// What every call refuses: tensors on the CPU or on several devices, forward-mode AD
bool check_devices(const char* what, const variable_list& ts) {
    for (const Tensor& t : ts) {
        if (!t.defined()) continue;
        if (!t.is_cuda()) { fail(PyExc_RuntimeError, NEED_CUDA); return false; }
        if (t.device() != ts[0].device()) { fail(PyExc_RuntimeError, std::string(what) + ": all tensors must be on the same device"); return false; }
        if (t._fw_grad(0).defined()) { fail(PyExc_NotImplementedError, std::string(what) + ": forward-mode AD is not supported"); return false; }
    }
    return true;
}
bool parse_tensors(const char* what, PyObject* const* a, int n, int required, variable_list& ts) {
    ts.resize(n);
    for (int i = 0; i < n; ++i) {
        if (!tensor_arg(a[i], ts[i])) return false;
        if (i < required && !ts[i].defined()) { PyErr_Format(PyExc_TypeError, "%s: argument %d must be a tensor", what, i + 1); return false; }
    }
    return true;
}
PyObject* pair(const Tensor& a, const Tensor& b) {
    PyObject* pa = THPVariable_Wrap(a);
    if (!pa) return nullptr;
    PyObject* pb = Py_None;
    if (b.defined()) pb = THPVariable_Wrap(b);
    else Py_INCREF(pb);
    PyObject* r = pb ? PyTuple_Pack(2, pa, pb) : nullptr;
    Py_DECREF(pa);
    Py_XDECREF(pb);
    return r;
}
std::string count_error(int64_t want, int64_t got) {
    return "The number of initial states is expected to be equal to the number of input sequences, i.e., " + std::to_string(want) + " rather than " +
           std::to_string(got) + ".";
}
constexpr int64_t MOST_CHANNELS = 1 << 24;
constexpr int64_t MOST_TOKENS = MKDA_SEQS_MAX_TOKENS;

int64_t row_count(const Tensor& x) {
    int64_t n = 1;
    for (int64_t d = 0; d + 1 < x.dim(); ++d) n *= x.size(d);
    return n;
}
// the single-token forms: no gradient, and a state that is updated where it lies
bool check_step(const char* what, const variable_list& t, const Tensor& state) {
    if (any_requires_grad(t)) { fail(PyExc_RuntimeError, std::string(what) + " has no backward pass: call it under torch.no_grad()"); return false; }
    if (!state.is_contiguous() || reinterpret_cast<uintptr_t>(state.data_ptr()) % 16) {
        fail(PyExc_AssertionError, std::string(what) + ": the state is updated in place and must be contiguous and 16-byte aligned");
        return false;
    }
    if (state.is_inference() && !c10::InferenceMode::is_enabled()) {
        fail(PyExc_RuntimeError, std::string(what) + ": an inference tensor can only be updated in place in inference mode");
        return false;
    }
    return true;
}
void changed(const Tensor& t) {          // what an in-place operation tells autograd
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

}  // namespace
