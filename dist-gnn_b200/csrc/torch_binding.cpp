// Native side of the training path's hot calls: what a PyTorch program issues per step, without the interpreter in between.
//
// A training step on a small graph is bound by the host.  Issued from Python, autograd nodes, argument conversions and views
// cost three times what the step's kernels take (10,000-node graph: 0.4 ms of host work for 0.12 ms of kernels).  Here the
// one-rank network, the loss of the train rows and the local product are C++ autograd nodes and functions over the C ABI
// of include/dist_gnn_b200.h; torch owns memory, streams and the graph, as everywhere in this package.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <algorithm>
#include <atomic>
#include <functional>
#include <mutex>
#include <unordered_map>
#include "dist_gnn_b200.h"

namespace {

using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

std::atomic<int64_t> g_launches{0};       // dense-transform launches since the last take_launches()

void check(int code)
{
    if (code != DG_OK) throw std::runtime_error("dist_gnn_b200 error " + std::to_string(code) + ": " + dg_strerror(code));
}

void* stream_of(const Tensor& t) { return (void*)at::cuda::getCurrentCUDAStream(t.get_device()).stream(); }
int64_t pad4(int64_t w) { return (w + 3) / 4 * 4; }

// ---- time marks of regions that no Python code sees: kept until the timer they belong to asks ---------------------------
// One list per call: the points between its products and transforms, which alternate.  A region read out one by one from the
// interpreter was 5 us of host work, a quarter of a small training step; here it is what cudaEventElapsedTime takes.
struct Regions {
    std::vector<int32_t> marks;
    bool backward;                        // every layer then counts an all-reduce that a rank without peers has not to do
};
std::mutex g_regions_mu;
std::unordered_map<int64_t, std::vector<Regions>> g_regions;

void add_regions(int64_t timer, std::vector<int32_t>&& marks, bool backward)
{
    std::lock_guard<std::mutex> lock(g_regions_mu);
    g_regions[timer].push_back({std::move(marks), backward});
}
int64_t pending_regions(int64_t timer)
{
    std::lock_guard<std::mutex> lock(g_regions_mu);
    int64_t n = 0;
    const auto it = g_regions.find(timer);
    if (it != g_regions.end())
        for (const Regions& r : it->second) n += (int64_t)r.marks.size() - 1;
    return n;
}
// (seconds, regions) of the products, the transforms and the all-reduces since the last call.  The device has passed the marks.
std::vector<std::pair<double, int64_t>> resolve_regions(int64_t timer)
{
    std::vector<Regions> calls;
    {
        std::lock_guard<std::mutex> lock(g_regions_mu);
        const auto it = g_regions.find(timer);
        if (it != g_regions.end()) {
            calls = std::move(it->second);
            g_regions.erase(it);
        }
    }
    std::vector<std::pair<double, int64_t>> sums(3, {0.0, 0});
    int failed = DG_OK;
    for (const Regions& r : calls) {
        for (size_t i = 0; i + 1 < r.marks.size(); ++i) {
            auto& sum = sums[i & 1];
            ++sum.second;
            float ms = 0.f;
            if (r.marks[i] < 0 || r.marks[i + 1] < 0) continue;
            const int rc = dg_mark_elapsed(r.marks[i], r.marks[i + 1], &ms);
            if (rc != DG_OK) failed = rc;
            else sum.first += ms / 1000.0;
        }
        for (int32_t id : r.marks)
            if (id >= 0) dg_mark_release(id);
        if (r.backward) sums[2].second += (int64_t)r.marks.size() / 2;
    }
    check(failed);
    return sums;
}

// ---- a plan that the autograd graph can keep alive ----------------------------------------------------------------------
struct PlanRef {
    dg_plan* plan;
    Tensor col, values;                   // borrowed by the plan
    PlanRef(int64_t handle, Tensor c, Tensor v) : plan(reinterpret_cast<dg_plan*>(handle)), col(std::move(c)), values(std::move(v)) {}
    PlanRef(const PlanRef&) = delete;
    ~PlanRef() { dg_plan_destroy(plan); }
};

// ---- the local product --------------------------------------------------------------------------------------------------
int64_t operand(const Tensor& t, int64_t rows, const char* what)
{
    if (!t.defined() || !t.is_cuda() || t.scalar_type() != at::kFloat || t.dim() != 2)
        throw std::runtime_error(std::string(what) + " must be a 2-D fp32 CUDA tensor");
    if (t.size(0) != rows || (t.size(1) > 1 && t.stride(1) != 1)) {
        std::ostringstream s;
        s << what << " has shape " << t.sizes() << " / strides " << t.strides() << ", expected " << rows << " rows, unit column stride";
        throw std::runtime_error(s.str());
    }
    return t.size(0) > 1 ? t.stride(0) : std::max<int64_t>(t.size(1), 1);
}
const float* vector_ptr(const std::optional<Tensor>& t, const char* what)
{
    if (!t.has_value()) return nullptr;
    if (!t->is_cuda()) throw std::runtime_error(std::string(what) + " must be a CUDA tensor: this library has no CPU path");
    if (t->scalar_type() != at::kFloat || !t->is_contiguous()) throw std::runtime_error(std::string(what) + " must be a contiguous torch.float32 tensor");
    return t->data_ptr<float>();
}

void spmm(const std::shared_ptr<PlanRef>& ref, int64_t m, int64_t k, int64_t val, const Tensor& B, const Tensor& C, double alpha, double beta,
          const std::optional<Tensor>& row_scale, const std::optional<Tensor>& bias, bool relu)
{
    const int64_t ldb = operand(B, k, "B"), ldc = operand(C, m, "C");
    if (B.size(1) != C.size(1)) throw std::runtime_error("B and C differ in width");
    const float *scale = vector_ptr(row_scale, "row_scale"), *shift = vector_ptr(bias, "bias");
    const uint32_t flags = (scale ? DG_EPI_ROW_SCALE : 0u) | (shift ? DG_EPI_BIAS : 0u) | (relu ? DG_EPI_RELU : 0u);
    c10::cuda::CUDAGuard guard(ref->values.device());
    check(dg_spmm_csr(ref->plan, reinterpret_cast<const float*>(val), B.data_ptr<float>(), ldb, C.data_ptr<float>(), ldc, (int32_t)B.size(1), (float)alpha,
                      (float)beta, flags, scale, shift, stream_of(ref->values)));
}

// ---- operands with rows of whole 16-byte pieces ---------------------------------------------------------------------------
// t [n x w] as [n x pad4(w)] where it can be read that way in place (the columns beyond w are read and their results dropped).
bool readable_padded(const Tensor& t, int64_t width)
{
    const int64_t n = t.size(0), ld = t.stride(0);
    if (t.stride(1) != 1 || ld % 4 || ld < width || (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15)) return false;
    return width == t.size(1) || t.storage_offset() + (n - 1) * ld + width <= (int64_t)(t.storage().nbytes() / 4);
}
Tensor padded_copy(const Tensor& t)
{
    const Tensor src = (t.size(1) > 1 && t.stride(1) != 1) || t.stride(0) < t.size(1) ? t.contiguous() : t;
    Tensor wide = at::empty({t.size(0), pad4(t.size(1))}, t.options());
    check(dg_pad_rows(src.data_ptr<float>(), src.size(0) > 1 ? src.stride(0) : src.size(1), src.size(0), (int32_t)src.size(1), wide.data_ptr<float>(),
                      wide.size(1), stream_of(t)));
    return wide;
}

// ---- partial results of weight gradients ------------------------------------------------------------------------------------
// A product's own, from torch's allocator: products on two streams may run at the same time, and the memory serves the next one on its stream.
int tn_ctas(const Tensor& x) { return at::cuda::getDeviceProperties(x.get_device())->multiProcessorCount; }
int64_t tn_floats(int64_t Km, int64_t Nn, int ctas)
{
    return ctas * ((std::min<int64_t>(Km, 256) + 127) / 128 * 128) * ((std::min<int64_t>(Nn, 256) + 15) / 16 * 16);
}
std::pair<Tensor, int> tn_scratch(const Tensor& x, int64_t Km, int64_t Nn)
{
    const int ctas = tn_ctas(x);
    return {at::empty({tn_floats(Km, Nn, ctas)}, x.options()), ctas};
}

// ---- the whole GCN on one rank ----------------------------------------------------------------------------------------------
struct Net {                              // shapes and buffers of one call
    std::vector<int32_t> dims;
    std::vector<float*> act;
    std::vector<int64_t> ld_act;
    std::vector<int32_t> marks;
    dg_gcn_net net{};
    Net(const PlanRef& plan, const Tensor& x, const std::vector<int32_t>& d, std::vector<float*> a) : dims(d), act(std::move(a)), marks(2 * d.size() - 1, -1)
    {
        const int L = (int)dims.size() - 1;
        for (int l = 0; l < L; ++l) ld_act.push_back(l + 1 < L ? pad4(dims[l + 1]) : dims[l + 1]);
        net.plan = plan.plan;
        net.val = plan.values.data_ptr<float>();
        net.dims = dims.data();
        net.x = x.data_ptr<float>();
        net.ldx = x.size(0) > 1 ? x.stride(0) : pad4(dims[0]);
        net.act = act.data();
        net.ld_act = ld_act.data();
        net.marks = marks.data();
        net.n = (int32_t)x.size(0);
        net.layers = L;
    }
};

struct GcnNode : public torch::autograd::Node {
    std::shared_ptr<PlanRef> plan;
    SavedVariable features;               // only to notice that they were changed in place
    std::vector<SavedVariable> weights;
    Tensor x, hidden, splits;
    std::vector<int32_t> dims;
    std::vector<int64_t> act_start, bwd_split;
    int64_t timer = 0;

    std::string name() const override { return "OneRankGcnBackward"; }
    void release_variables() override
    {
        features.reset_data();
        for (auto& w : weights) w.reset_data();
        x.reset(), hidden.reset(), splits.reset();
    }
    variable_list apply(variable_list&& grads) override
    {
        const int L = (int)dims.size() - 1;
        variable_list out((size_t)L);
        if (!grads[0].defined()) return out;
        TORCH_CHECK(x.defined(), "Trying to backward through the graph a second time");
        features.unpack();
        std::vector<Tensor> w;
        for (auto& s : weights) w.push_back(s.unpack());
        c10::cuda::CUDAGuard guard(x.device());
        const int64_t n = x.size(0), width = pad4(dims[L]);
        Tensor g = grads[0].scalar_type() == at::kFloat ? grads[0] : grads[0].to(at::kFloat);
        if (!readable_padded(g, width)) g = width == g.size(1) ? g.contiguous() : padded_copy(g);
        std::vector<float*> act;
        float* base = hidden.data_ptr<float>();
        for (int l = 0; l + 1 < L; ++l) act.push_back(base + act_start[l]);
        act.push_back(x.data_ptr<float>());               // the last activation is not read
        Net call(*plan, x, dims, act);
        int64_t widest = 0, widest_hidden = 0;
        for (int l = 1; l <= L; ++l) widest = std::max(widest, pad4(dims[l]));
        for (int l = 1; l < L; ++l) widest_hidden = std::max(widest_hidden, pad4(dims[l]));
        Tensor work = at::empty({n * (widest + widest_hidden)}, x.options());
        call.net.z = work.data_ptr<float>();
        call.net.g = L > 1 ? call.net.z + n * widest : nullptr;
        std::vector<const float*> split((size_t)L, nullptr);
        for (int l = 1; l < L; ++l) split[l] = splits.data_ptr<float>() + bwd_split[l];
        std::vector<float*> dw((size_t)L, nullptr);
        int64_t launches = 0;
        auto panels = [](int64_t d) { return (d + 255) / 256; };
        for (int l = 0; l < L; ++l) {
            if (l > 0) launches += panels(dims[l]);
            if (!task_should_compute_output((size_t)l)) continue;
            out[l] = at::empty_like(w[l]);
            dw[l] = out[l].data_ptr<float>();
            launches += 2 * panels(dims[l]) * panels(dims[l + 1]);
        }
        call.net.grad = g.data_ptr<float>();
        call.net.ld_grad = n > 1 ? g.stride(0) : width;
        call.net.dw = dw.data();
        call.net.bwd_split = split.data();
        const int ctas = tn_ctas(x);
        int64_t partials = 0;
        for (int l = 0; l < L; ++l)
            if (dw[l]) partials = std::max(partials, tn_floats(dims[l], dims[l + 1], ctas));
        Tensor partial = at::empty({std::max<int64_t>(partials, 1)}, x.options());
        call.net.tn_scratch = partial.data_ptr<float>();
        call.net.tn_scratch_floats = partial.numel();
        call.net.max_ctas = ctas;
        check(dg_gcn_backward(&call.net, stream_of(x)));
        g_launches += launches;
        add_regions(timer, std::move(call.marks), true);
        return out;
    }
};

Tensor gcn(const std::shared_ptr<PlanRef>& plan, const Tensor& features, const Tensor& x, const std::vector<Tensor>& weights, int64_t timer)
{
    const int L = (int)weights.size();
    const int64_t n = x.size(0);
    bool train = false;
    for (const Tensor& w : weights) train = train || w.requires_grad();
    train = train && at::GradMode::is_enabled();
    c10::cuda::CUDAGuard guard(x.device());
    Tensor out, hidden, splits;
    std::vector<int64_t> act_start, fwd_split((size_t)L), bwd_split((size_t)L, -1);
    std::vector<int32_t> dims(1, (int32_t)features.size(1));
    for (const Tensor& w : weights) dims.push_back((int32_t)w.size(1));
    {
        at::AutoDispatchBelowADInplaceOrView below;
        // all weights split by one launch: W^T for the forward pass, W for the backward pass of every layer but the first
        int64_t floats = 0;
        for (int l = 0; l < L; ++l) {
            fwd_split[l] = floats;
            floats += 2 * dims[l + 1] * pad4(dims[l]);
            if (train && l > 0) {
                bwd_split[l] = floats;
                floats += 2 * dims[l] * pad4(dims[l + 1]);
            }
        }
        splits = at::empty({floats}, x.options());
        std::vector<dg_split_job> jobs;
        float* sbase = splits.data_ptr<float>();
        for (int l = 0; l < L; ++l) {
            const float* w = weights[l].data_ptr<float>();
            const int32_t K = dims[l], N = dims[l + 1];
            float* f = sbase + fwd_split[l];
            jobs.push_back({w, N, f, f + N * pad4(K), pad4(K), N, K, 1, 0});
            if (bwd_split[l] >= 0) {
                float* b = sbase + bwd_split[l];
                jobs.push_back({w, N, b, b + K * pad4(N), pad4(N), K, N, 0, 0});
            }
        }
        check(dg_dense_split_operands(jobs.data(), (int32_t)jobs.size(), stream_of(x)));
        // hidden activations in one buffer: side by side while a backward pass will read them, else every layer over the last
        int64_t sum = 0, widest_in = 0, widest_hidden = 0;
        for (int l = 0; l < L; ++l) widest_in = std::max(widest_in, pad4(dims[l]));
        for (int l = 1; l < L; ++l) {
            act_start.push_back(train ? sum : 0);
            sum += n * pad4(dims[l]);
            widest_hidden = std::max(widest_hidden, pad4(dims[l]));
        }
        hidden = at::empty({train ? sum : n * widest_hidden}, x.options());
        out = at::empty({n, dims[L]}, x.options());
        Tensor z = at::empty({n * widest_in}, x.options());
        std::vector<float*> act;
        for (int64_t s : act_start) act.push_back(hidden.data_ptr<float>() + s);
        act.push_back(out.data_ptr<float>());
        Net call(*plan, x, dims, act);
        std::vector<const float*> heads;
        for (int64_t s : fwd_split) heads.push_back(sbase + s);
        call.net.z = z.data_ptr<float>();
        call.net.fwd_split = heads.data();
        check(dg_gcn_forward(&call.net, stream_of(x)));
        int64_t launches = 1;
        for (int l = 1; l <= L; ++l) launches += (dims[l] + 255) / 256;
        g_launches += launches;
        add_regions(timer, std::move(call.marks), false);
    }
    if (train) {
        auto node = std::shared_ptr<GcnNode>(new GcnNode(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(weights));
        node->plan = plan;
        node->features = SavedVariable(features, false);
        for (const Tensor& w : weights) node->weights.emplace_back(w, false);
        node->x = x.detach();
        node->hidden = hidden;
        node->splits = splits;
        node->dims = dims;
        node->act_start = act_start;
        node->bwd_split = bwd_split;
        node->timer = timer;
        torch::autograd::set_history(out, node);
    }
    return out;
}

// ---- mean cross-entropy of the rows with a target ------------------------------------------------------------------------------
struct RowLossNode : public torch::autograd::Node {
    SavedVariable logits;
    Tensor targets, lse;
    int64_t count = 0;

    std::string name() const override { return "RowCrossEntropyBackward"; }
    void release_variables() override
    {
        logits.reset_data();
        targets.reset(), lse.reset();
    }
    variable_list apply(variable_list&& grads) override
    {
        if (!grads[0].defined()) return {Tensor()};
        TORCH_CHECK(lse.defined(), "Trying to backward through the graph a second time");
        const Tensor x = logits.unpack();
        c10::cuda::CUDAGuard guard(x.device());
        const Tensor up = grads[0].contiguous();
        const int64_t n = x.size(0), C = x.size(1), width = pad4(C);
        Tensor grad = at::empty({n, width}, x.options());
        check(dg_rows_cross_entropy_grad(x.data_ptr<float>(), n > 1 ? x.stride(0) : C, n, (int32_t)C, targets.data_ptr<int32_t>(), count, lse.data_ptr<float>(),
                                         up.data_ptr<float>(), grad.data_ptr<float>(), width, stream_of(x)));
        return {width == C ? grad : grad.narrow(1, 0, C)};
    }
};

Tensor row_cross_entropy(const Tensor& x, const Tensor& targets, int64_t count)
{
    if (!x.is_cuda() || x.scalar_type() != at::kFloat || x.dim() != 2 || (x.size(1) > 1 && x.stride(1) != 1) || (x.size(0) > 1 && x.stride(0) < x.size(1)))
        throw std::runtime_error("logits must be a row-major fp32 CUDA matrix");
    if (!targets.is_cuda() || targets.scalar_type() != at::kInt || !targets.is_contiguous() || targets.numel() != x.size(0))
        throw std::runtime_error("targets must be a contiguous int32 CUDA tensor with one entry per row");
    const bool train = x.requires_grad() && at::GradMode::is_enabled();
    c10::cuda::CUDAGuard guard(x.device());
    Tensor loss, lse;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        const int64_t n = x.size(0), parts = dg_rows_loss_scratch();
        lse = at::empty({n}, x.options());
        const Tensor sums = at::empty({parts}, x.options().dtype(at::kDouble));
        loss = at::empty({}, x.options());
        check(dg_rows_cross_entropy(x.data_ptr<float>(), n > 1 ? x.stride(0) : x.size(1), n, (int32_t)x.size(1), targets.data_ptr<int32_t>(), count,
                                    lse.data_ptr<float>(), sums.data_ptr<double>(), loss.data_ptr<float>(), stream_of(x)));
    }
    if (train) {
        auto node = std::shared_ptr<RowLossNode>(new RowLossNode(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(x));
        node->logits = SavedVariable(x, false);
        node->targets = targets;
        node->lse = lse;
        node->count = count;
        torch::autograd::set_history(loss, node);
    }
    return loss;
}

int32_t type_of(const Tensor& t)
{
    switch (t.scalar_type()) {
        case at::kFloat: return DG_FLOAT32;
        case at::kBFloat16: return DG_BFLOAT16;
        case at::kHalf: return DG_FLOAT16;
        default: return -1;
    }
}

// ---- linear layer with bias, activation and residual --------------------------------------------------------------------------------
int64_t item_of(const Tensor& t) { return t.scalar_type() == at::kFloat ? 4 : 2; }
int64_t pad_row(int64_t w, int64_t item) { return (w * item + 15) / 16 * 16 / item; }
int64_t ld_of(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : std::max(t.stride(0), t.size(1)); }
// t itself, or a copy of it, with elements of a row side by side and rows that do not overlap
Tensor by_rows(const Tensor& t)
{
    return (t.size(1) > 1 && t.stride(1) != 1) || (t.size(0) > 1 && t.stride(0) < t.size(1)) ? t.contiguous() : t;
}
bool on_rows(const Tensor& t) { return ld_of(t) * item_of(t) % 16 == 0 && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }
Tensor whole_rows(int64_t rows, int64_t cols, const Tensor& like)
{
    const int64_t width = pad_row(cols, item_of(like));
    const Tensor t = at::empty({rows, width}, like.options().requires_grad(false));
    return width == cols ? t : t.narrow(1, 0, cols);
}
// whole_rows that go to the caller.  Products of this library read padded rows of fp32 operands whole: what they find there is zero.
Tensor result_rows(int64_t rows, int64_t cols, const Tensor& like)
{
    const Tensor t = whole_rows(rows, cols, like);
    if (item_of(like) == 4 && t.stride(0) != cols && rows > 0) t.as_strided({rows, t.stride(0) - cols}, {t.stride(0), 1}, t.storage_offset() + cols).zero_();
    return t;
}
// by_rows(t), with rows of whole 16-byte pieces
Tensor to_rows(const Tensor& t, int64_t* launches)
{
    const Tensor src = by_rows(t);
    if (on_rows(src)) return src;
    const Tensor out = whole_rows(src.size(0), src.size(1), src);
    check(item_of(src) == 4 ? dg_pad_rows(src.data_ptr<float>(), ld_of(src), src.size(0), (int32_t)src.size(1), out.data_ptr<float>(), out.stride(0), stream_of(src))
                            : dg_pad_rows16(src.data_ptr(), ld_of(src), src.size(0), (int32_t)src.size(1), out.data_ptr(), out.stride(0), stream_of(src)));
    ++*launches;
    return out;
}

// A weight [K x N] as the matrix that lies in memory: its rows are inputs, or outputs where out_in.
struct Weight {
    Tensor t;
    bool out_in;
};
Weight stored(const Tensor& w)
{
    const int64_t K = w.size(0), N = w.size(1);
    const bool in_out = (N == 1 || w.stride(1) == 1) && (K == 1 || w.stride(0) >= N), out_in = (K == 1 || w.stride(0) == 1) && (N == 1 || w.stride(1) >= K);
    if (out_in && (N == 1 || !in_out)) return {w.t(), true};
    return {in_out ? w : w.contiguous(), false};
}

// What the gradients read goes through saved variables, so that changes in place are noticed and saved-tensor hooks (offloading, checkpoints) have all of it: x where the weight wants
// its gradient, the weight, and what the product made.  Where the product read a copy of x or of the weight (odd rows, odd strides) the copy is kept in its place.
struct LinearNode : public torch::autograd::Node {
    SavedVariable x_saved, w_saved, splits_saved, z_saved, bits_saved;
    at::TensorOptions options;            // of x
    int64_t M = 0, N = 0, K = 0;
    int32_t act = 0;
    bool w_copied = false, w_out_in = false;      // the kept copy, as it lies in memory

    std::string name() const override { return "LinearBackward"; }
    void release_variables() override
    {
        for (SavedVariable* v : {&x_saved, &w_saved, &splits_saved, &z_saved, &bits_saved}) v->reset_data();
    }
    variable_list apply(variable_list&& grads) override
    {
        variable_list out(4);
        if (!grads[0].defined()) return out;
        TORCH_CHECK(!at::GradMode::is_enabled(), "the gradient of linear cannot be differentiated again");
        const bool dx = task_should_compute_output(0), dw = task_should_compute_output(1), db = task_should_compute_output(2), dr = task_should_compute_output(3);
        c10::cuda::CUDAGuard guard(options.device());
        const Tensor x = x_saved.unpack(), splits = splits_saved.unpack(), bits = bits_saved.unpack();
        Tensor z = z_saved.unpack();
        if (z.defined()) z = by_rows(z);
        Weight weight{w_saved.unpack(), w_out_in};
        if (weight.t.defined() && !w_copied) weight = stored(weight.t);
        Tensor& w = weight.t;
        const bool out_in = weight.out_in;
        const at::ScalarType dtype = options.dtype().toScalarType();
        const Tensor dy = grads[0].scalar_type() == dtype ? grads[0] : grads[0].to(dtype);
        void* stream = stream_of(dy);
        const int64_t item = item_of(dy);
        const int32_t type = type_of(dy);
        if (dr) out[3] = dy;
        if (M == 0) {
            if (dx) out[0] = at::empty({M, K}, options);
            if (dw) out[1] = at::zeros({K, N}, options);
            if (db) out[2] = at::zeros({N}, options);
            return out;
        }
        int64_t launches = 0;
        Tensor g = by_rows(dy);
        if (db) out[2] = at::empty({N}, options);
        const uint32_t* signs = bits.defined() ? reinterpret_cast<const uint32_t*>(bits.data_ptr<int32_t>()) : nullptr;
        const int64_t ldbits = bits.defined() ? bits.size(1) : 0;
        if (N <= 32 && K <= 32) {                                 // narrow: all of them in one pass
            const Tensor d = !dw ? Tensor() : out_in ? at::empty({N, K}, options) : at::empty({K, N}, options);
            const Tensor scratch = dw || db ? at::empty({dg_linear_grad_scratch(M, (int32_t)N, (int32_t)K)}, options.dtype(at::kFloat)) : Tensor();
            dg_linear_grad_args a{};
            const Tensor rows = dw ? by_rows(x) : Tensor();
            if (dw) a.x = rows.data_ptr(), a.ldx = ld_of(rows);
            if (dx) a.w = w.data_ptr(), a.ldw = ld_of(w);
            a.dy = g.data_ptr(), a.lddy = ld_of(g), a.bits = signs, a.ldbits = ldbits;
            if (z.defined()) a.z = z.data_ptr(), a.ldz = ld_of(z);
            if (dx) out[0] = at::empty({M, K}, options), a.dx = out[0].data_ptr(), a.lddx = K;
            if (dw) a.dw = d.data_ptr(), a.row_stride = out_in ? 1 : N, a.col_stride = out_in ? K : 1, out[1] = out_in ? d.t() : d;
            if (db) a.db = out[2].data_ptr();
            if (scratch.defined()) a.scratch = scratch.data_ptr<float>(), a.scratch_floats = scratch.numel();
            a.M = M, a.N = (int32_t)N, a.K = (int32_t)K, a.type = type, a.act = act, a.out_in = out_in;
            if (dx || dw || db) check(dg_linear_grad(&a, stream));
            g_launches += (dx || dw || db) + (a.scratch_floats > 0);
            return out;
        }
        auto weight_gradient = [&](const Tensor& from, int32_t with, const Tensor* dz) {
            const Tensor rows = to_rows(x, &launches), d = out_in ? at::empty({N, K}, options) : at::empty({K, N}, options);
            const Tensor partial = at::empty({dg_linear_dw_scratch(M, (int32_t)N, (int32_t)K, type)}, options.dtype(at::kFloat));
            dg_linear_dw_args a{};
            a.x = rows.data_ptr(), a.ldx = ld_of(rows), a.dy = from.data_ptr(), a.lddy = ld_of(from), a.dw = d.data_ptr();
            a.row_stride = out_in ? 1 : N, a.col_stride = out_in ? K : 1, a.M = M, a.N = (int32_t)N, a.K = (int32_t)K, a.type = type, a.act = with;
            a.scratch = partial.data_ptr<float>(), a.scratch_floats = partial.numel();
            if (dz) {
                if (z.defined()) a.z = z.data_ptr(), a.ldz = ld_of(z);
                a.bits = signs, a.ldbits = ldbits, a.db = db ? out[2].data_ptr() : nullptr;
                if (dz->defined()) a.dz = dz->data_ptr(), a.lddz = dz->stride(0);
            }
            check(dg_linear_dw(&a, stream));
            launches += item == 4 ? 2 * ((K + 255) / 256) * ((N + 255) / 256) : partial.numel() == 0 ? 1 : a.db ? 3 : 2;
            out[1] = out_in ? d.t() : d;
        };
        // 16 bits, x of up to 256 columns: dz and its sums on the way to the weight gradient
        const bool together = item == 2 && dw && K <= 256 && (act != DG_ACT_NONE || db) && on_rows(g) && (!z.defined() || on_rows(z));
        if (together) {
            const Tensor dz = dx && act != DG_ACT_NONE ? whole_rows(M, N, dy) : Tensor();
            weight_gradient(g, act, &dz);
            if (dz.defined()) g = dz;
        } else if (act != DG_ACT_NONE || db || ((dx || dw) && !on_rows(g))) {
            const Tensor dz = (dx || dw) && (act != DG_ACT_NONE || !on_rows(g)) ? whole_rows(M, N, dy) : Tensor();
            const Tensor scratch = db ? at::empty({dg_linear_dz_scratch(M, (int32_t)N)}, options.dtype(at::kFloat)) : Tensor();
            if (dz.defined() || db) {
                check(dg_linear_dz(g.data_ptr(), ld_of(g), z.defined() ? z.data_ptr() : nullptr, z.defined() ? ld_of(z) : 0, signs, ldbits, act,
                                   dz.defined() ? dz.data_ptr() : nullptr, dz.defined() ? dz.stride(0) : 0, db ? out[2].data_ptr() : nullptr, M, (int32_t)N, type,
                                   db ? scratch.data_ptr<float>() : nullptr, stream));
                launches += db && scratch.numel() > 0 ? 2 : 1;
            }
            if (dz.defined()) g = dz;
        }
        if (dx) {
            if (item == 2 && M > dg_linear_few((int32_t)K, (int32_t)N, type)) w = to_rows(w, &launches);
            out[0] = result_rows(M, K, dy);
            dg_linear_args a{};
            a.x = g.data_ptr(), a.ldx = ld_of(g), a.w = w.data_ptr(), a.ldw = ld_of(w), a.out_in = !out_in;
            a.y = out[0].data_ptr(), a.ldy = out[0].stride(0), a.M = M, a.N = (int32_t)K, a.K = (int32_t)N, a.type = type;
            if (splits.defined()) {
                a.ldb = pad4(N), a.head = splits.data_ptr<float>(), a.tail = a.head + K * a.ldb;
            }
            check(dg_linear(&a, stream));
            ++launches;
        }
        if (dw && !together) weight_gradient(g, DG_ACT_NONE, nullptr);
        g_launches += launches;
        return out;
    }
};

Tensor linear(const Tensor& x, const Tensor& w, const std::optional<Tensor>& bias, const std::optional<Tensor>& residual, int64_t act)
{
    auto refuse = [](const std::string& why) { throw std::runtime_error("linear: " + why); };
    auto same = [&](const Tensor& t, const char* what) {
        if (!t.is_cuda()) refuse(std::string(what) + " must be a CUDA tensor: this library has no CPU path");
        if (t.device() != x.device() || t.scalar_type() != x.scalar_type()) refuse(std::string(what) + " must have the type and device of x");
    };
    if (!x.is_cuda()) refuse("x must be a CUDA tensor: this library has no CPU path");
    if (type_of(x) < 0) refuse("x must be fp32, bf16 or fp16");
    if (x.dim() != 2 || w.dim() != 2 || x.size(1) != w.size(0)) {
        std::ostringstream s;
        s << "x must be [M x K] and weight [K x N], got " << x.sizes() << " and " << w.sizes();
        refuse(s.str());
    }
    same(w, "weight");
    const int64_t M = x.size(0), K = x.size(1), N = w.size(1);
    if (K < 1 || N < 1 || K >= (int64_t)1 << 24 || N >= (int64_t)1 << 24 || M >= (int64_t)1 << 31) refuse("sizes out of range");
    if (bias) {
        same(*bias, "bias");
        if (bias->dim() != 1 || bias->size(0) != N) refuse("bias must have one element for every column of weight");
    }
    if (residual) {
        same(*residual, "residual");
        if (residual->dim() != 2 || residual->size(0) != M || residual->size(1) != N) refuse("residual must have the shape of the result");
    }
    const Tensor b = bias.value_or(Tensor()), r = residual.value_or(Tensor());
    for (const Tensor* t : {&x, &w, &b, &r})
        if (t->defined() && t->_fw_grad(0).defined()) refuse("tangents of forward-mode differentiation are not carried on");
    auto wants = [](const Tensor& t) { return t.defined() && t.requires_grad(); };
    const bool train = at::GradMode::is_enabled() && (wants(x) || wants(w) || wants(b) || wants(r));
    c10::cuda::CUDAGuard guard(x.device());
    const int32_t type = type_of(x);
    Tensor y, x2, splits, z, bits;
    Weight weight;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        int64_t launches = 0;
        void* stream = stream_of(x);
        const bool few = M <= dg_linear_few((int32_t)N, (int32_t)K, type);
        weight = stored(w);
        x2 = few ? by_rows(x) : to_rows(x, &launches);
        if (!few && type != DG_FLOAT32) weight.t = to_rows(weight.t, &launches);
        y = few ? at::empty({M, N}, x.options().requires_grad(false)) : result_rows(M, N, x);
        const bool dz = train && (wants(x) || wants(w) || wants(b));
        if (dz && (act == DG_ACT_GELU || act == DG_ACT_SILU)) z = few ? at::empty({M, N}, y.options()) : whole_rows(M, N, x);
        if (dz && act == DG_ACT_RELU) bits = at::empty({M, (N + 63) / 64 * 2}, y.options().dtype(at::kInt));
        dg_linear_args a{};
        Tensor split, res;
        if (!few && type == DG_FLOAT32) {                     // w^T for the product and, where x wants its gradient, w for that: one launch
            const int64_t forward = 2 * N * pad4(K), backward = train && wants(x) ? 2 * K * pad4(N) : 0;
            split = at::empty({forward}, y.options());
            if (backward) splits = at::empty({backward}, y.options());
            const float* from = weight.t.data_ptr<float>();
            dg_split_job jobs[2] = {};
            float* f = split.data_ptr<float>();
            jobs[0] = {from, ld_of(weight.t), f, f + N * pad4(K), pad4(K), (int32_t)N, (int32_t)K, !weight.out_in, 0};
            if (backward) {
                float* h = splits.data_ptr<float>();
                jobs[1] = {from, ld_of(weight.t), h, h + K * pad4(N), pad4(N), (int32_t)K, (int32_t)N, weight.out_in, 0};
            }
            check(dg_dense_split_operands(jobs, backward ? 2 : 1, stream));
            ++launches;
            a.head = f, a.tail = f + N * pad4(K), a.ldb = pad4(K);
        }
        if (r.defined()) {
            res = few ? by_rows(r) : to_rows(r, &launches);
            a.residual = res.data_ptr(), a.ldr = ld_of(res);
        }
        const Tensor flat = b.defined() ? b.contiguous() : b;
        a.x = x2.data_ptr(), a.ldx = ld_of(x2), a.w = weight.t.data_ptr(), a.ldw = ld_of(weight.t), a.out_in = weight.out_in;
        a.bias = flat.defined() ? flat.data_ptr() : nullptr;
        a.y = y.data_ptr(), a.ldy = ld_of(y);
        if (z.defined()) a.z = z.data_ptr(), a.ldz = ld_of(z);
        if (bits.defined()) a.bits = reinterpret_cast<uint32_t*>(bits.data_ptr<int32_t>()), a.ldbits = bits.size(1);
        a.M = M, a.N = (int32_t)N, a.K = (int32_t)K, a.type = type, a.act = (int32_t)act;
        if (M > 0) check(dg_linear(&a, stream));
        g_launches += launches + (M > 0);
    }
    if (train) {
        auto node = std::shared_ptr<LinearNode>(new LinearNode(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(x, w, b, r));
        if (wants(w)) node->x_saved = SavedVariable(x2.is_same(x) ? x : x2.detach(), false);
        if (wants(x) || wants(w)) {
            node->w_copied = weight.t.data_ptr() != w.data_ptr(), node->w_out_in = weight.out_in;
            node->w_saved = SavedVariable(node->w_copied ? weight.t.detach() : w, false);
        }
        if (splits.defined()) node->splits_saved = SavedVariable(splits, false);
        if (z.defined()) node->z_saved = SavedVariable(z, false);
        if (bits.defined()) node->bits_saved = SavedVariable(bits, false);
        node->options = y.options().requires_grad(false);
        node->M = M, node->N = N, node->K = K, node->act = (int32_t)act;
        torch::autograd::set_history(y, node);
    }
    return y;
}

// ---- AdamW over all tensors of an optimiser ----------------------------------------------------------------------------------
// What spmm_cpp.AdamW steps: its parameters and their state, group after group.  A step takes the gradients' addresses anew; whether the optimiser's state
// is still the one this was made from is asked by identity (same_state), without hashing a parameter.
struct AdamwEntry {
    Tensor p, m, v, m_scale, v_scale, step;
    int64_t place;
    int32_t group;
};

struct AdamwTable {
    std::vector<AdamwEntry> entries;
    std::vector<py::object> seen;         // every parameter of the state, its dict and that dict's values, in their order
    Tensor workspace, norm;
    int32_t bits;
    bool captured = false;                // a graph holds addresses of these tensors: they have to live on

    static void walk(PyObject* state, const std::function<bool(PyObject*)>& use)
    {
        PyObject *key, *value, *name, *item;
        Py_ssize_t i = 0;
        while (PyDict_Next(state, &i, &key, &value)) {
            if (!use(key) || !use(value)) return;
            if (!PyDict_Check(value)) continue;
            Py_ssize_t j = 0;
            while (PyDict_Next(value, &j, &name, &item))
                if (!use(item)) return;
        }
    }
    AdamwTable(const py::dict& state, const std::vector<std::tuple<Tensor, Tensor, Tensor, std::optional<Tensor>, std::optional<Tensor>, Tensor, int64_t, int32_t>>& rows,
               int32_t bits_) : bits(bits_)
    {
        walk(state.ptr(), [&](PyObject* o) { return seen.push_back(py::reinterpret_borrow<py::object>(o)), true; });
        const auto kept = bits == 8 ? at::kFloat8_e4m3fn : at::kFloat;
        for (const auto& [p, m, v, ms, vs, step, place, group] : rows) {
            const at::Device device = std::get<0>(rows[0]).device();
            const int64_t n = p.numel(), blocks = (n + 255) / 256;
            auto fits = [&](const Tensor& t, at::ScalarType type, int64_t count) {
                return t.device() == device && t.scalar_type() == type && t.is_contiguous() && t.numel() == count;
            };
            if (!p.is_cuda()) throw std::runtime_error("parameters must be CUDA tensors: this library has no CPU path");
            if (p.device() != device) throw std::runtime_error("parameters must be on one device");
            if (type_of(p) < 0 || !p.is_contiguous()) throw std::runtime_error("parameters must be contiguous fp32, bf16 or fp16 tensors");
            if (!fits(m, kept, n) || !fits(v, kept, n) || !fits(step, at::kLong, 1))
                throw std::runtime_error("optimiser state does not fit its parameter: expected contiguous " + std::string(bits == 8 ? "float8_e4m3fn" : "float32") +
                                         " tensors of its size and an int64 step, on its device");
            if (bits == 8 && (!ms || !vs || !fits(*ms, at::kFloat, blocks) || !fits(*vs, at::kFloat, blocks)))
                throw std::runtime_error("optimiser state does not fit its parameter: expected one float32 scale for every 256 elements");
            entries.push_back({p, m, v, ms.value_or(Tensor()), vs.value_or(Tensor()), step, place, group});
        }
        if (entries.empty()) return;
        std::vector<std::pair<uintptr_t, uintptr_t>> spans;        // all tensors are stepped at once: none may share elements with another
        for (const AdamwEntry& e : entries)
            if (e.p.numel() > 0) spans.emplace_back(reinterpret_cast<uintptr_t>(e.p.data_ptr()), reinterpret_cast<uintptr_t>(e.p.data_ptr()) + e.p.nbytes());
        std::sort(spans.begin(), spans.end());
        for (size_t i = 1; i < spans.size(); ++i)
            if (spans[i].first < spans[i - 1].second) throw std::runtime_error("parameters must not share memory");
        c10::cuda::CUDAGuard guard(entries[0].p.device());
        std::vector<dg_adamw_tensor> all;
        for (const AdamwEntry& e : entries) {
            dg_adamw_tensor t{};
            t.n = e.p.numel(), t.type = type_of(e.p);
            all.push_back(t);
        }
        const int64_t bytes = dg_adamw_workspace(all.data(), (int32_t)all.size());
        if (bytes < 0) check((int)bytes);
        workspace = at::zeros({bytes}, entries[0].p.options().dtype(at::kByte).requires_grad(false));
        norm = at::zeros({2}, entries[0].p.options().dtype(at::kFloat).requires_grad(false));
    }
    bool same_state(const py::dict& state) const
    {
        size_t i = 0;
        bool same = true;
        walk(state.ptr(), [&](PyObject* o) { return same = i < seen.size() && seen[i++].ptr() == o; });
        return same && i == seen.size();
    }
    // groups: (lr, beta1, beta2, eps, weight decay) each
    void step(const std::vector<std::tuple<double, double, double, double, double>>& groups, double max_norm, uint32_t seed)
    {
        if (entries.empty()) return;
        const at::Device device = entries[0].p.device();
        c10::cuda::CUDAGuard guard(device);
        std::vector<dg_adamw_tensor> all;
        std::vector<Tensor> copies;                       // of gradients whose elements do not lie side by side
        std::vector<size_t> end(groups.size(), 0);
        all.reserve(entries.size());
        for (const AdamwEntry& e : entries) {
            const Tensor& grad = e.p.grad();
            if (grad.defined() && e.p.numel() > 0) {
                if (grad.layout() != at::kStrided) throw std::runtime_error("AdamW takes dense gradients only");
                if (e.p.device() != device || e.p.numel() != e.m.numel() || !e.p.is_contiguous() || grad.device() != device ||
                    grad.scalar_type() != e.p.scalar_type() || grad.sizes() != e.p.sizes())
                    throw std::runtime_error("a parameter or its gradient has changed its device, type, size or layout");
                const Tensor* g = &grad;
                if (!grad.is_contiguous()) {
                    copies.push_back(grad.contiguous());
                    g = &copies.back();
                }
                const bool small = bits == 8;
                all.push_back({e.p.data_ptr(), g->data_ptr(), e.m.data_ptr(), e.v.data_ptr(), small ? e.m_scale.data_ptr<float>() : nullptr,
                               small ? e.v_scale.data_ptr<float>() : nullptr, e.step.data_ptr<int64_t>(), e.p.numel(), e.place, type_of(e.p), 0});
            }
            end[e.group] = all.size();
        }
        if (all.empty()) return;
        void* stream = stream_of(entries[0].p);
        captured |= c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None;
        const bool clipped = max_norm > 0;
        if (clipped) check(dg_grad_norm(all.data(), (int32_t)all.size(), max_norm, norm.data_ptr<float>(), workspace.data_ptr(), workspace.numel(), stream));
        size_t first = 0;
        for (size_t k = 0; k < groups.size(); ++k) {
            const size_t last = std::max(end[k], first);
            const auto& [lr, beta1, beta2, eps, decay] = groups[k];
            const dg_adamw_options options{lr, beta1, beta2, eps, decay, seed, bits};
            if (last > first)
                check(dg_adamw_step(all.data() + first, (int32_t)(last - first), &options, clipped ? norm.data_ptr<float>() + 1 : nullptr, workspace.data_ptr(),
                                    workspace.numel(), stream));
            first = last;
        }
        for (const AdamwEntry& e : entries) {             // copies that are kept of a weight go by its version
            if (!e.p.grad().defined()) continue;
            for (const Tensor* t : {&e.p, &e.m, &e.v, &e.m_scale, &e.v_scale, &e.step})
                if (t->defined()) t->unsafeGetTensorImpl()->bump_version();
        }
    }
};

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m)
{
    py::class_<PlanRef, std::shared_ptr<PlanRef>>(m, "PlanRef").def(py::init<int64_t, Tensor, Tensor>());
    py::class_<AdamwTable>(m, "AdamwTable")
        .def(py::init<const py::dict&, const std::vector<std::tuple<Tensor, Tensor, Tensor, std::optional<Tensor>, std::optional<Tensor>, Tensor, int64_t, int32_t>>&, int32_t>())
        .def("same_state", &AdamwTable::same_state)
        .def("step", &AdamwTable::step)
        .def_readonly("captured", &AdamwTable::captured)
        .def_readonly("norm", &AdamwTable::norm);
    m.def("linear", &linear);
    m.def("spmm", &spmm);
    m.def("gcn", &gcn);
    m.def("readable_padded", &readable_padded);
    m.def("tn_scratch", &tn_scratch);
    m.def("row_cross_entropy", &row_cross_entropy);
    m.def("pending_regions", &pending_regions);
    m.def("resolve_regions", &resolve_regions);
    m.def("take_launches", [] { return g_launches.exchange(0); });
}
