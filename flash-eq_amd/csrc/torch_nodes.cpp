// PyTorch bindings of the layer norm, the expert routing and the fine-tuning operators (dropout, biased edge
// attention, adapters): argument checks, outputs and workspaces from the caching allocator, autograd nodes, and the calls of the C ABI
// (flasheq.h) on the tensors' device and its current stream.
//
// A training call of a small graph is host work: a torch.autograd.Function spends about 20 us forward
// and 70 us backward in Python (an engine thread waits for the interpreter lock for each node), nodes
// written here a third of it.  Nothing here synchronises, and no Python runs between the checks
// and the launches, so the interpreter lock is released.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <pybind11/pybind11.h>
#include <pybind11/stl.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/utils/pybind.h>

#include "flasheq.h"

namespace {

namespace py = pybind11;
using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
typedef std::optional<Tensor> OptTensor;

constexpr int64_t kMaxExperts = 1024, kMaxTopk = 64;

// ---- checks --------------------------------------------------------------------------

// A tensor off the GPU: CUDANotAvailableError in Python.
struct NotOnGpu : std::runtime_error {
    using std::runtime_error::runtime_error;
};

template <class... A>
[[noreturn]] void value_error(const A&... a) { throw py::value_error(c10::str(a...)); }
template <class... A>
[[noreturn]] void type_error(const A&... a) { throw py::type_error(c10::str(a...)); }

const char* dtype_name(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return "torch.float32";
        case at::kHalf: return "torch.float16";
        case at::kBFloat16: return "torch.bfloat16";
        case at::kDouble: return "torch.float64";
        case at::kLong: return "torch.int64";
        case at::kInt: return "torch.int32";
        case at::kBool: return "torch.bool";
        default: return c10::toString(t);
    }
}

void need_gpu(const Tensor& t, const char* name) {
    if (!t.is_cuda())
        throw NotOnGpu(c10::str(name, " must be a GPU tensor: the flash-eq hot path runs only on the GPU (got device ",
                                t.device(), ")."));
}

// feq_dtype of a GPU tensor.
int code_of(const Tensor& t, const char* name) {
    need_gpu(t, name);
    switch (t.scalar_type()) {
        case at::kFloat: return FEQ_F32;
        case at::kHalf: return FEQ_F16;
        case at::kBFloat16: return FEQ_BF16;
        default: type_error(name, ": dtype ", dtype_name(t.scalar_type()), " is not supported (float32, float16 or bfloat16)");
    }
}

void same_device(const Tensor& a, const Tensor& b) {
    if (a.device() != b.device()) value_error("tensors on different devices: ", a.device(), " and ", b.device());
}

void done(int rc, const char* what) {
    if (rc != FEQ_OK) throw std::runtime_error(c10::str(what, ": ", feq_last_error(), " (code ", rc, ")"));
}

// ---- tensors -------------------------------------------------------------------------

bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }
const Tensor& get(const OptTensor& t) {
    static const Tensor none;
    return t.has_value() ? *t : none;
}

Tensor dense_long(const Tensor& t) {
    return !t.defined() ? t : (t.scalar_type() == at::kLong ? t : t.to(at::kLong)).contiguous();
}
Tensor dense(const Tensor& t) { return t.is_contiguous() ? t : t.contiguous(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
template <class T>
T* ptr_as(const Tensor& t) { return static_cast<T*>(ptr(t)); }

Tensor make(at::IntArrayRef shape, const Tensor& like, at::ScalarType dtype) {
    return at::empty(shape, like.options().dtype(dtype));
}
Tensor scratch(size_t bytes, const Tensor& like) {
    return bytes ? make({static_cast<int64_t>(bytes)}, like, at::kByte) : Tensor();
}
size_t bytes_of(const Tensor& t) { return t.defined() ? static_cast<size_t>(t.numel()) : 0; }

// Launches go to the device of `t` and its current stream.
struct On {
    c10::DeviceGuard guard;
    feq_stream_t stream;
    explicit On(const Tensor& t)
        : guard(t.device()), stream(reinterpret_cast<feq_stream_t>(c10::hip::getCurrentHIPStream(t.device().index()).stream())) {}
};

// ---- autograd ------------------------------------------------------------------------

// The backward of every node below runs once: under create_graph its results carry an error
// for a second derivative instead of being constants without one.
variable_list once(variable_list&& grads, const char* ops) {
    if (!at::GradMode::is_enabled()) return std::move(grads);
    for (auto& g : grads)
        if (g.defined()) g = g.detach().requires_grad_();
    auto error = std::make_shared<torch::autograd::DelayedError>(
        c10::str(ops, " of flash_eq have no second derivative"), static_cast<int64_t>(grads.size()));
    return (*error)(std::move(grads));
}

struct OnceNode : torch::autograd::Node {
    static constexpr const char* kOps = "the layer norm and the expert routing";     // as errors name them
    variable_list apply(variable_list&& grads) final {
        variable_list out;
        {
            std::lock_guard<std::mutex> lock(mutex_);      // a backward of the same graph in another thread frees
            at::NoGradGuard none;
            out = backward(grads);
        }
        return once(std::move(out), ops());
    }
    void release_variables() final {
        std::lock_guard<std::mutex> lock(mutex_);
        release();
    }
    virtual variable_list backward(variable_list& grads) = 0;
    virtual void release() {}
    virtual const char* ops() const { return kOps; }
    bool need(size_t i) const { return task_should_compute_output(i); }
};

// The node of a call whose inputs `in` some gradient may reach, else none.
template <class N, class... In>
std::shared_ptr<N> node_for(const In&... in) {
    TORCH_CHECK_NOT_IMPLEMENTED(!(torch::autograd::isFwGradDefined(in) || ...),
                                N::kOps, " of flash_eq have no forward-mode derivative");
    if (!at::GradMode::is_enabled() || !(wants_grad(in) || ...)) return nullptr;
    std::shared_ptr<N> node(new N(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(in...));
    return node;
}

// A tensor kept for the backward; in-place changes until then are errors.  A saved-tensor hook may hand out
// another tensor: one of other strides is copied, one that could not stand for the kept one is refused.
class Kept {
   public:
    // `output`: of the node that keeps it
    void keep(const Tensor& t, bool output = false) {
        saved_ = SavedVariable(t, output);
        defined_ = t.defined();
        if (!defined_) return;
        sizes_.assign(t.sizes().begin(), t.sizes().end());
        type_ = t.scalar_type();
        device_ = t.device();
    }
    // As kept, its rows apart where they were (rows_of takes those).
    Tensor get(std::shared_ptr<torch::autograd::Node> node = nullptr) const {
        Tensor t = saved_.unpack(std::move(node));
        TORCH_CHECK(t.defined() == defined_, "a saved-tensor hook returned no tensor");
        if (defined_)
            TORCH_CHECK(t.sizes() == at::IntArrayRef(sizes_) && t.scalar_type() == type_ && t.device() == device_,
                        "a saved-tensor hook returned a ", dtype_name(t.scalar_type()), " tensor of shape ", t.sizes(), " on ",
                        t.device(), " for a ", dtype_name(type_), " one of shape ", at::IntArrayRef(sizes_), " on ", device_);
        return t;
    }
    Tensor get_dense(std::shared_ptr<torch::autograd::Node> node = nullptr) const {
        const Tensor t = get(std::move(node));
        return t.defined() ? dense(t) : t;
    }
    void reset_data() { saved_.reset_data(); }

   private:
    SavedVariable saved_;
    bool defined_ = false;
    c10::SmallVector<int64_t, 4> sizes_;
    at::ScalarType type_ = at::kFloat;
    c10::Device device_ = at::kCPU;
};

// ---- layer norm ----------------------------------------------------------------------

// `t` or a contiguous copy, and the distance of its rows: two-dimensional tables whose rows lie
// apart (a slice of a wider table) are read where they are.
Tensor rows_of(const Tensor& t, int64_t& ld) {
    ld = t.size(-1);
    if (t.is_contiguous()) return t;
    if (t.dim() == 2 && t.stride(1) == 1 && t.stride(0) >= t.size(1)) {
        ld = t.stride(0);
        return t;
    }
    return t.contiguous();
}

struct LayerNormNode final : OnceNode {
    Kept x, w;
    Tensor stats;             // (2, rows): mean, 1 / standard deviation
    int pdtype = 0;           // feq_dtype of the parameters
    at::ScalarType ptype = at::kFloat;

    variable_list backward(variable_list& grads) override {
        variable_list out(3);
        if (!grads[0].defined()) return out;
        const Tensor xs = x.get(), ws = w.get_dense();
        int64_t ldx, ldg;
        const Tensor xr = rows_of(xs, ldx), g = rows_of(grads[0], ldg);
        const int64_t width = xr.size(-1), rows = xr.numel() / width;
        const bool nx = need(0), nw = need(1), nb = need(2);
        if (nx) out[0] = make(xr.sizes(), xr, xr.scalar_type());
        if (nw) out[1] = make({width}, xr, ptype);
        if (nb) out[2] = make({width}, xr, ptype);
        const Tensor ws_ = (nw || nb) ? scratch(feq_layernorm_bwd_workspace(rows, width, code_of(xr, "x")), xr) : Tensor();
        On on(xr);
        done(feq_layernorm_bwd(ptr(g), ldg, ptr(xr), rows, width, ldx, code_of(xr, "x"), ptr(ws), pdtype,
                               ptr_as<float>(stats), ptr_as<float>(stats) + rows, ptr(out[0]), ptr(out[1]), ptr(out[2]),
                               ptr(ws_), bytes_of(ws_), on.stream),
             "feq_layernorm_bwd");
        return out;
    }
    void release() override {
        x.reset_data();
        w.reset_data();
        stats.reset();
    }
    std::string name() const override { return "FeqLayerNormBackward"; }
};

Tensor layer_norm(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
    const int code = code_of(x, "x");
    if (x.dim() < 1 || x.size(-1) < 1) value_error("x must have a last axis to normalise, got shape ", x.sizes());
    const int64_t width = x.size(-1);
    const Tensor &w = get(weight), &b = get(bias);
    int pcode = FEQ_F32;
    for (const auto& [t, name] : {std::pair<const Tensor&, const char*>{w, "weight"}, {b, "bias"}}) {
        if (!t.defined()) continue;
        pcode = code_of(t, name);
        if (t.dim() != 1 || t.size(0) != width) value_error(name, " must have shape (", width, ",), got ", t.sizes());
        same_device(x, t);
    }
    if (w.defined() && b.defined() && w.scalar_type() != b.scalar_type())
        type_error("weight and bias of different dtypes: ", dtype_name(w.scalar_type()), " and ", dtype_name(b.scalar_type()));
    const auto node = node_for<LayerNormNode>(x, w, b);
    Tensor y;
    {
        at::NoGradGuard none;
        int64_t ld;
        const Tensor xs = rows_of(x, ld), wc = w.defined() ? dense(w) : w, bc = b.defined() ? dense(b) : b;
        const int64_t rows = xs.numel() / width;
        y = make(x.sizes(), x, x.scalar_type());
        Tensor stats;
        if (node) stats = make({2, rows}, x, at::kFloat);
        On on(x);
        done(feq_layernorm_fwd(ptr(xs), rows, width, ld, code, ptr(wc), ptr(bc), pcode, static_cast<float>(eps), ptr(y),
                               ptr_as<float>(stats), stats.defined() ? ptr_as<float>(stats) + rows : nullptr, on.stream),
             "feq_layernorm_fwd");
        if (node) {
            node->x.keep(xs);
            node->w.keep(wc);
            node->stats = stats;
            node->pdtype = pcode;
            node->ptype = w.defined() ? w.scalar_type() : b.defined() ? b.scalar_type() : at::kFloat;
        }
    }
    if (node) torch::autograd::set_history(y, node);
    return y;
}

// ---- top-k ---------------------------------------------------------------------------

struct TopkNode final : OnceNode {
    Kept logits, ids, weights;      // weights: the node's own first output
    bool normalize = true;

    variable_list backward(variable_list& grads) override {
        variable_list out(1);
        if (!grads[0].defined() && !grads[1].defined()) return out;
        const Tensor l = logits.get_dense(), chosen = ids.get_dense(), w = weights.get_dense(shared_from_this());
        const Tensor gw = grads[0].defined() ? dense(grads[0]) : Tensor(), gm = grads[1].defined() ? dense(grads[1]) : Tensor();
        out[0] = make(l.sizes(), l, l.scalar_type());
        On on(l);
        done(feq_expert_topk_bwd(ptr(l), ptr_as<int64_t>(chosen), ptr_as<float>(w), ptr_as<float>(gw), ptr_as<float>(gm),
                                 l.size(0), l.size(1), code_of(l, "logits"), chosen.size(1), normalize, ptr(out[0]), on.stream),
             "feq_expert_topk_bwd");
        return out;
    }
    void release() override {
        logits.reset_data();
        ids.reset_data();
        weights.reset_data();
    }
    std::string name() const override { return "FeqExpertTopkBackward"; }
};

// logits (rows, experts)
std::tuple<Tensor, Tensor, Tensor> expert_topk(const Tensor& logits, int64_t top_k, bool normalize) {
    const int code = code_of(logits, "logits");
    if (logits.dim() < 1) value_error("logits must be (..., experts)");
    const int64_t experts = logits.size(-1);
    if (experts < 1 || experts > kMaxExperts) value_error("experts must be 1 to ", kMaxExperts, ", got ", experts);
    if (top_k < 1 || top_k > std::min(experts, kMaxTopk))
        value_error("top_k must be 1 to ", std::min(experts, kMaxTopk), " of ", experts, " experts, got ", top_k);
    const Tensor flat = logits.dim() == 2 ? logits : logits.reshape({-1, experts});
    const auto node = node_for<TopkNode>(flat);
    const int64_t rows = flat.size(0);
    Tensor ids, weights, mean;
    {
        at::NoGradGuard none;
        const Tensor lc = dense(flat);
        ids = make({rows, top_k}, lc, at::kLong);
        weights = make({rows, top_k}, lc, at::kFloat);
        mean = make({experts}, lc, at::kFloat);
        const Tensor ws = scratch(feq_expert_topk_workspace(rows, static_cast<int32_t>(experts)), lc);
        On on(lc);
        done(feq_expert_topk_fwd(ptr(lc), rows, experts, code, top_k, normalize, ptr_as<int64_t>(ids), ptr_as<float>(weights),
                                 ptr_as<float>(mean), ptr(ws), bytes_of(ws), on.stream),
             "feq_expert_topk_fwd");
        if (node) {
            node->logits.keep(lc);
            node->ids.keep(ids);
            node->normalize = normalize;
        }
    }
    if (node) {
        torch::autograd::set_history(weights, node);
        torch::autograd::set_history(mean, node);
        node->weights.keep(weights, true);
    }
    if (logits.dim() != 2) {
        auto shape = logits.sizes().vec();
        shape.back() = top_k;
        ids = ids.view(shape);
        weights = weights.view(shape);
    }
    return {ids, weights, mean};
}

// ---- plan and rows -------------------------------------------------------------------

std::tuple<Tensor, Tensor, Tensor> expert_plan(const Tensor& ids, int64_t experts) {
    need_gpu(ids, "ids");
    if (!at::isIntegralType(ids.scalar_type(), false)) type_error("ids must be integers, got ", dtype_name(ids.scalar_type()));
    if (ids.dim() != 1 && ids.dim() != 2) value_error("ids must be (rows, top_k) or (rows,), got shape ", ids.sizes());
    if (experts < 1 || experts > kMaxExperts) value_error("num_experts must be 1 to ", kMaxExperts, ", got ", experts);
    const int64_t k = ids.dim() == 2 ? ids.size(1) : 1;
    if (k < 1 || k > kMaxTopk) value_error("top_k must be 1 to ", kMaxTopk, ", got ", k);
    const int64_t slots = ids.size(0) * k;
    if (slots > (int64_t{1} << 30)) value_error("more than 2^30 slots: ", slots);
    at::NoGradGuard none;
    c10::InferenceMode tracked(false);      // in-place changes of a plan made in inference mode are counted too (check_plan)
    at::AutoDispatchBelowADInplaceOrView uncounted;   // at::empty fills what it makes where algorithms have to be deterministic
    const Tensor flat = dense(ids.scalar_type() == at::kLong ? ids : ids.to(at::kLong));
    Tensor order = make({slots}, flat, at::kInt), positions = make({ids.size(0), k}, flat, at::kInt),
           offsets = make({experts + 1}, flat, at::kInt);
    const Tensor ws = scratch(feq_expert_plan_workspace(slots, static_cast<int32_t>(experts)), flat);
    On on(flat);
    done(feq_expert_plan(ptr_as<int64_t>(flat), slots, experts, ptr_as<int32_t>(order), ptr_as<int32_t>(positions),
                         ptr_as<int32_t>(offsets), ptr(ws), bytes_of(ws), on.stream),
         "feq_expert_plan");
    return {order, positions, offsets};
}

// The kernels write to the places a plan holds, so one whose tensors are not those that expert_plan
// returned, as it returned them, is refused.  Theirs are no inference tensors, whose changes nothing counts.
void check_plan(const Tensor& t, const char* name, int64_t dims) {
    need_gpu(t, name);
    if (t.scalar_type() != at::kInt || t.dim() != dims || !t.is_contiguous() || t.is_inference())
        value_error("not an ExpertPlan's ", name, ": ", dtype_name(t.scalar_type()), " of shape ", t.sizes());
    TORCH_CHECK(t._version() == 0, "the ", name, " of an ExpertPlan have been modified in place");
}

// A copy of a plan's tensor (any device) that check_plan takes: of version 0, no inference tensor.
Tensor plan_copy(const Tensor& t) {
    c10::InferenceMode tracked(false);
    at::AutoDispatchBelowADInplaceOrView uncounted;      // a clone of an inference tensor is filled in place
    return t.clone();
}

// A plan as the row moves need it.
struct Places {
    Tensor positions, offsets;
    int64_t rows() const { return positions.size(0); }
    int64_t k() const { return positions.size(1); }
    int64_t slots() const { return positions.numel(); }
    const int32_t* placed() const { return ptr_as<int32_t>(offsets) + offsets.numel() - 1; }
    void check() const {
        check_plan(positions, "positions", 2);
        check_plan(offsets, "offsets", 1);
    }
};

void check_table(const Tensor& t, const char* name, int64_t rows, const Places& p) {
    code_of(t, name);
    p.check();
    same_device(p.positions, t);
    if (t.dim() < 2 || t.size(-2) != rows) value_error(name, " must be (..., ", rows, ", width), got shape ", t.sizes());
}

int64_t planes_of(const Tensor& t) { return t.numel() / (t.size(-1) * t.size(-2)); }

Tensor like_table(const Tensor& t, int64_t rows) {
    c10::SmallVector<int64_t, 6> shape(t.sizes().begin(), t.sizes().end());
    shape[shape.size() - 2] = rows;
    return make(shape, t, t.scalar_type());
}

// Sums of the places of every row, weighted or not.
Tensor combined(const Places& p, const Tensor& ys, const Tensor& weights) {
    Tensor y = like_table(ys, p.rows());
    if (y.numel() == 0) return y;
    On on(ys);
    done(feq_expert_combine(ptr(ys), planes_of(ys), p.rows(), p.k(), ys.size(-1), code_of(ys, "ys"),
                            ptr_as<int32_t>(p.positions), p.placed(), ptr(weights),
                            weights.defined() ? code_of(weights, "weights") : FEQ_F32, ptr(y), on.stream),
         "feq_expert_combine");
    return y;
}

struct DispatchNode final : OnceNode {
    Places places;
    variable_list backward(variable_list& grads) override {
        variable_list out(1);
        places.check();
        if (grads[0].defined()) out[0] = combined(places, dense(grads[0]), Tensor());
        return out;
    }
    std::string name() const override { return "FeqExpertDispatchBackward"; }
};

Tensor expert_dispatch(const Tensor& x, const Tensor& positions, const Tensor& offsets) {
    const Places p{positions, offsets};
    check_table(x, "x", p.rows(), p);
    const auto node = node_for<DispatchNode>(x);
    Tensor xs;
    {
        at::NoGradGuard none;
        const Tensor xc = dense(x);
        xs = like_table(x, p.slots());
        if (xs.numel()) {
            On on(x);
            done(feq_expert_dispatch(ptr(xc), planes_of(xc), p.rows(), p.k(), xc.size(-1), code_of(xc, "x"),
                                     ptr_as<int32_t>(positions), p.placed(), ptr(xs), on.stream),
                 "feq_expert_dispatch");
        }
    }
    if (node) {
        node->places = p;
        torch::autograd::set_history(xs, node);
    }
    return xs;
}

struct CombineNode final : OnceNode {
    Kept ys, weights;
    Places places;
    variable_list backward(variable_list& grads) override {
        variable_list out(2);
        if (!grads[0].defined()) return out;
        const Tensor in = ys.get_dense(), w = weights.get_dense(), g = dense(grads[0]);   // an error when they have been freed
        places.check();
        if (need(0)) out[0] = make(in.sizes(), in, in.scalar_type());
        if (need(1)) out[1] = make(w.sizes(), w, w.scalar_type());
        if (in.numel()) {
            On on(in);
            done(feq_expert_combine_bwd(ptr(g), ptr(in), planes_of(in), places.rows(), places.k(), in.size(-1),
                                        code_of(in, "ys"), ptr_as<int32_t>(places.positions), places.placed(), ptr(w),
                                        code_of(w, "weights"), ptr(out[0]), ptr(out[1]), on.stream),
                 "feq_expert_combine_bwd");
        } else if (out[1].defined()) {
            out[1].zero_();
        }
        return out;
    }
    void release() override {
        ys.reset_data();
        weights.reset_data();
        places = Places();
    }
    std::string name() const override { return "FeqExpertCombineBackward"; }
};

Tensor expert_combine(const Tensor& ys, const Tensor& weights, const Tensor& positions, const Tensor& offsets) {
    const Places p{positions, offsets};
    check_table(ys, "ys", p.slots(), p);
    code_of(weights, "weights");
    same_device(ys, weights);
    const bool flat = weights.dim() == 1 && p.k() == 1;
    if (!(flat && weights.size(0) == p.rows()) &&
        !(weights.dim() == 2 && weights.size(0) == p.rows() && weights.size(1) == p.k()))
        value_error("weights must be (", p.rows(), ", ", p.k(), "), got shape ", weights.sizes());
    const auto node = node_for<CombineNode>(ys, weights);
    Tensor y;
    {
        at::NoGradGuard none;
        const Tensor yc = dense(ys), wc = dense(weights);
        y = combined(p, yc, wc);
        if (node) {
            node->ys.keep(yc);
            node->weights.keep(wc);
            node->places = p;
        }
    }
    if (node) torch::autograd::set_history(y, node);
    return y;
}

// ---- the experts' maps ---------------------------------------------------------------

// Degrees of the irreps and the bias column of each: its number among the scalar ones, -1 for the others.
struct Irreps {
    std::vector<int32_t> lvals, cols;
    int64_t dim = 0, nscalar = 0;
    explicit Irreps(const std::vector<int64_t>& l) {
        for (const int64_t v : l) {
            if (v < 0 || v > FEQ_MAX_SLOTS) value_error("lvals must be non-negative degrees of at most ", FEQ_MAX_SLOTS / 2);
            lvals.push_back(static_cast<int32_t>(v));
            cols.push_back(v == 0 ? static_cast<int32_t>(nscalar++) : -1);
            dim += 2 * v + 1;
        }
        if (l.empty()) value_error("lvals must be non-negative degrees, got none");
    }
    int32_t n() const { return static_cast<int32_t>(lvals.size()); }
};

struct ExpertLinearNode final : OnceNode {
    Kept x, weight;
    Tensor offsets;
    Irreps irreps{{0}};
    int64_t nbias = 0;

    variable_list backward(variable_list& grads) override {
        variable_list out(3);
        if (!grads[0].defined()) return out;
        const Tensor xs = x.get_dense(), w = weight.get_dense(), g = dense(grads[0]);     // an error when they have been freed
        check_plan(offsets, "offsets", 1);
        const int64_t experts = w.size(0), co = w.size(2), ci = w.size(3), slots = xs.size(-2);
        const int code = code_of(xs, "x");
        On on(xs);
        const int32_t *lv = irreps.lvals.data(), n = irreps.n(), *off = ptr_as<int32_t>(offsets);
        const int32_t nb = need(2) ? static_cast<int32_t>(nbias) : 0;
        Tensor gw, gb, ws;
        if (need(0)) out[0] = make(xs.sizes(), xs, xs.scalar_type());
        if (need(1) || need(2)) gw = make(w.sizes(), w, w.scalar_type());
        if (nb) gb = make({experts, co, nbias}, w, w.scalar_type());
        if (gw.defined()) ws = scratch(feq_expert_linear_bwd_workspace(lv, n, experts, slots, ci, co, nb), xs);
        if (need(0) && gw.defined())
            done(feq_expert_linear_bwd(lv, n, experts, slots, ci, co, code, ptr(g), ptr(xs), ptr(w), off, nb, irreps.cols.data(),
                                       ptr(out[0]), ptr(gw), ptr(gb), ptr(ws), bytes_of(ws), on.stream),
                 "feq_expert_linear_bwd");
        else if (need(0))
            done(feq_expert_linear_bwd_x(lv, n, experts, slots, ci, co, code, ptr(g), ptr(w), off, ptr(out[0]), on.stream),
                 "feq_expert_linear_bwd_x");
        else if (gw.defined())
            done(feq_expert_linear_bwd_w(lv, n, experts, slots, ci, co, code, ptr(g), ptr(xs), off, nb, irreps.cols.data(),
                                         ptr(gw), ptr(gb), ptr(ws), bytes_of(ws), on.stream),
                 "feq_expert_linear_bwd_w");
        if (need(1)) out[1] = gw;
        if (need(2)) out[2] = gb;
        return out;
    }
    void release() override {
        x.reset_data();
        weight.reset_data();
        offsets.reset();
    }
    std::string name() const override { return "FeqExpertLinearBackward"; }
};

Tensor expert_linear(const Tensor& x, const Tensor& weight, const OptTensor& bias, const Tensor& offsets, int64_t slots,
                     const std::vector<int64_t>& lvals) {
    const Irreps irreps(lvals);
    const int code = code_of(x, "x");
    const Tensor& b = get(bias);
    for (const auto& [t, name] : {std::pair<const Tensor&, const char*>{weight, "weight"}, {b, "bias"}}) {
        if (!t.defined()) continue;
        code_of(t, name);
        if (t.scalar_type() != x.scalar_type())
            type_error("x and ", name, " of different dtypes: ", dtype_name(x.scalar_type()), " and ", dtype_name(t.scalar_type()));
        same_device(x, t);
    }
    check_plan(offsets, "offsets", 1);
    same_device(x, offsets);
    const int64_t experts = offsets.size(0) - 1;
    if (weight.dim() != 4 || weight.size(0) != experts || weight.size(1) != irreps.n())
        value_error("weight must be (", experts, ", ", irreps.n(), ", cout, cin), got shape ", weight.sizes());
    const int64_t co = weight.size(2), ci = weight.size(3);
    const bool flat = x.dim() == 2 && irreps.n() == 1 && irreps.dim == 1;
    if (!(flat && x.size(0) == slots && x.size(1) == ci) &&
        !(x.dim() == 3 && x.size(0) == irreps.dim && x.size(1) == slots && x.size(2) == ci))
        value_error("x must be (", irreps.dim, ", ", slots, ", ", ci, "), got shape ", x.sizes());
    if (ci < 1 || co < 1) value_error("weight has no channels: shape ", weight.sizes());
    if (b.defined() && (irreps.nscalar == 0 || b.dim() != 3 || b.size(0) != experts || b.size(1) != co || b.size(2) != irreps.nscalar))
        value_error("bias must be (", experts, ", ", co, ", ", irreps.nscalar, "), one column per scalar irrep, got shape ", b.sizes());
    const auto node = node_for<ExpertLinearNode>(x, weight, b);
    Tensor y;
    {
        at::NoGradGuard none;
        const Tensor xc = dense(x), wc = dense(weight), bc = b.defined() ? dense(b) : b;
        c10::SmallVector<int64_t, 3> shape(x.sizes().begin(), x.sizes().end());
        shape.back() = co;
        y = make(shape, x, x.scalar_type());
        On on(x);
        done(feq_expert_linear_fwd(irreps.lvals.data(), irreps.n(), experts, slots, ci, co, code, ptr(xc), ptr(wc),
                                   ptr_as<int32_t>(offsets), ptr(bc), static_cast<int32_t>(irreps.nscalar), irreps.cols.data(),
                                   ptr(y), on.stream),
             "feq_expert_linear_fwd");
        if (node) {
            node->x.keep(xc);
            node->weight.keep(wc);
            node->offsets = offsets;
            node->irreps = irreps;
            node->nbias = irreps.nscalar;
        }
    }
    if (node) torch::autograd::set_history(y, node);
    return y;
}

// ---- dropout -------------------------------------------------------------------------

struct TuneNode : OnceNode {
    static constexpr const char* kOps = "the dropout, edge attention and adapters";
    const char* ops() const override { return kOps; }
};

void check_share(double p) {
    if (!(p >= 0.0 && p <= 1.0)) value_error("dropout must be between 0 and 1, got ", p);
}

// The seed of a dropout of `like`: one int64 on its device.
void check_seed(const Tensor& seed, const Tensor& like) {
    need_gpu(seed, "seed");
    if (seed.scalar_type() != at::kLong || seed.numel() != 1)
        value_error("seed must be one int64 (dropout_seed), got ", dtype_name(seed.scalar_type()), " of shape ", seed.sizes());
    same_device(like, seed);
}

struct DropoutCall {
    std::vector<int32_t> lvals;
    bool cm = false;
    double p = 0.0;

    Tensor run(const Tensor& x, const Tensor& seed) const {
        Tensor y = make(x.sizes(), x, x.scalar_type());
        int64_t dim = 0;
        for (const int32_t l : lvals) dim += 2 * l + 1;
        On on(x);
        done(feq_dropout(lvals.data(), static_cast<int32_t>(lvals.size()), x.numel() / dim, cm, code_of(x, "x"), ptr(x), p,
                         ptr_as<int64_t>(seed), ptr(y), on.stream),
             "feq_dropout");
        return y;
    }
};

struct DropoutNode final : TuneNode {
    Kept seed;
    DropoutCall call;

    variable_list backward(variable_list& grads) override {
        const Tensor s = seed.get();                     // an error when it has been freed
        if (!grads[0].defined()) return {Tensor()};
        return {call.run(dense(grads[0]), s)};
    }
    void release() override { seed.reset_data(); }
    std::string name() const override { return "FeqDropoutBackward"; }
};

// `lvals` none: element by element.
Tensor feature_dropout(const Tensor& x, double p, const Tensor& seed, const std::optional<std::vector<int64_t>>& lvals, bool cm) {
    code_of(x, "x");
    check_share(p);
    check_seed(seed, x);
    DropoutCall call{{0}, cm && lvals.has_value(), p};
    if (lvals) {
        const Irreps irreps(*lvals);
        call.lvals = irreps.lvals;
        if (irreps.n() > FEQ_MAX_IRREPS || irreps.dim > FEQ_MAX_SLOTS)
            value_error("at most ", FEQ_MAX_IRREPS, " irreps and ", FEQ_MAX_SLOTS, " components, got ", irreps.n(), " and ", irreps.dim);
        if (x.dim() < 1 || x.size(cm ? 0 : -1) != irreps.dim)
            value_error("x must be ", cm ? "(" : "(..., ", irreps.dim, cm ? ", ...)" : ")", ", got shape ", x.sizes());
    }
    const auto node = node_for<DropoutNode>(x);
    Tensor y;
    {
        at::NoGradGuard none;
        y = call.run(dense(x), seed);
        if (node) {
            node->seed.keep(seed);
            node->call = call;
        }
    }
    if (node) torch::autograd::set_history(y, node);
    return y;
}

// ---- biased edge attention -----------------------------------------------------------

Tensor distance_buckets(const Tensor& dist, const Tensor& bounds) {
    need_gpu(dist, "distances");
    need_gpu(bounds, "boundaries");
    for (const auto& [t, name] : {std::pair<const Tensor&, const char*>{dist, "distances"}, {bounds, "boundaries"}})
        if (t.scalar_type() != at::kFloat) type_error(name, " must be float32, got ", dtype_name(t.scalar_type()));
    if (dist.dim() != 1 || bounds.dim() != 1)
        value_error("distances (edges,) and boundaries (buckets - 1,) expected, got shapes ", dist.sizes(), " and ", bounds.sizes());
    same_device(dist, bounds);
    if (bounds.size(0) > INT32_MAX) value_error("more than 2^31 - 1 boundaries");
    at::NoGradGuard none;
    const Tensor d = dense(dist), b = dense(bounds);
    Tensor out = make({d.size(0)}, d, at::kInt);
    On on(d);
    done(feq_distance_buckets(ptr_as<float>(d), d.size(0), ptr_as<float>(b), static_cast<int32_t>(b.size(0)), ptr_as<int32_t>(out),
                              on.stream),
         "feq_distance_buckets");
    return out;
}

// The edges of a graph: indices by destination and source, and their CSRs.
struct EdgeIndex {
    Tensor src, dst, perm, offsets, perm_s, offsets_s;
    int64_t nodes = 0;
};

struct EdgeAttentionCall {
    bool node_form, cm;
    int64_t nodes, heads;
    double decay, p;

    // The ABI's view of a call on these (contiguous) tensors.
    feq_edge_attn on(const Tensor& qt, const Tensor& kt, const Tensor& ls, const Tensor& b, const Tensor& d, const Tensor& bk,
                       const Tensor& sd, const EdgeIndex& g) const {
        feq_edge_attn a{};
        a.num_nodes = nodes;
        a.heads = static_cast<int32_t>(heads);
        a.dtype = code_of(qt, "q");
        const int64_t size = qt.element_size();
        char* base = static_cast<char*>(ptr(qt));
        a.q = base;
        if (node_form) {
            const int64_t mult = qt.size(cm ? 2 : 1) / 2, dim = qt.size(cm ? 0 : 2), n = qt.size(cm ? 1 : 0);
            a.num_edges = g.src.size(0);
            a.num_k = n;
            a.head_len = static_cast<int32_t>(cm ? mult / heads : mult / heads * dim);
            a.head_runs = static_cast<int32_t>(cm ? dim : 1);
            a.ldq = a.ldk = cm ? 2 * mult : 2 * mult * dim;
            a.head_stride = a.head_len;
            a.run_stride = cm ? n * 2 * mult : 0;
            a.k = base ? base + size * (cm ? mult : mult * dim) : nullptr;
            a.q_idx = ptr_as<int64_t>(g.dst);
            a.k_idx = ptr_as<int64_t>(g.src);
        } else {
            a.num_edges = qt.size(0);
            a.head_len = static_cast<int32_t>(qt.size(2));
            a.head_runs = 1;
            a.ldq = a.ldk = heads * qt.size(2);
            a.head_stride = a.head_len;
            a.k = ptr(kt);
        }
        a.perm = ptr_as<int32_t>(g.perm);
        a.offsets = ptr_as<int32_t>(g.offsets);
        a.log_scale = ptr(ls);
        a.scale_dtype = code_of(ls, "log_scale");
        a.decay = static_cast<float>(decay);
        a.dist = ptr_as<float>(d);
        if (b.defined()) {
            a.bias = ptr(b);
            a.bias_dtype = code_of(b, "bias");
            a.num_buckets = static_cast<int32_t>(b.size(0));
            a.buckets = ptr(bk);
            a.wide_buckets = bk.scalar_type() == at::kLong;
        }
        a.dropout = p;
        a.seed = ptr_as<int64_t>(sd);
        return a;
    }
};

struct EdgeAttentionNode final : TuneNode {
    // inputs: qk (node form) or q, then k (edge form), log_scale, bias, distances
    Kept q, k, log_scale, bias, dist, buckets, seed, weights;
    Kept src, dst, perm, offsets, perm_s, offsets_s;
    EdgeAttentionCall call{};
    bool own_weights = false;
    at::ScalarType dist_type = at::kFloat;

    variable_list backward(variable_list& grads) override {
        variable_list out(5);
        if (!grads[0].defined()) return out;
        const Tensor qt = q.get_dense(), kt = k.get_dense(), ls = log_scale.get_dense(), b = bias.get_dense(), d = dist.get_dense(),
                     bk = buckets.get_dense(), sd = seed.get();
        const Tensor w = own_weights ? weights.get_dense() : weights.get_dense(shared_from_this());
        const EdgeIndex ix{src.get_dense(), dst.get_dense(), perm.get_dense(), offsets.get_dense(), perm_s.get_dense(), offsets_s.get_dense(), call.nodes};
        const Tensor g = dense(grads[0]);
        const feq_edge_attn a = call.on(qt, kt, ls, b, d, bk, sd, ix);
        const bool rows = need(0) || need(1) || need(2);
        Tensor gq, gk, gls, gb, gd;
        if (rows) gq = make(qt.sizes(), qt, qt.scalar_type());
        if (rows && !call.node_form) gk = make(kt.sizes(), kt, kt.scalar_type());
        if (need(2)) gls = make(ls.sizes(), ls, ls.scalar_type());
        if (need(3)) gb = make(b.sizes(), b, b.scalar_type());
        if (need(4)) gd = make(d.sizes(), d, at::kFloat);
        if (a.num_edges == 0) {
            for (Tensor* t : {&gq, &gk, &gls, &gb, &gd})
                if (t->defined()) t->zero_();
        } else {
            const Tensor gz = make(w.sizes(), w, at::kFloat);
            const Tensor ws = scratch(feq_edge_attn_bwd_workspace(&a, gb.defined(), gls.defined()), qt);
            const char* kbase = static_cast<const char*>(static_cast<const void*>(a.k));
            char* gkp = !rows ? nullptr
                        : call.node_form ? static_cast<char*>(ptr(gq)) + (kbase - static_cast<const char*>(a.q))
                                    : static_cast<char*>(ptr(gk));
            On on(qt);
            done(feq_edge_attn_bwd(&a, ptr_as<int32_t>(ix.perm_s), ptr_as<int32_t>(ix.offsets_s), ptr_as<float>(w), ptr(g),
                                   ptr_as<float>(gz), ptr(gq), a.ldq, gkp, a.ldk, ptr(gb), ptr(gls), ptr_as<float>(gd), ptr(ws),
                                   bytes_of(ws), on.stream),
                 "feq_edge_attn_bwd");
        }
        if (need(0)) out[0] = gq;
        if (need(1)) out[1] = gk;
        out[2] = gls;
        out[3] = gb;
        if (need(4)) out[4] = gd.to(dist_type);
        return out;
    }
    void release() override {
        for (Kept* t : {&q, &k, &log_scale, &bias, &dist, &buckets, &seed, &weights, &src, &dst, &perm, &offsets, &perm_s, &offsets_s})
            t->reset_data();
    }
    std::string name() const override { return "FeqEdgeAttentionBackward"; }
};

// q: (nodes, 2 mult, dim), component-major (dim, nodes, 2 mult), or with k the edges' (edges, heads, head dim).
Tensor edge_attention(const Tensor& q, const OptTensor& k_, const OptTensor& src_, const OptTensor& dst_, const Tensor& perm,
                      const Tensor& offsets, const OptTensor& perm_s_, const OptTensor& offsets_s_, int64_t nodes, int64_t edges,
                      int64_t heads, const Tensor& log_scale, bool cm, const OptTensor& dist_, double decay, const OptTensor& bias_,
                      const OptTensor& buckets_, double p, const OptTensor& seed_) {
    const Tensor &k = get(k_), &dist = get(dist_), &b = get(bias_), &buckets = get(buckets_), &seed = get(seed_);
    const bool node_form = !k.defined();
    code_of(q, node_form ? "qk" : "Q");
    if (heads < 1 || heads > 1024) value_error("num_heads must be 1 to 1024, got ", heads);
    if (node_form) {
        if (q.dim() != 3 || q.size(cm ? 2 : 1) % 2 || q.size(cm ? 2 : 1) / 2 % heads || q.size(cm ? 2 : 1) == 0 || q.size(cm ? 0 : 2) < 1)
            value_error("qk must be ", cm ? "(dim, nodes, 2 mult)" : "(nodes, 2 mult, dim)", " with ", heads,
                        " heads dividing mult, got shape ", q.sizes());
        if (cm && q.size(0) > FEQ_MAX_SLOTS) value_error("at most ", FEQ_MAX_SLOTS, " components, got ", q.size(0));
        if (q.size(cm ? 1 : 0) != nodes) value_error("qk has ", q.size(cm ? 1 : 0), " rows but the graph has ", nodes, " nodes");
    } else {
        code_of(k, "K");
        if (q.scalar_type() != k.scalar_type())
            type_error("Q and K of different dtypes: ", dtype_name(q.scalar_type()), " and ", dtype_name(k.scalar_type()));
        if (q.dim() != 3 || q.size(0) != edges || q.size(1) != heads || q.size(2) < 1 || q.sizes() != k.sizes())
            value_error("Q and K must be (", edges, ", ", heads, ", head dim), got shapes ", q.sizes(), " and ", k.sizes());
        same_device(q, k);
    }
    const int64_t head = node_form ? q.numel() / std::max<int64_t>(nodes, 1) / 2 / heads : q.size(2);
    if (head > 1 << 20) value_error("heads of more than 2^20 elements");
    code_of(log_scale, "log_scale");
    if (log_scale.numel() != 1) value_error("log_scale must be one number, got shape ", log_scale.sizes());
    same_device(q, log_scale);
    same_device(q, perm);
    if (!(decay >= 0.0)) value_error("distance decay must not be negative, got ", decay);
    if (decay > 0.0) {
        if (static_cast<float>(decay) == 0.0f) value_error("a distance decay of ", decay, " is 0 in float32");
        if (!dist.defined()) value_error("distance decay needs distances");
        code_of(dist, "distances");
        if (dist.dim() != 1 || dist.size(0) != edges) value_error("distances must be (", edges, ",), got shape ", dist.sizes());
        same_device(q, dist);
    }
    if (b.defined() != buckets.defined()) value_error("bias and buckets come together");
    if (b.defined()) {
        code_of(b, "bias");
        if (b.dim() != 2 || b.size(1) != heads || b.size(0) < 1 || b.size(0) > 4096)
            value_error("bias must be (1 to 4096 buckets, ", heads, "), got shape ", b.sizes());
        same_device(q, b);
        need_gpu(buckets, "buckets");
        if (buckets.scalar_type() != at::kInt && buckets.scalar_type() != at::kLong)
            type_error("buckets must be int32 or int64, got ", dtype_name(buckets.scalar_type()));
        if (buckets.dim() != 1 || buckets.size(0) != edges) value_error("buckets must be (", edges, ",), got shape ", buckets.sizes());
        same_device(q, buckets);
    }
    check_share(p);
    if (p > 0.0) {
        if (!seed.defined()) value_error("dropout needs a seed (dropout_seed)");
        check_seed(seed, q);
    }
    const Tensor used_dist = decay > 0.0 ? dist : Tensor();
    const auto node = node_for<EdgeAttentionNode>(q, k, log_scale, b, used_dist);
    Tensor out;
    {
        at::NoGradGuard none;
        EdgeIndex ix{dense_long(get(src_)), dense_long(get(dst_)), dense(perm), dense(offsets), get(perm_s_), get(offsets_s_), nodes};
        if (ix.perm.size(0) != edges || ix.offsets.size(0) != nodes + 1 ||
            (node_form && (ix.src.size(0) != edges || ix.dst.size(0) != edges || ix.perm_s.size(0) != edges || ix.offsets_s.size(0) != nodes + 1)))
            value_error("the graph's CSRs do not cover ", edges, " edges and ", nodes, " nodes");
        const EdgeAttentionCall call{node_form, cm, nodes, heads, decay, p};
        const Tensor qc = dense(q), kc = k.defined() ? dense(k) : k, ls = dense(log_scale), bc = b.defined() ? dense(b) : b,
                     bk = b.defined() ? dense(buckets) : Tensor(),
                     dc = used_dist.defined() ? dense(used_dist.scalar_type() == at::kFloat ? used_dist : used_dist.to(at::kFloat)) : used_dist;
        const Tensor sd = p > 0.0 ? seed : Tensor();
        out = make({edges, heads}, q, q.scalar_type());
        const bool same = q.scalar_type() == at::kFloat && p == 0.0;
        const Tensor w = same ? out : make({edges, heads}, q, at::kFloat);
        if (edges) {
            const feq_edge_attn a = call.on(qc, kc, ls, bc, dc, bk, sd, ix);
            On on(q);
            done(feq_edge_attn_fwd(&a, ptr_as<float>(w), same ? nullptr : ptr(out), on.stream), "feq_edge_attn_fwd");
        }
        if (node) {
            node->call = call;
            node->own_weights = !same;
            if (used_dist.defined()) node->dist_type = used_dist.scalar_type();
            node->q.keep(qc);
            node->k.keep(kc);
            node->log_scale.keep(ls);
            node->bias.keep(bc);
            node->dist.keep(dc);
            node->buckets.keep(bk);
            node->seed.keep(sd);
            node->src.keep(ix.src);
            node->dst.keep(ix.dst);
            node->perm.keep(ix.perm);
            node->offsets.keep(ix.offsets);
            node->perm_s.keep(ix.perm_s);
            node->offsets_s.keep(ix.offsets_s);
            if (!same) node->weights.keep(w);
        }
    }
    if (node) {
        torch::autograd::set_history(out, node);
        if (!node->own_weights) node->weights.keep(out, true);
    }
    return out;
}

// ---- adapters beside a shared map ----------------------------------------------------

struct AdapterLinearNode final : TuneNode {
    Kept x, weight, down, up, low;
    Tensor order, offsets;
    Irreps irreps{{0}};
    int64_t nbias = 0;
    float scale = 1.0f;

    variable_list backward(variable_list& grads) override {
        variable_list out(5);
        if (!grads[0].defined()) return out;
        const Tensor xs = x.get_dense(), w = weight.get_dense(), dn = down.get_dense(), u = up.get_dense(), lo = low.get_dense(),
                     g = dense(grads[0]);
        check_plan(order, "order", 1);
        check_plan(offsets, "offsets", 1);
        const int64_t adapters = dn.size(0), rank = dn.size(2), ci = dn.size(3), co = u.size(2), rows = xs.size(-2);
        const int32_t *lv = irreps.lvals.data(), n = irreps.n();
        const bool shared = need(1) || need(4);
        const int32_t nb = need(4) ? static_cast<int32_t>(nbias) : 0;
        Tensor gx, gw, gd, gu, gb;
        if (need(0) || need(2) || need(3)) gx = make(xs.sizes(), xs, xs.scalar_type());
        if (shared) gw = make(w.sizes(), w, w.scalar_type());
        if (need(2)) gd = make(dn.sizes(), dn, dn.scalar_type());
        if (need(3)) gu = make(u.sizes(), u, u.scalar_type());
        if (nb) gb = make({co, nbias}, w, w.scalar_type());
        if (rows == 0) {
            for (Tensor* t : {&gx, &gw, &gd, &gu, &gb})
                if (t->defined()) t->zero_();
        } else {
            const Tensor ws = scratch(feq_adapter_linear_bwd_workspace(lv, n, adapters, rows, ci, co, rank, code_of(xs, "x"), shared, nb), xs);
            On on(xs);
            done(feq_adapter_linear_bwd(lv, n, adapters, rows, ci, co, rank, code_of(xs, "x"), ptr(g), ptr(xs), ptr(w), ptr(dn), ptr(u),
                                        scale, ptr_as<int32_t>(order), ptr_as<int32_t>(offsets), ptr_as<float>(lo), nb,
                                        irreps.cols.data(), ptr(gx), ptr(gd), ptr(gu), ptr(gw), ptr(gb), ptr(ws), bytes_of(ws), on.stream),
                 "feq_adapter_linear_bwd");
        }
        if (need(0)) out[0] = gx;
        if (need(1)) out[1] = gw;
        out[2] = gd;
        out[3] = gu;
        out[4] = gb;
        return out;
    }
    void release() override {
        for (Kept* t : {&x, &weight, &down, &up, &low}) t->reset_data();
        order.reset();
        offsets.reset();
    }
    std::string name() const override { return "FeqAdapterLinearBackward"; }
};

Tensor adapter_linear(const Tensor& x, const Tensor& weight, const Tensor& down, const Tensor& up, const OptTensor& bias, const Tensor& order,
                      const Tensor& offsets, int64_t rows, int64_t top_k, const std::vector<int64_t>& lvals, double scale) {
    const Irreps irreps(lvals);
    const int code = code_of(x, "x");
    const Tensor& b = get(bias);
    for (const auto& [t, name] : {std::pair<const Tensor&, const char*>{weight, "weight"}, {down, "down"}, {up, "up"}, {b, "bias"}}) {
        if (!t.defined()) continue;
        code_of(t, name);
        if (t.scalar_type() != x.scalar_type())
            type_error("x and ", name, " of different dtypes: ", dtype_name(x.scalar_type()), " and ", dtype_name(t.scalar_type()));
        same_device(x, t);
    }
    check_plan(order, "order", 1);
    check_plan(offsets, "offsets", 1);
    same_device(x, offsets);
    if (top_k != 1) value_error("a row has one adapter: a plan of ids (rows,) or (rows, 1), got top_k ", top_k);
    const int64_t adapters = offsets.size(0) - 1, n = irreps.n();
    if (down.dim() != 4 || down.size(0) != adapters || down.size(1) != n || down.size(2) < 1 || down.size(2) > 64 || down.size(3) < 1)
        value_error("down must be (", adapters, ", ", n, ", rank 1 to 64, cin), got shape ", down.sizes());
    const int64_t rank = down.size(2), ci = down.size(3);
    if (up.dim() != 4 || up.size(0) != adapters || up.size(1) != n || up.size(2) < 1 || up.size(3) != rank)
        value_error("up must be (", adapters, ", ", n, ", cout, ", rank, "), got shape ", up.sizes());
    const int64_t co = up.size(2);
    if (!(weight.dim() == 3 && weight.size(0) == n && weight.size(1) == co && weight.size(2) == ci) &&
        !(weight.dim() == 2 && weight.size(0) == n * co && weight.size(1) == ci))
        value_error("weight must be (", n, ", ", co, ", ", ci, ") or (", n * co, ", ", ci, "), got shape ", weight.sizes());
    const bool flat = x.dim() == 2 && n == 1 && irreps.dim == 1;
    if (!(flat && x.size(0) == rows && x.size(1) == ci) && !(x.dim() == 3 && x.size(0) == irreps.dim && x.size(1) == rows && x.size(2) == ci))
        value_error("x must be (", irreps.dim, ", ", rows, ", ", ci, "), got shape ", x.sizes());
    if (b.defined() && (irreps.nscalar == 0 || b.dim() != 2 || b.size(0) != co || b.size(1) != irreps.nscalar))
        value_error("bias must be (", co, ", ", irreps.nscalar, "), one column per scalar irrep, got shape ", b.sizes());
    if (!(scale - scale == 0.0)) value_error("scale must be finite, got ", scale);
    const auto node = node_for<AdapterLinearNode>(x, weight, down, up, b);
    Tensor y;
    {
        at::NoGradGuard none;
        const Tensor xc = dense(x), wc = dense(weight), dc = dense(down), uc = dense(up), bc = b.defined() ? dense(b) : b;
        c10::SmallVector<int64_t, 3> shape(x.sizes().begin(), x.sizes().end());
        shape.back() = co;
        y = make(shape, x, x.scalar_type());
        Tensor low;
        const size_t floats = feq_adapter_linear_low_floats(irreps.lvals.data(), irreps.n(), rows, ci, co, rank, node && wants_grad(up));
        if (floats) low = make({static_cast<int64_t>(floats)}, x, at::kFloat);
        On on(x);
        done(feq_adapter_linear_fwd(irreps.lvals.data(), irreps.n(), adapters, rows, ci, co, rank, code, ptr(xc), ptr(wc), ptr(dc), ptr(uc),
                                    static_cast<float>(scale), ptr_as<int32_t>(order), ptr_as<int32_t>(offsets), ptr(bc),
                                    static_cast<int32_t>(irreps.nscalar), irreps.cols.data(), ptr(y), ptr_as<float>(low), on.stream),
             "feq_adapter_linear_fwd");
        if (node) {
            node->x.keep(xc);
            node->weight.keep(wc);
            node->down.keep(dc);
            node->up.keep(uc);
            if (wants_grad(up)) node->low.keep(low);     // for its gradient alone
            node->order = order;
            node->offsets = offsets;
            node->irreps = irreps;
            node->nbias = irreps.nscalar;
            node->scale = static_cast<float>(scale);
        }
    }
    if (node) torch::autograd::set_history(y, node);
    return y;
}

}  // namespace

PYBIND11_MODULE(flasheq_torch, m) {
    m.doc() = "Layer norm, expert routing and fine-tuning operators of flash_eq on PyTorch tensors";
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const NotOnGpu& e) {
            const py::object type = py::module_::import("flash_eq._native").attr("CUDANotAvailableError");
            PyErr_SetString(type.ptr(), e.what());
        }
    });
    const auto released = py::call_guard<py::gil_scoped_release>();
    m.def("layer_norm", &layer_norm, released);
    m.def("expert_topk", &expert_topk, released);
    m.def("expert_plan", &expert_plan, released);
    m.def("plan_copy", &plan_copy, released);
    m.def("expert_dispatch", &expert_dispatch, released);
    m.def("expert_combine", &expert_combine, released);
    m.def("expert_linear", &expert_linear, released);
    m.def("feature_dropout", &feature_dropout, released);
    m.def("distance_buckets", &distance_buckets, released);
    m.def("edge_attention", &edge_attention, released);
    m.def("adapter_linear", &adapter_linear, released);
}
