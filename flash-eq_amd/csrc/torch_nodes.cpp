// PyTorch bindings of the layer norm and the expert routing: argument checks, outputs and
// workspaces from the caching allocator, autograd nodes, and the calls of the C ABI
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
variable_list once(variable_list&& grads) {
    if (!at::GradMode::is_enabled()) return std::move(grads);
    for (auto& g : grads)
        if (g.defined()) g = g.detach().requires_grad_();
    auto error = std::make_shared<torch::autograd::DelayedError>(
        "the layer norm and the expert routing of flash_eq have no second derivative", static_cast<int64_t>(grads.size()));
    return (*error)(std::move(grads));
}

struct OnceNode : torch::autograd::Node {
    variable_list apply(variable_list&& grads) final {
        variable_list out;
        {
            std::lock_guard<std::mutex> lock(mutex_);      // a backward of the same graph in another thread frees
            at::NoGradGuard none;
            out = backward(grads);
        }
        return once(std::move(out));
    }
    void release_variables() final {
        std::lock_guard<std::mutex> lock(mutex_);
        release();
    }
    virtual variable_list backward(variable_list& grads) = 0;
    virtual void release() {}
    bool need(size_t i) const { return task_should_compute_output(i); }
};

// The node of a call whose inputs `in` some gradient may reach, else none.
template <class N, class... In>
std::shared_ptr<N> node_for(const In&... in) {
    TORCH_CHECK_NOT_IMPLEMENTED(!(torch::autograd::isFwGradDefined(in) || ...),
                                "the layer norm and the expert routing of flash_eq have no forward-mode derivative");
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

}  // namespace

PYBIND11_MODULE(flasheq_torch, m) {
    m.doc() = "Layer norm and expert routing of flash_eq on PyTorch tensors";
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
}
