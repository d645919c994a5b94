// A layer of experts (include/dl/ops.h, include/dl/decoder.h).
#include "nn/ops_internal.h"

#include <algorithm>
#include <stdexcept>

namespace dl {

using namespace detail;

Mixture expert_mixture(const Tensor& input, const Tensor& router, const Tensor& gate, const Tensor& up, const Tensor& down,
                       Index top, bool normalise) {
    constexpr const char* name = "expert_mixture";
    GpuContext& context = gpu_of(input, name);
    const auto refuse = [](const std::string& what) { throw std::invalid_argument("expert_mixture: " + what); };
    if (input.ndim() < 1 || router.ndim() != 2 || gate.ndim() != 3 || down.ndim() != 3)
        refuse("expects input [..., d], router [E, d], gate and up [E, F, d], down [E, d, F]");
    const Index dim = input.size(-1), experts = router.size(0), hidden = gate.size(1);
    if (router.size(1) != dim || gate.shape() != Shape{experts, hidden, dim} || up.shape() != gate.shape() ||
        down.shape() != Shape{experts, dim, hidden})
        refuse("expects input [..., d], router [E, d], gate and up [E, F, d], down [E, d, F]; got " + shape_string(input.shape()) + ", " +
               shape_string(router.shape()) + ", " + shape_string(gate.shape()) + ", " + shape_string(up.shape()) + ", " + shape_string(down.shape()));
    if (dim <= 0 || hidden <= 0 || experts <= 0) refuse("d, F and E must be positive");
    // (a launch has fewer than 2^32 threads)
    if (experts > DLK_EXPERTS_MOST || std::max(dim, hidden) > (1 << 25) / experts) refuse("too many experts or entries");
    if (top <= 0 || top > std::min<Index>(experts, DLK_EXPERTS_TOP_MOST)) refuse("top must be from 1 to the number of experts, and at most 64");
    if (input.dtype() != DType::f32 && input.dtype() != DType::bf16) refuse("input must be f32 or bf16");
    for (const Tensor* t : {&router, &gate, &up, &down})
        if (!(t->device() == input.device())) refuse("weights on another device");
    if (up.dtype() != gate.dtype() || down.dtype() != gate.dtype()) refuse("the experts' weights must be of one type");

    dlk_experts_params p{};
    p.router = weight_data(router, p.router_bf16, name);
    p.gate = weight_data(gate, p.weights_bf16, name);
    p.up = weight_data(up, p.weights_bf16, name);
    p.down = weight_data(down, p.weights_bf16, name);
    const Tensor x = input.contiguous();
    Shape few = input.shape();
    few.back() = top;
    p.tokens = x.numel() / dim;
    Mixture out{empty_tensor(input.shape(), DType::f32, input.device()), empty_tensor(few, DType::i64, input.device()),
                empty_tensor(few, DType::f32, input.device())};
    if (p.tokens == 0) return out;
    p.x_bf16 = x.dtype() == DType::bf16;
    p.dim = static_cast<int>(dim);
    p.hidden = static_cast<int>(hidden);
    p.experts = static_cast<int>(experts);
    p.top = static_cast<int>(top);
    p.normalise = normalise;
    // (many rows in parts, over one workspace, released to the pool in stream order)
    const Index rows = p.tokens, most = std::min<Index>(rows, dlk_experts_rows(&p));
    p.tokens = most;
    p.x = x.data<void>();
    const Tensor workspace = empty_tensor({dlk_experts_workspace(&p) / 4 + 1}, DType::f32, input.device());
    p.workspace = mutable_data(workspace);
    for (Index first = 0; first < rows; first += most) {
        p.tokens = std::min(most, rows - first);
        p.x = x.data<char>() + first * dim * static_cast<Index>(element_size(x.dtype()));
        p.y = static_cast<float*>(mutable_data(out.output)) + first * dim;
        p.chosen = static_cast<Index*>(mutable_data(out.chosen)) + first * top;
        p.weights = static_cast<float*>(mutable_data(out.weights)) + first * top;
        hip_check(dlk_experts(&p, context.stream), name);
    }
    return out;
}

namespace nn {

ExpertMixture::ExpertMixture(Index dimensions, Index hidden, Index experts, Index top, bool normalise, TensorOptions options)
    : top_(top), normalise_(normalise) {
    if (dimensions <= 0 || hidden <= 0 || experts <= 0) throw std::invalid_argument("ExpertMixture: sizes must be positive");
    if (experts > DLK_EXPERTS_MOST || top <= 0 || top > std::min<Index>(experts, DLK_EXPERTS_TOP_MOST))
        throw std::invalid_argument("ExpertMixture: at most 1024 experts, and top from 1 to their number, at most 64");
    router_ = register_parameter("router", linear_parameter({experts, dimensions}, dimensions, options));
    gate_ = register_parameter("gate", linear_parameter({experts, hidden, dimensions}, dimensions, options));
    up_ = register_parameter("up", linear_parameter({experts, hidden, dimensions}, dimensions, options));
    down_ = register_parameter("down", linear_parameter({experts, dimensions, hidden}, hidden, options));
}

Mixture ExpertMixture::mix(const Tensor& input) const { return expert_mixture(input, router_, gate_, up_, down_, top_, normalise_); }

} // namespace nn
} // namespace dl
