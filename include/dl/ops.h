#pragma once
// Free functions on the decode path.  Mirrors include/dl/ops.h:100-101,149-158,191,341 of the reference
// (argmax, rotary_embedding, grouped_query_attention, linear, embedding, rms_norm); `sample` has no
// reference counterpart (the reference samples on the host, examples/text_generate.cpp:29-41), nor have `rotary_tables`,
// `rotary_positions`, `verify_drafted` and `expert_mixture`.
// All arithmetic runs on the GPU; bf16 storage computes and returns f32.

#include "dl/random.h"

namespace dl {

/// Index of the first maximum along `axis` (a NaN wins, first NaN first).  Result is i64.
DL_API Tensor argmax(const Tensor& input, Index axis, KeepDim keep = KeepDim::no);
/// Rotates interleaved pairs (2i, 2i+1) of the last axis by cosine/sine [L, D/2] (broadcast over leading
/// axes, L = input.size(-2)).
DL_API Tensor rotary_embedding(const Tensor& input, const Tensor& cosine, const Tensor& sine);
/// Which entries of a head's rotated part make a pair: neighbours (2i, 2i + 1), or those half the part apart (i, i + R/2).
enum class RotaryLayout { interleaved, half };
/// How rotary_tables changes the angles p * base^(-2i/R) for positions beyond the `trained` ones: `linear` divides every
/// angle by `factor`; `base` raises the base to base * factor^(R / (R - 2)), which leaves the fastest pair alone and
/// slows the slowest by `factor`; `parts` divides by `factor` the angles of pairs that turn at most `slow_turns` times
/// over the trained positions, leaves those that turn `fast_turns` times and more, and blends linearly in between.
/// Every entry is multiplied by `magnitude`.
struct RotaryScaling {
    enum class Kind { none, linear, base, parts } kind = Kind::none;
    double factor = 1.0;
    Index trained = 0;
    double slow_turns = 1.0, fast_turns = 32.0;
    double magnitude = 1.0;
};
/// Cosine and sine tables [capacity, dimensions / 2], f32, the angles taken in 64 bits (RotaryEmbedding's own tables
/// keep the reference's f32 angles).  `device` is where they will be used: operators copy tables from elsewhere in each call.
DL_API std::pair<Tensor, Tensor> rotary_tables(Index dimensions, Index capacity, double base = 10000.0,
                                               const RotaryScaling& scaling = {}, Device device = Device::cpu());
/// Rotates the first R = 2 * cosine.size(1) entries of each head of input [T, H, D] (f32 or bf16) by row positions[t]
/// of the tables [capacity, R/2], and copies the others; f32 [T, H, D].  Where positions[t] lies outside the tables the
/// rotated entries come out NaN.
DL_API Tensor rotary_positions(const Tensor& input, const Tensor& positions, const Tensor& cosine, const Tensor& sine,
                               RotaryLayout layout = RotaryLayout::interleaved);
/// Q [B,H,L,D], K [B,KV,S,D], V [B,KV,S,D]; query head h reads KV head h / (H/KV).  With no mask every query
/// row sees all S keys, as in the reference (src/ops/attention.cpp:161-164: no causal window); the decoder's
/// causal rule is applied by its own layers.  An explicit keep mask (reference include/dl/ops.h:149-153,
/// src/ops/attention.cpp:48-50,156-183) is a bool tensor broadcast to [B,H,L,S] by the trailing-axis rule: a
/// false entry drops that key from that row's softmax (its score becomes -inf), and a row that keeps no key
/// comes out NaN, as the reference's softmax of an all -inf row does.  Masked calls take the general kernels.
DL_API Tensor grouped_query_attention(const Tensor& query, const Tensor& key, const Tensor& value,
                                      std::optional<Tensor> keep_mask = std::nullopt);
/// input [..., in] times weight [out, in]^T (+ bias [out]).
DL_API Tensor linear(const Tensor& input, const Tensor& weight, std::optional<Tensor> bias = std::nullopt);
/// Row gather of weight [V, D] by i64 indices of any shape; the weight dtype is preserved.
DL_API Tensor embedding(const Tensor& indices, const Tensor& weight);
/// x / sqrt(mean(x*x) + epsilon) * weight over the trailing `normalized_shape`.
DL_API Tensor rms_norm(const Tensor& input, const Shape& normalized_shape,
                       std::optional<Tensor> weight = std::nullopt, std::optional<double> epsilon = std::nullopt);
/// Draws one index per row of logits [B, V]: temperature <= 0 is argmax; otherwise Gumbel-max,
/// argmax_i(logit_i / T + g_i) with g = -log(-log u), u from Philox(key, b*V + i) on (0, 1).
DL_API Tensor sample(const Tensor& logits, double temperature, RandomKey key);
/// Verifies drafted [B, K] (i64; a negative id ends a row) against the target's logits [B, K + 1, V], given uniforms
/// [B, K + 1] (f32, from [0, 1)).  With p and q the softmax of the target's and the draft's logits over the temperature, draft
/// x = drafted[b, i] is accepted while uniforms[b, i] * q_i(x) < p_i(x).  The next token is drawn with uniforms[b, K]: behind
/// the last draft from p, at the first refused one from max(p - q, 0) (from p where that is zero), as the first index whose
/// cumulative weight exceeds uniforms[b, K] times the total.  Without draft logits [B, K, V] a draft was certain: q(x) = 1.  A
/// temperature <= 0 accepts the target's argmax and nothing else.  A draft beyond the vocabulary is not accepted; a row whose
/// weights have no positive finite sum (NaN logits) takes its argmax.  Probabilities are of 64 bits, off by 2e-12 of their value;
/// a weight below e^-700 of the row's largest is zero.  The temperature is any finite number, K at most 2^20.  Returns tokens
/// [B, K + 1] (the accepted drafts, the drawn token, then -1) and the number accepted [B], both i64.
DL_API std::pair<Tensor, Tensor> verify_drafted(const Tensor& drafted, const Tensor& target,
                                                const std::optional<Tensor>& draft, double temperature,
                                                const Tensor& uniforms);

/// A feed-forward layer of E SwiGLU experts, of which each row x of input [..., d] (f32 or bf16) takes the `top` best: with
/// z = router x (router [E, d]) and p = softmax(z), those with the largest z, the lowest index first among equals (a NaN wins, the
/// first NaN first); their weights w are their p, divided by their sum where `normalise` is set; and
///   y = sum_j w_j down[e_j] (silu(gate[e_j] x) * (up[e_j] x)),   gate and up [E, F, d], down [E, d, F].
/// All matrices are f32 or bf16, the experts' of one type.  z and p are taken in 64 bits, so that rows choose as the exact
/// numbers do; the experts' products keep all bits of an f32.  An output that a number which is not finite takes part in is not finite
/// either, and no other row's (a logit of -inf takes part with p = 0, unless all of a row's are).  E is at most 1024, `top` at most 64, and E times the larger of d and F at most 2^25.
struct Mixture {
    Tensor output;  ///< f32 [..., d]
    Tensor chosen;  ///< i64 [..., top], the largest z first
    Tensor weights; ///< f32 [..., top]
};
DL_API Mixture expert_mixture(const Tensor& input, const Tensor& router, const Tensor& gate, const Tensor& up,
                              const Tensor& down, Index top, bool normalise = true);

} // namespace dl
