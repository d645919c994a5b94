#pragma once
// The gated delta rule: a token mixer whose memory of a request is a matrix of fixed size per head instead of a cache that
// grows (no counterpart in the reference).  Requests keep their states in slots of a DeltaStates; a step's batch says how many
// new tokens of which requests it computes, from which slots and to which.

#include "dl/ops.h"

#include <memory>
#include <optional>
#include <span>
#include <vector>

namespace dl::nn {

/// States [slots, heads, key_dim, value_dim] of each layer, f32, on a GPU, zero at first.  key_dim 32, 64 or 128, value_dim a
/// multiple of 32 up to 256.
class DL_API DeltaStates {
public:
    DeltaStates(Index layers, Index slots, Index heads, Index key_dim, Index value_dim, Device device);
    Index layers() const { return static_cast<Index>(state_.size()); }
    Index slots() const { return slots_; }
    Index heads() const { return heads_; }
    Index key_dim() const { return key_dim_; }
    Index value_dim() const { return value_dim_; }
    Device device() const { return device_; }
    /// The live storage of a layer.
    const Tensor& state(Index layer) const { return state_.at(static_cast<std::size_t>(layer)); }

private:
    Index slots_, heads_, key_dim_, value_dim_;
    Device device_;
    std::vector<Tensor> state_;
};

/// What one step computes: request b goes on from the state in slot sources[b] (-1: from zero) by counts[b] new tokens (0: none
/// this time, its slots are not looked at) and leaves its new state in slot targets[b], which may be the same.  With another
/// one the old state is kept: to take refused drafts back, or for a fork.  A slot is the target of one request alone, and
/// then the source of no other.  The new tokens' rows lie one request after another.  Queries and keys have key_heads heads,
/// each of which serves states.heads() / key_heads heads of values.  Made once and used for every layer; the states may
/// be others of the same layout.  Making it copies the plan to the device and waits for the library's stream.
class DL_API DeltaBatch {
public:
    struct Plan;
    DeltaBatch(const DeltaStates& states, Index key_heads, std::span<const Index> sources, std::span<const Index> targets,
               std::span<const Index> counts);
    Index tokens() const;
    const Plan& plan() const { return *plan_; }

private:
    std::shared_ptr<const Plan> plan_;
};

} // namespace dl::nn

namespace dl {

/// For each new token, in order, and each head, with S the head's state [key_dim, value_dim]:
///   S = e^decay S;   S = S + k (rate (v - S^T k))^T;   out = scale S^T q
/// query and key [tokens, key_heads, key_dim] and value [tokens, heads, value_dim] are f32 or bf16 and may be views of one
/// projection output; decay and rate [tokens, heads], f32 or bf16.  A decay of -inf forgets everything before the token.  The
/// default scale is 1 / sqrt(key_dim), and one beyond f32 is refused.  f32 [tokens, heads, value_dim].  The arithmetic is of
/// f32: keys of length 1, rates up to 2 and decays up to 0 keep a state bounded; others let it grow as the rule does (decays of 64
/// tokens in a row that add up to more than 88 may overflow although the state would not).  A number that is not finite makes its
/// token's output and what follows it in its request not finite: of its column from a value or a state, of its heads from a key
/// or a gate, and from a query its own row of its heads alone.  A later decay of -inf does not take that back, and nothing before
/// the token knows of it.
DL_API Tensor gated_delta(const nn::DeltaStates& states, Index layer, const nn::DeltaBatch& batch, const Tensor& query,
                          const Tensor& key, const Tensor& value, const Tensor& decay, const Tensor& rate,
                          std::optional<double> scale = std::nullopt);

/// Copies the states in slots sources[i] to slots targets[i] in every layer, each source as it was before the call; no slot
/// is a target twice.
DL_API void delta_copy(const nn::DeltaStates& states, std::span<const Index> sources, std::span<const Index> targets);

} // namespace dl
