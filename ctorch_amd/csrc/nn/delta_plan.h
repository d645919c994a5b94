#pragma once
// What a DeltaBatch keeps: the arrays that the kernels of a step read, made and checked on the host.

#include "nn/ops_internal.h"

#include "dl/delta.h"

namespace dl::nn {

struct DeltaBatch::Plan {
    // the layout it was made for
    Index heads, key_heads, key_dim, value_dim, slots;
    Device device;

    Index tokens = 0;
    // what a launch goes through: the requests with few new tokens, and, in rounds of so many chunks as a workspace holds, the
    // others' (a request that goes on in the next round does so from its target)
    struct Round {
        Index first = 0, items = 0, first_chunk = 0, chunks = 0;
    };
    Index few = 0; // items of few tokens, the first ones
    std::vector<Round> rounds;
    Tensor blob; // dlk_delta_item [..], then dlk_delta_chunk [..], on the device
    std::size_t chunks = 0; // where they begin
};

} // namespace dl::nn
