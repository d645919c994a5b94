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
    Index items = 0; // requests with new tokens
    Tensor blob;     // dlk_delta_item [items], on the device
};

} // namespace dl::nn
