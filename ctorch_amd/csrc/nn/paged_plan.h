#pragma once
// What a PagedBatch keeps: the arrays that the kernels of a step read, made and checked on the host.

#include "nn/ops_internal.h"

#include "dl/paged.h"

namespace dl::nn {

struct PagedBatch::Plan {
    // the layout it was made for
    Index heads, kv_heads, head_dim, page_size, pages;
    DType dtype;
    Device device;

    Index tokens = 0, last = -1; // new positions, and the largest of them
    int row_tiles = 1, shared_row_tiles = 1, shared_splits = 0;
    Index slots = 0, shared_slots = 0; // of partials
    Index item_count = 0, shared_count = 0, merge_count = 0;
    Tensor blob; // the arrays below, on the device
    std::size_t tables = 0, items = 0, shared_items = 0, merges = 0, positions = 0, places = 0; // byte offsets
    template <class T> const T* at(std::size_t offset) const {
        return reinterpret_cast<const T*>(blob.data<char>() + offset);
    }
};

} // namespace dl::nn
