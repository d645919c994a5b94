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
    struct List {
        Index rows = 16, count = 0; // the most rows of an item, and items
        std::size_t items = 0;      // where the items are
    } lists[2];                     // by DLK_PAGED_FEW, DLK_PAGED_MANY
    Index partials = 0;             // rows of partials
    Index shared_splits = 0, shared_stride = 0, merge_count = 0, merge_most = 0;
    Tensor blob; // the arrays below, on the device
    std::size_t tables = 0, merges = 0, positions = 0, places = 0; // byte offsets
    template <class T> const T* at(std::size_t offset) const {
        return reinterpret_cast<const T*>(blob.data<char>() + offset);
    }
};

} // namespace dl::nn
