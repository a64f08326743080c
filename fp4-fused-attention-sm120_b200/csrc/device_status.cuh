// device_status.cuh -- the device error word of the serving kernels (rotary
// positions, paged cache, paged attention) and their bounded barrier waits.
//
// word 0: 0, FP4ATTN_ETIMEOUT or FP4ATTN_EINDEX; word 1: the wait or the kind
// of index; words 2, 3: the block (x) or the index that was out of range.
// The first error stays until fp4attn_status_query reads and clears it.
#pragma once

#include <cstdint>

#include "ptx_sm100.cuh"

namespace fp4attn {

static __device__ int g_serving_error[4];

enum IndexKind : int {
    kIndexPosition = 1,  // a position outside the rotary table
    kIndexPage,          // a page number outside the cache
    kIndexSequence,      // a sequence number outside the block table
    kIndexLength,        // a position or length beyond the block table's pages, or a negative length
};

__device__ __forceinline__ void record_index_error(int kind, int64_t value)
{
    if (atomicCAS(&g_serving_error[0], 0, 6 /*FP4ATTN_EINDEX*/) == 0) {
        g_serving_error[1] = kind;
        g_serving_error[2] = static_cast<int>(value);
        g_serving_error[3] = static_cast<int>(value >> 32);
    }
}

}  // namespace fp4attn
