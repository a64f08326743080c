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

// Bounded waits, as the attention kernels have them: on expiry the wait records
// its site, raises the block's abort flag and returns false, and so does every
// later wait of the block.
enum ServingSite : int {
    kPagedKFull = 1,
    kPagedVFull,
    kPagedEmpty,
    kPagedQFull,
    kPagedSFull,
    kPagedSFree,
    kPagedPFull,
    kPagedOFull,
    kPagedOFree,
    kPagedDrain,
};

__device__ __forceinline__ void record_serving_timeout(int site)
{
    if (atomicCAS(&g_serving_error[0], 0, 4 /*FP4ATTN_ETIMEOUT*/) == 0) {
        g_serving_error[1] = site;
        g_serving_error[2] = blockIdx.x;
    }
}

struct ServingWait {
    volatile int* abort_flag;
    unsigned long long timeout_ns;
};

// The part of a wait that runs when the phase is not complete at first sight,
// out of line: a role's loop has several waits, and the roles of a block share
// the SM's small instruction cache.
static __device__ __noinline__ bool bounded_wait_on(uint64_t* bar, uint32_t parity, volatile int* abort_flag,
                                                    unsigned long long timeout_ns, int site)
{
    const uint64_t t0 = ptx::globaltimer_ns();
    for (uint32_t it = 1; it < (1u << 30); ++it) {
        if (ptx::mbar_try_wait(bar, parity)) return true;
        if ((it & 31u) == 0u) {
            if (*abort_flag) return false;
            if (ptx::globaltimer_ns() - t0 > timeout_ns) break;
        }
    }
    *abort_flag = 1;
    record_serving_timeout(site);
    return false;
}

__device__ __forceinline__ bool bounded_wait(uint64_t* bar, uint32_t parity, const ServingWait& w, int site)
{
    return ptx::mbar_try_wait(bar, parity) || bounded_wait_on(bar, parity, w.abort_flag, w.timeout_ns, site);
}

// On the way out: waits for what is in flight whatever the abort flag says.
static __device__ __noinline__ void bounded_drain(uint64_t* bar, uint32_t parity, unsigned long long ns)
{
    const uint64_t t0 = ptx::globaltimer_ns();
    for (uint32_t it = 0; it < (1u << 30); ++it) {
        if (ptx::mbar_try_wait(bar, parity)) return;
        if ((it & 31u) == 0u && ptx::globaltimer_ns() - t0 > ns) {
            record_serving_timeout(kPagedDrain);
            return;
        }
    }
}

}  // namespace fp4attn
