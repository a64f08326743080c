// paged_attention.cuh -- attention of one new token per sequence over the
// paged FP4 key / FP16 value cache (sm_100a).
//
//     z_j = scale * Qq . Kq_j,   o = sum_j exp(z_j) v_j / sum_j exp(z_j),
// j over the first seq_lens[b] tokens of sequence b, Qq the query quantised
// as the forward quantises it, Kq the cache's keys.  A sequence of length 0
// gives o = 0 and log-sum-exp +inf, as a row without visible keys does in the
// forward.
//
// Bound by reading the cache: a token of one head is D/2 + D/32 + 2 D bytes
// for 4 D group operations, so the tensor cores idle and everything else must
// stay off the path of the loads.  The products are formed the other way
// round than in the forward, with the keys as the MMA's M, because there are
// few query rows and a thread per key spreads the softmax over the warps:
//     S^T = K Q^T     kind::mxf4 block-scaled, M = 128 keys, N = NH heads: the
//                     codes go from the cache to the tensor core untouched;
//     O^T = V^T P^T   kind::f16, M = head_dim, N = NH heads, K = 128 keys: V is
//                     used in the layout in which it lies in the cache.
//
// Work: a tile is 128 keys of one sequence and one group of query heads.  All
// tiles, sequence after sequence and head after head, are dealt evenly to the
// blocks (one per SM), a contiguous range each, whatever the lengths; the
// blocks find their ranges from seq_lens, so nothing is planned on the host
// and a captured launch follows the lengths.  A block whose range holds a
// whole item (sequence, head group) writes its output; of an item that spans
// blocks each writes a partial result (unnormalised O, running maximum, sum),
// and paged_join_kernel joins them, in order, so results repeat bit for bit.
//
// Roles (256 threads):
//   warp 0     producer: a lane per page of the tile loads its codes, scales
//              (raw) and values with TMA into a ring of stages.
//   warp 1     MMA issuer (one thread): S^T of tile g + 1, then O^T of tile g.
//   warp 2     scales: raw scale bytes to the tensor core's scale layout.
//   warp 3     queries: quantises the next item's query heads.
//   warps 4-7  softmax: thread = key (row of S^T), then head-dim row of O^T.
//
// The softmax reference m starts as the item's first tile's maximum and is
// moved only when a score exceeds it by more than 2^8 (FP16 P would come near
// its range at 2^16); all threads hold the same m in registers and agree by
// one barrier with a vote.  P is rounded to FP16 for FP16 output (2^-11 of
// each weight, below the rounding of the result); for FP32 output it is split
// into two FP16 parts, which the same accumulation adds.  Each tile's O^T is
// added to FP32 registers with proper rounding: only 128 keys are summed
// inside the tensor core.
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>
#include <cstdint>

#include "paged.cuh"

namespace fp4attn {

// Blocks of the attention kernel at most (one per SM of a B200), a fixed
// number so that the workspace is a function of the shape alone.
constexpr int kPagedBlocks = 148;
constexpr int kPagedTile = 128;

template <int D, int NH, bool kSplitP>
struct PagedCfg {
    static constexpr int THREADS = 256;
    static constexpr int KROW = D <= 64 ? 32 : D <= 128 ? 64 : 128;  // bytes of a key's codes in shared memory (= swizzle)
    static constexpr int KSTEPS = (D + 63) / 64;                     // mxf4 MMAs of K = 64 per S^T tile
    static constexpr int ATOMS = (KSTEPS + 1) / 2;                   // 512-byte scale atoms (four blocks of 32)
    static constexpr int NB = D / 32;                                // scale bytes per key
    // V in chunks of CHE columns, CB-byte swizzled rows, per page [chunk][token].
    static constexpr int CHE = D % 64 == 0 ? 64 : 32;
    static constexpr int CB = 2 * CHE;
    static constexpr uint32_t VSW = CB == 128 ? ptx::kSwizzle128B : ptx::kSwizzle64B;
    static constexpr int DCH = D / CHE;
    static constexpr int MT = (D + 127) / 128;                       // O^T MMAs of M = 128 (rows past D are not read)
    static constexpr int PARTS = kSplitP ? 2 : 1;
    static constexpr int PROW = 2 * NH;                              // bytes of a key's P row (= swizzle)
    static constexpr uint32_t PSW = PROW == 32 ? ptx::kSwizzle32B : ptx::kSwizzle64B;
    // Tensor Memory columns
    static constexpr int S_COL = 0;                                  // two buffers
    static constexpr int O_COL = 2 * NH;                             // two buffers of MT
    static constexpr int SFA_COL = O_COL + 2 * MT * NH;
    static constexpr int SFB_COL = SFA_COL + 4 * ATOMS;
    static constexpr int TMEM_USED = SFB_COL + 4 * ATOMS;
    static constexpr int TMEM_COLS = TMEM_USED <= 128 ? 128 : 256;
    static_assert(TMEM_USED <= 256, "TMEM budget exceeded");
    // shared memory, offsets from a 1024-aligned base
    static constexpr int align1k(int x) { return (x + 1023) / 1024 * 1024; }
    static constexpr int K_BYTES = kPagedTile * KROW;
    static constexpr int V_BYTES = kPagedTile * D * 2;
    static constexpr int S_BYTES = align1k(kPagedTile * NB);
    static constexpr int STAGE = K_BYTES + V_BYTES + S_BYTES;
    static constexpr int OFF_P = 0;                                  // [2][PARTS][128 keys][PROW]
    static constexpr int P_BYTES = kPagedTile * PROW;
    static constexpr int OFF_Q = OFF_P + 2 * PARTS * P_BYTES;        // [2][NH rows][KROW]
    static constexpr int Q_BYTES = align1k(NH * KROW);
    static constexpr int OFF_QSF = OFF_Q + 2 * Q_BYTES;              // [2][ATOMS][512]
    static constexpr int OFF_KSF = OFF_QSF + 2 * ATOMS * 512;        // [2][ATOMS][512]
    static constexpr int OFF_STAGE = align1k(OFF_KSF + 2 * ATOMS * 512);
    // The O^T MMA reads 128 rows (head-dim columns) of V: past head_dim it
    // reads on into what follows; those rows of O^T are not used.
    static constexpr int V_OVER = (MT * 128 - D) / CHE * kPagedTile * CB;
    static constexpr int MISC = 2048;                                // barriers, reductions
    static constexpr int kBudget = 227 * 1024 - 1024 - OFF_STAGE - MISC - V_OVER;
    static constexpr int STAGES = kBudget / STAGE < 8 ? kBudget / STAGE : 8;
    static_assert(STAGES >= 2, "shared memory budget exceeded");
    static constexpr int OFF_MISC = OFF_STAGE + STAGES * STAGE + V_OVER;
    static constexpr int SMEM_BYTES = OFF_MISC + MISC + 1024;
};

// The partial results of an item that spans blocks: slot 2 * block for a range
// that began inside the item, 2 * block + 1 for the item begun in the range.
struct PagedPartials {
    float* o;        // [2 * kPagedBlocks][NH][D]
    float2* ml;      // [2 * kPagedBlocks][NH]  maximum (log2 domain), sum
    int4* items;     // [kPagedBlocks]  sequence, head group, last block; sequence -1: none begun here spans on
};

struct PagedArgs {
    const void* q;
    int q_half;           // Q is FP16 (else FP32)
    int64_t qb, qh;       // element strides of batch and head
    int batch, q_heads, group;
    int head_groups;      // kv_heads * groups of heads_per_group query heads
    int splits;           // groups per key/value head
    int heads_per_group;
    CacheView c;
    TableView t;
    const int32_t* seq_lens;
    float scale_log2;     // softmax scale * log2(e)
    int ocp;
    void* out;            // [batch][q_heads][head_dim]
    float* lse;           // [batch][q_heads] or null
    PagedPartials p;
    unsigned long long timeout_ns;
};

__device__ __forceinline__ int paged_length(const PagedArgs& a, int b)
{
    const int len = __ldg(a.seq_lens + b);
    const int64_t most = static_cast<int64_t>(a.t.max_pages) << a.c.page_shift;
    return len < 0 ? 0 : len > most ? static_cast<int>(most) : len;
}

// Tiles of a sequence; an empty one has one (without keys), which writes its zeros.
__device__ __forceinline__ int paged_tiles(int len) { return len <= 0 ? 1 : (len + kPagedTile - 1) / kPagedTile; }

// First tile of a block's range out of `total`.
__device__ __forceinline__ int paged_first(int64_t total, int block, int blocks)
{
    return static_cast<int>(total * block / blocks);
}

// The walk over a block's tiles; every role makes its own.
struct TileWalk {
    int b, hg, tile, tiles, len, left;
    bool first;  // the first tile of an item in this block's range
    __device__ __forceinline__ void begin(const PagedArgs& a, const int4& start, int n)
    {
        b = start.x;
        hg = start.y;
        tile = start.z;
        left = n;
        first = true;
        if (left > 0) {
            len = paged_length(a, b);
            tiles = paged_tiles(len);
        }
    }
    __device__ __forceinline__ int keys() const { return max(0, min(kPagedTile, len - tile * kPagedTile)); }
    __device__ __forceinline__ bool last() const { return tile + 1 == tiles || left == 1; }
    __device__ __forceinline__ void next(const PagedArgs& a)
    {
        left--;
        tile++;
        first = false;
        if (tile == tiles) {
            tile = 0;
            first = true;
            if (++hg == a.head_groups) {
                hg = 0;
                b++;
                if (left > 0) {
                    len = paged_length(a, b);
                    tiles = paged_tiles(len);
                }
            }
        }
    }
};

// A block's share of the work.
struct PagedRange {
    int4 start;        // sequence, head group and tile that it begins at
    int first, count;  // its tiles, in the order of all
    int total;         // tiles of the call
    int blocks;        // blocks that have any (the first ones)
};

// This block's range, by a scan of the lengths with all 256 threads.
__device__ __forceinline__ void find_range(const PagedArgs& a, PagedRange* range, int* scratch)
{
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
    int sum = 0;
    for (int b = tid; b < a.batch; b += 256) sum += paged_tiles(paged_length(a, b));
    for (int i = 16; i; i >>= 1) sum += __shfl_xor_sync(~0u, sum, i);
    if (lane == 0) scratch[warp] = sum;
    __syncthreads();
    int64_t total = 0;
    for (int i = 0; i < 8; i++) total += scratch[i];
    total *= a.head_groups;
    const int blocks = static_cast<int>(min(total, static_cast<int64_t>(gridDim.x)));
    const bool idle = static_cast<int>(blockIdx.x) >= blocks;
    const int t0 = idle ? 0 : paged_first(total, blockIdx.x, blocks), t1 = idle ? 0 : paged_first(total, blockIdx.x + 1, blocks);
    if (tid == 0) {
        range->first = t0;
        range->count = t1 - t0;
        range->total = static_cast<int>(total);
        range->blocks = blocks;
    }
    if (idle) return;
    int carry = 0;  // tiles (of one head group) of the sequences before this chunk
    for (int b0 = 0; b0 < a.batch; b0 += 256) {
        const int mine = b0 + tid < a.batch ? paged_tiles(paged_length(a, b0 + tid)) : 0;
        int inc = mine;
        for (int i = 1; i < 32; i <<= 1) {
            const int v = __shfl_up_sync(~0u, inc, i);
            if (lane >= i) inc += v;
        }
        __syncthreads();
        if (lane == 31) scratch[warp] = inc;
        __syncthreads();
        int before = carry, all = 0;
        for (int i = 0; i < 8; i++) {
            if (i < warp) before += scratch[i];
            all += scratch[i];
        }
        const int64_t at = static_cast<int64_t>(before + inc - mine) * a.head_groups;
        if (t1 > t0 && t0 >= at && t0 < at + static_cast<int64_t>(mine) * a.head_groups) {
            const int in = static_cast<int>(t0 - at);
            range->start = make_int4(b0 + tid, in / mine, in % mine, 0);
        }
        carry += all;
    }
}

template <typename OutT, int D, int NH>
__global__ void __launch_bounds__(256, 1)
    paged_attention_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                           const __grid_constant__ PagedArgs a)
{
    constexpr bool kSplitP = sizeof(OutT) == 4;
    using C = PagedCfg<D, NH, kSplitP>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_MISC);
    uint64_t* k_full = bars;               // [8] codes and scales of a stage landed
    uint64_t* v_full = k_full + 8;         // [8] values landed
    uint64_t* empty = v_full + 8;          // [8] the stage's MMAs are done (commit)
    uint64_t* sf_full = empty + 8;         // [2] scale atoms written (32)
    uint64_t* q_full = sf_full + 2;        // [2] query codes and scales written (32)
    uint64_t* q_empty = q_full + 2;        // [2] the item's S^T MMAs are done (commit)
    uint64_t* s_full = q_empty + 2;        // [2] S^T computed (commit)
    uint64_t* s_free = s_full + 2;         // [2] S^T in registers (128)
    uint64_t* p_full = s_free + 2;         // [2] P written (128)
    uint64_t* o_full = p_full + 2;         // [2] O^T computed, P read (commit)
    uint64_t* o_free = o_full + 2;         // [2] O^T in registers (128)
    uint64_t* drain = o_free + 2;          // everything issued is done (exit)
    float* red = reinterpret_cast<float*>(smem + C::OFF_MISC + 512);  // [4][NH]
    int* scratch = reinterpret_cast<int*>(smem + C::OFF_MISC + 1024 + 512);  // [8]
    PagedRange* range = reinterpret_cast<PagedRange*>(scratch + 8);
    uint32_t* tmem_sh = reinterpret_cast<uint32_t*>(scratch + 16);
    int* abort_sh = scratch + 17;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 8; i++) {
            ptx::mbar_init(&k_full[i], 1);
            ptx::mbar_init(&v_full[i], 1);
            ptx::mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            ptx::mbar_init(&sf_full[i], 32);
            ptx::mbar_init(&q_full[i], 32);
            ptx::mbar_init(&q_empty[i], 1);
            ptx::mbar_init(&s_full[i], 1);
            ptx::mbar_init(&s_free[i], 128);
            ptx::mbar_init(&p_full[i], 128);
            ptx::mbar_init(&o_full[i], 1);
            ptx::mbar_init(&o_free[i], 128);
        }
        ptx::mbar_init(drain, 1);
        *abort_sh = 0;
        ptx::fence_mbar_init();
        ptx::prefetch_tmap(&tm_k);
        ptx::prefetch_tmap(&tm_v);
    }
    if (warp == 1) {
        ptx::tmem_alloc(tmem_sh, C::TMEM_COLS);
        ptx::tmem_relinquish();
    }
    // Query rows past the group's heads and blocks past head_dim: codes 0,
    // scale 1, for both buffers.
    for (int i = threadIdx.x; i < 2 * C::Q_BYTES / 16; i += 256)
        reinterpret_cast<uint4*>(smem + C::OFF_Q)[i] = make_uint4(0u, 0u, 0u, 0u);
    for (int i = threadIdx.x; i < 2 * C::ATOMS * 32; i += 256)
        reinterpret_cast<uint4*>(smem + C::OFF_QSF)[i] = make_uint4(0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu);
    ptx::fence_proxy_async_smem();
    // Everything before this overlaps the grid before this one in the stream.
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    find_range(a, range, scratch);
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = *tmem_sh;
    const int count = range->count;
    const ServingWait w{abort_sh, a.timeout_ns};
    auto stage_of = [&](int g) { return smem + C::OFF_STAGE + (g % C::STAGES) * C::STAGE; };
    auto stage_parity = [&](int g) { return static_cast<uint32_t>(g / C::STAGES) & 1u; };
    auto two_parity = [](int g) { return static_cast<uint32_t>(g / 2) & 1u; };
    TileWalk t;
    t.begin(a, range->start, count);

    if (warp == 0) {
        // ------------------------------------------------------------ producer
        const int page = a.c.page_size;
        int g = 0;
        for (; t.left > 0; t.next(a), g++) {
            const int n = (t.keys() + page - 1) >> a.c.page_shift;  // pages of this tile, one per lane (at most 8)
            int id = 0;
            if (lane < n) {
                id = __ldg(a.t.pages + t.b * a.t.stride + ((t.tile * kPagedTile) >> a.c.page_shift) + lane);
                if (id < 0 || id >= a.c.pages) {
                    record_index_error(kIndexPage, id);
                    id = 0;
                }
            }
            if (lane == 0 && t.first && t.tile == 0 && t.hg == 0) {
                const int len = __ldg(a.seq_lens + t.b);
                if (len != t.len) record_index_error(kIndexLength, len);
            }
            const int s = g % C::STAGES;
            if (g >= C::STAGES && !__all_sync(~0u, bounded_wait(&empty[s], stage_parity(g - C::STAGES), w, kPagedEmpty))) break;
            if (lane == 0) {
                ptx::mbar_arrive_expect_tx(&k_full[s], n * page * (C::KROW + C::NB));
                ptx::mbar_arrive_expect_tx(&v_full[s], n * page * D * 2);
            }
            __syncwarp();
            if (lane < n) {
                uint8_t* st = stage_of(g);
                const int head = t.hg / a.splits;
                ptx::tma_load_4d(st + lane * page * C::KROW, &tm_k, &k_full[s], 0, head, id);
                ptx::bulk_load(st + C::K_BYTES + C::V_BYTES + lane * page * C::NB,
                               a.c.k_scales + id * a.c.k_scales_stride + static_cast<int64_t>(head) * page * C::NB,
                               page * C::NB, &k_full[s]);
                ptx::tma_load_5d(st + C::K_BYTES + lane * page * D * 2, &tm_v, &v_full[s], 0, 0, head, id);
            }
            __syncwarp();
        }
        // Every copy issued lands before the block exits.
        if (lane == 0)
            for (int i = max(0, g - C::STAGES); i < g; i++) {
                bounded_drain(&k_full[i % C::STAGES], stage_parity(i), 2 * a.timeout_ns);
                bounded_drain(&v_full[i % C::STAGES], stage_parity(i), 2 * a.timeout_ns);
            }
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer
        if (lane == 0) {
            constexpr uint32_t qk_sw = ptx::swizzle_mode_for_bytes(C::KROW);
            constexpr uint32_t idesc_o = ptx::idesc_f16x(128, NH, 0, true, true);
            int item = -1;
            auto issue_s = [&](const TileWalk& x, int g) {
                const int s = g % C::STAGES, buf = g & 1;
                if (x.first) {
                    item++;
                    if (!bounded_wait(&q_full[item & 1], two_parity(item), w, kPagedQFull)) return false;
                }
                if (!bounded_wait(&k_full[s], stage_parity(g), w, kPagedKFull)) return false;
                if (!bounded_wait(&sf_full[buf], two_parity(g), w, kPagedScales)) return false;
                if (g >= 2 && !bounded_wait(&s_free[buf], two_parity(g - 2), w, kPagedSFree)) return false;
                ptx::tc_fence_after();
                if (x.first)
#pragma unroll
                    for (int i = 0; i < C::ATOMS; i++)
                        ptx::tc_cp_32x128b_warpx4(tmem + C::SFB_COL + 4 * i,
                                                  ptx::make_sdesc(ptx::smem_u32(smem + C::OFF_QSF + ((item & 1) * C::ATOMS + i) * 512),
                                                                  0, 128, ptx::kSwizzleNone));
#pragma unroll
                for (int i = 0; i < C::ATOMS; i++)
                    ptx::tc_cp_32x128b_warpx4(tmem + C::SFA_COL + 4 * i,
                                              ptx::make_sdesc(ptx::smem_u32(smem + C::OFF_KSF + (buf * C::ATOMS + i) * 512), 0,
                                                              128, ptx::kSwizzleNone));
                const uint64_t kd = ptx::make_sdesc(ptx::smem_u32(stage_of(g)), 16, 8 * C::KROW, qk_sw);
                const uint64_t qd = ptx::make_sdesc(ptx::smem_u32(smem + C::OFF_Q + (item & 1) * C::Q_BYTES), 16, 8 * C::KROW, qk_sw);
#pragma unroll
                for (int kk = 0; kk < C::KSTEPS; kk++) {
                    const uint32_t id = 2u * (kk & 1);
                    ptx::mma_mxf4(tmem + C::S_COL + buf * NH, kd + 2 * kk, qd + 2 * kk, ptx::idesc_mxf4(128, NH, id, id),
                                  (tmem + C::SFA_COL + 4 * (kk / 2)) | (id << 30),
                                  (tmem + C::SFB_COL + 4 * (kk / 2)) | (id << 30), kk > 0 ? 1u : 0u);
                }
                ptx::tc_commit(&s_full[buf]);
                if (x.last()) ptx::tc_commit(&q_empty[item & 1]);
                return true;
            };
            const int page = a.c.page_size;
            auto issue_o = [&](const TileWalk& x, int g) {
                const int s = g % C::STAGES, buf = g & 1;
                if (!bounded_wait(&v_full[s], stage_parity(g), w, kPagedVFull)) return false;
                if (!bounded_wait(&p_full[buf], two_parity(g), w, kPagedPFull)) return false;
                if (g >= 2 && !bounded_wait(&o_free[buf], two_parity(g - 2), w, kPagedOFree)) return false;
                ptx::tc_fence_after();
                const int steps = max(1, (x.keys() + 15) / 16);
                const uint32_t v0 = ptx::smem_u32(stage_of(g) + C::K_BYTES);
                for (int kk = 0; kk < steps; kk++) {
                    const int row = kk * 16, pg = row >> a.c.page_shift;
                    const uint32_t at = v0 + pg * page * D * 2 + (row & (page - 1)) * C::CB;
#pragma unroll
                    for (int part = 0; part < C::PARTS; part++) {
                        const uint64_t pd = ptx::make_sdesc(
                            ptx::smem_u32(smem + C::OFF_P + (buf * C::PARTS + part) * C::P_BYTES) + row * C::PROW,
                            C::P_BYTES, 8 * C::PROW, C::PSW);
#pragma unroll
                        for (int m = 0; m < C::MT; m++)
                            ptx::mma_f16_ss(tmem + C::O_COL + (buf * C::MT + m) * NH,
                                            ptx::make_sdesc(at + m * (128 / C::CHE) * page * C::CB, page * C::CB, 8 * C::CB, C::VSW),
                                            pd, idesc_o, (kk > 0 || part > 0) ? 1u : 0u);
                    }
                }
                ptx::tc_commit(&o_full[buf]);
                ptx::tc_commit(&empty[s]);
                return true;
            };
            TileWalk o = t;
            int gs = 0, go = 0;
            bool ok = true;
            if (t.left > 0) {
                ok = issue_s(t, gs++);
                t.next(a);
            }
            while (ok && o.left > 0) {
                if (t.left > 0) {
                    if (!(ok = issue_s(t, gs++))) break;
                    t.next(a);
                }
                ok = issue_o(o, go++);
                o.next(a);
            }
            // Everything issued completes before Tensor Memory is freed.
            ptx::tc_commit(drain);
            bounded_drain(drain, 0, 2 * a.timeout_ns);
        }
        __syncwarp();
    } else if (warp == 2) {
        // ------------------------------------------------------------ scales
        // Lane l writes row l of each atom: the scales of keys l, 32 + l, 64 + l, 96 + l.
        for (int g = 0; t.left > 0; t.next(a), g++) {
            const int buf = g & 1;
            if (!__all_sync(~0u, bounded_wait(&k_full[g % C::STAGES], stage_parity(g), w, kPagedKFull))) break;
            // (the S^T MMAs of tile g - 2 have read this atom buffer)
            if (g >= 2 && !__all_sync(~0u, bounded_wait(&s_full[buf], two_parity(g - 2), w, kPagedSFull))) break;
            const uint8_t* raw = stage_of(g) + C::K_BYTES + C::V_BYTES;
#pragma unroll
            for (int i = 0; i < C::ATOMS; i++) {
                uint32_t word[4];
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const uint8_t* p = raw + (c * 32 + lane) * C::NB + 4 * i;
                    if constexpr (C::NB % 4 == 0) {
                        word[c] = *reinterpret_cast<const uint32_t*>(p);
                    } else {
                        word[c] = 0u;
#pragma unroll
                        for (int j = 0; j < 4; j++) word[c] |= (4 * i + j < C::NB ? p[j] : 127u) << (8 * j);
                    }
                }
                *reinterpret_cast<uint4*>(smem + C::OFF_KSF + (buf * C::ATOMS + i) * 512 + lane * 16) =
                    make_uint4(word[0], word[1], word[2], word[3]);
            }
            ptx::fence_proxy_async_smem();
            ptx::mbar_arrive(&sf_full[buf]);
        }
    } else if (warp == 3) {
        // ------------------------------------------------------------ queries
        int item = 0;
        for (; t.left > 0; t.next(a)) {
            if (!t.first) continue;
            const int buf = item & 1;
            if (item >= 2 && !__all_sync(~0u, bounded_wait(&q_empty[buf], two_parity(item - 2), w, kPagedQEmpty))) break;
            const int h0 = (t.hg % a.splits) * a.heads_per_group, nh = min(a.heads_per_group, a.group - h0);
            const int64_t q0 = t.b * a.qb + (static_cast<int64_t>(t.hg / a.splits) * a.group + h0) * a.qh;
            for (int i = lane; i < nh * C::NB; i += 32) {
                const int r = i / C::NB, blk = i % C::NB;
                uint4 packed;
                const int64_t at = q0 + r * a.qh + blk * 32;
                uint32_t sb = a.q_half ? quantize32<__half>(static_cast<const __half*>(a.q) + at, a.ocp, packed)
                                       : quantize32<float>(static_cast<const float*>(a.q) + at, a.ocp, packed);
                if (sb == 255u) sb = 254u;
                const int sw = C::KROW == 32 ? (r >> 2) & 1 : C::KROW == 64 ? (r >> 1) & 3 : r & 7;
                *reinterpret_cast<uint4*>(smem + C::OFF_Q + buf * C::Q_BYTES + r * C::KROW + ((blk ^ sw) * 16)) = packed;
                smem[C::OFF_QSF + (buf * C::ATOMS + blk / 4) * 512 + r * 16 + blk % 4] = static_cast<uint8_t>(sb);
            }
            ptx::fence_proxy_async_smem();
            ptx::mbar_arrive(&q_full[buf]);
            item++;
        }
    } else {
        // ------------------------------------------------------------ softmax
        const int wq = warp - 4, row = wq * 32 + lane;  // key of the tile; head-dim row of O^T
        const uint32_t lanes = tmem + (static_cast<uint32_t>(wq * 32) << 16);
        constexpr float kGrowth = 8.f;  // how far (log2) a score may exceed the reference
        float m[NH], l[NH], o[C::MT][NH];
        bool ok = true;  // no wait of this thread has run out
        auto load_cols = [&](uint32_t col, uint32_t (&r)[NH]) {
            if constexpr (NH == 16) ptx::tmem_ld16(lanes + col, r);
            else ptx::tmem_ld32(lanes + col, r);
        };
        // Adds tile g's O^T to the registers.
        auto add_o = [&](int g) {
            const int buf = g & 1;
            if (!__all_sync(~0u, bounded_wait(&o_full[buf], two_parity(g), w, kPagedOFull))) {
                ok = false;
                return;
            }
            ptx::tc_fence_after();
            uint32_t r[C::MT][NH];
#pragma unroll
            for (int i = 0; i < C::MT; i++) load_cols(C::O_COL + (buf * C::MT + i) * NH, r[i]);
            ptx::tc_wait_ld();
            ptx::tc_fence_before();
            ptx::mbar_arrive(&o_free[buf]);
#pragma unroll
            for (int i = 0; i < C::MT; i++)
#pragma unroll
                for (int h = 0; h < NH; h++) o[i][h] += __uint_as_float(r[i][h]);
        };
        int g = 0;
        bool pending = false;  // tile g - 1's O^T is not yet added
        for (; t.left > 0; t.next(a), g++) {
            const int buf = g & 1, n = t.keys();
            const int h0 = (t.hg % a.splits) * a.heads_per_group, nh = min(a.heads_per_group, a.group - h0);
            if (t.first) {
#pragma unroll
                for (int h = 0; h < NH; h++) {
                    m[h] = -INFINITY;
                    l[h] = 0.f;
#pragma unroll
                    for (int i = 0; i < C::MT; i++) o[i][h] = 0.f;
                }
            }
            ok = __all_sync(~0u, bounded_wait(&s_full[buf], two_parity(g), w, kPagedSFull)) && ok;
            ptx::tc_fence_after();
            uint32_t sr[NH];
            load_cols(C::S_COL + buf * NH, sr);
            ptx::tc_wait_ld();
            ptx::tc_fence_before();
            ptx::mbar_arrive(&s_free[buf]);
            float x[NH];
            bool over = t.first || !ok;
#pragma unroll
            for (int h = 0; h < NH; h++) {
                x[h] = row < n ? __uint_as_float(sr[h]) * a.scale_log2 : -INFINITY;
                over |= h < nh && x[h] > m[h] + kGrowth;
            }
            if (ptx::named_bar_any(1, 128, over)) {
                // Rare: a new item, a score that outgrew the reference, or a
                // wait that ran out.  All 128 threads come here together.
                if (ptx::named_bar_any(1, 128, !ok)) break;
                if (pending) {
                    add_o(g - 1);
                    pending = false;
                }
#pragma unroll
                for (int h = 0; h < NH; h++) {
                    const float v = ptx::warp_max(x[h]);
                    if (lane == 0) red[wq * NH + h] = v;
                }
                ptx::named_bar_sync(1, 128);
#pragma unroll
                for (int h = 0; h < NH; h++) {
                    const float top = fmaxf(fmaxf(red[h], red[NH + h]), fmaxf(red[2 * NH + h], red[3 * NH + h]));
                    const float to = fmaxf(m[h], top);
                    const float alpha = m[h] == -INFINITY ? 0.f : ptx::ex2_approx(m[h] - to);
                    m[h] = to;
                    l[h] *= alpha;
#pragma unroll
                    for (int i = 0; i < C::MT; i++) o[i][h] *= alpha;
                }
                ptx::named_bar_sync(1, 128);  // (red is written again at the item's end)
            }
            // P of this key.  Its buffer was last read by tile g - 2's O^T, which is added.
            uint32_t ph[NH / 2], pl[NH / 2];
#pragma unroll
            for (int h = 0; h < NH; h += 2) {
                const float p0 = ptx::ex2_approx(x[h] - (m[h] == -INFINITY ? 0.f : m[h]));
                const float p1 = ptx::ex2_approx(x[h + 1] - (m[h + 1] == -INFINITY ? 0.f : m[h + 1]));
                l[h] += p0;
                l[h + 1] += p1;
                ph[h / 2] = ptx::pack_half2(p0, p1);
                if constexpr (kSplitP) {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&ph[h / 2]));
                    pl[h / 2] = ptx::pack_half2(p0 - f.x, p1 - f.y);
                }
            }
            uint8_t* p = smem + C::OFF_P + buf * C::PARTS * C::P_BYTES + row * C::PROW;
            const int sw = C::PROW == 32 ? (row >> 2) & 1 : (row >> 1) & 3;
#pragma unroll
            for (int u = 0; u < NH / 8; u++) {
                *reinterpret_cast<uint4*>(p + ((u ^ sw) * 16)) = make_uint4(ph[4 * u], ph[4 * u + 1], ph[4 * u + 2], ph[4 * u + 3]);
                if constexpr (kSplitP)
                    *reinterpret_cast<uint4*>(p + C::P_BYTES + ((u ^ sw) * 16)) =
                        make_uint4(pl[4 * u], pl[4 * u + 1], pl[4 * u + 2], pl[4 * u + 3]);
            }
            if (row >= n && row < max(16, (n + 15) / 16 * 16)) {
                // A key behind the last: whatever lies in its place of V (NaN
                // included) must not meet its weight of zero.
                ok = bounded_wait(&v_full[g % C::STAGES], stage_parity(g), w, kPagedVFull) && ok;
                const int page = a.c.page_size;
                uint8_t* v = stage_of(g) + C::K_BYTES + (row >> a.c.page_shift) * page * D * 2 + (row & (page - 1)) * C::CB;
                for (int c = 0; c < C::DCH; c++)
#pragma unroll
                    for (int u = 0; u < C::CB / 16; u++)
                        *reinterpret_cast<uint4*>(v + c * page * C::CB + u * 16) = make_uint4(0u, 0u, 0u, 0u);
            }
            __syncwarp();
            ptx::fence_proxy_async_smem();
            ptx::mbar_arrive(&p_full[buf]);
            if (pending) add_o(g - 1);
            pending = true;
            if (!t.last()) continue;
            // The item's end in this block.
            add_o(g);
            pending = false;
#pragma unroll
            for (int h = 0; h < NH; h++) {
                float v = l[h];
#pragma unroll
                for (int i = 16; i; i >>= 1) v += __shfl_xor_sync(~0u, v, i);
                if (lane == 0) red[wq * NH + h] = v;
            }
            ptx::named_bar_sync(1, 128);
#pragma unroll
            for (int h = 0; h < NH; h++) l[h] = (red[h] + red[NH + h]) + (red[2 * NH + h] + red[3 * NH + h]);
            const int at = count - t.left;          // this tile's place in the range
            const bool begun = t.tile <= at;        // the item's first tile is in the range
            const bool whole = begun && t.tile + 1 == t.tiles;
            const int slot = 2 * blockIdx.x + (t.tile < at ? 1 : 0);
            if (whole) {
                const int64_t o0 = static_cast<int64_t>(t.b) * a.q_heads + (t.hg / a.splits) * a.group + h0;
#pragma unroll
                for (int h = 0; h < NH; h++) {
                    if (h >= nh) break;
                    const float inv = l[h] > 0.f ? 1.0f / l[h] : 0.f;
#pragma unroll
                    for (int i = 0; i < C::MT; i++)
                        if (i * 128 + row < D)
                            static_cast<OutT*>(a.out)[(o0 + h) * D + i * 128 + row] = from_float<OutT>(o[i][h] * inv);
                    if (a.lse && row == h)
                        a.lse[o0 + h] = l[h] > 0.f ? (m[h] + log2f(l[h])) * 0.6931471805599453f : INFINITY;
                }
            } else {
                float* po = a.p.o + static_cast<int64_t>(slot) * NH * D;
#pragma unroll
                for (int h = 0; h < NH; h++) {
                    if (h >= nh) break;
#pragma unroll
                    for (int i = 0; i < C::MT; i++)
                        if (i * 128 + row < D) po[h * D + i * 128 + row] = o[i][h];
                    if (row == h) a.p.ml[slot * NH + h] = make_float2(m[h], l[h]);
                }
            }
            if (row == 0 && t.left == 1) {
                // What the join has to do for this block: the item begun here that goes on.
                int4 it = make_int4(-1, 0, 0, 0);
                if (begun && !whole) {
                    const int64_t total = range->total, last = range->first + at + (t.tiles - 1 - t.tile);  // its last tile
                    int c = static_cast<int>(last * range->blocks / total);
                    while (c + 1 < range->blocks && paged_first(total, c + 1, range->blocks) <= last) c++;
                    while (paged_first(total, c, range->blocks) > last) c--;
                    it = make_int4(t.b, t.hg, c, slot);
                }
                a.p.items[blockIdx.x] = it;
            }
            ptx::named_bar_sync(1, 128);  // (red is free again)
        }
        if (count == 0 && threadIdx.x == 128) a.p.items[blockIdx.x] = make_int4(-1, 0, 0, 0);
    }

    ptx::tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem, C::TMEM_COLS);
    }
}

// Block (j, h): head h of the item that attention block j began and others
// continued: their partial results, in the blocks' order.
template <typename OutT, int D, int NH>
__global__ void __launch_bounds__(128) paged_join_kernel(const __grid_constant__ PagedArgs a)
{
    ptx::grid_dependency_wait();
    const int4 it = a.p.items[blockIdx.x];
    if (it.x < 0) return;
    const int h = blockIdx.y, tid = threadIdx.x;
    const int h0 = (it.y % a.splits) * a.heads_per_group;
    if (h >= min(a.heads_per_group, a.group - h0)) return;
    __shared__ float weight[kPagedBlocks];
    __shared__ float red[8];
    const int parts = it.z - blockIdx.x + 1;
    auto slot = [&](int p) { return p == 0 ? it.w : 2 * (static_cast<int>(blockIdx.x) + p); };
    float top = -INFINITY;
    for (int p = tid; p < parts; p += 128) top = fmaxf(top, a.p.ml[slot(p) * NH + h].x);
    top = ptx::warp_max(top);
    if (tid % 32 == 0) red[tid / 32] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    float sum = 0.f;
    for (int p = tid; p < parts; p += 128) {
        const float2 ml = a.p.ml[slot(p) * NH + h];
        const float wgt = ptx::ex2_approx(ml.x - top);
        weight[p] = wgt;
        sum += wgt * ml.y;
    }
    for (int i = 16; i; i >>= 1) sum += __shfl_xor_sync(~0u, sum, i);
    if (tid % 32 == 0) red[4 + tid / 32] = sum;
    __syncthreads();
    sum = (red[4] + red[5]) + (red[6] + red[7]);
    const int64_t at = static_cast<int64_t>(it.x) * a.q_heads + (it.y / a.splits) * a.group + h0 + h;
    for (int d = tid; d < D; d += 128) {
        float o = 0.f;
#pragma unroll 4
        for (int p = 0; p < parts; p++) o = fmaf(weight[p], a.p.o[(static_cast<int64_t>(slot(p)) * NH + h) * D + d], o);
        static_cast<OutT*>(a.out)[at * D + d] = from_float<OutT>(o / sum);
    }
    if (a.lse && tid == 0) a.lse[at] = (top + log2f(sum)) * 0.6931471805599453f;
}

}  // namespace fp4attn
