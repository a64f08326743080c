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
// Roles (384 threads):
//   warp 0      key producer: a page's codes by TMA, its raw scales by a bulk
//               copy, into a ring of stages.
//   warp 1      value producer: a page's V by TMA.
//   warp 2      S^T issuer: brings the scales into the tensor core's layout,
//               then one thread issues the MMAs.
//   warp 3      O^T issuer (one thread).
//   warps 4-11  two softmax warpgroups, which take the items in turn, so that
//               one starts an item while the other finishes the one before:
//               thread = key (row of S^T), then head-dim row of O^T.  Each
//               quantises its own item's queries first.
// A single thread runs a dependent instruction in about six cycles and passes
// a ready barrier in about a hundred, and a tile has some 900 (head_dim 64) to
// 1,800 cycles (128) of the memory's time: one thread that issued both MMAs
// of a tile took 3,000 (0.196 ms for 64 sequences of up to 8192 tokens).
//
// The softmax reference m starts as the item's first tile's maximum and is
// moved only when a score exceeds it by more than 2^8; all threads hold the
// same m in registers and agree by one barrier with a vote.  The weights
// p = 2^(z - m), at most 2^8, enter the MMA as two FP16 parts in columns of
// their own,
//     hi = fp16(2^7 p),   lo = fp16(2^11 (2^7 p - hi)),   2^7 p ~ hi + 2^-11 lo,
// which keep 22 bits of every weight down to 2^-21 of the reference's, and
// below it lose at most 2^-43 of that: both factors use up FP16's range
// (2^7 2^8 = 2^15, and half a step there times 2^11 is 2^15 again).  One part,
// or parts that are not lifted, lose the weights of a long tail behind one
// dominating key (weights below 2^-25 vanish, while the sum still counts them).
// The second part costs FP16 output nothing where memory bounds it (113 us
// for 64 sequences of up to 8192 tokens, 8 x 32 heads of 128, either way) and
// the softmax's time for groups of 16 small heads (32 sequences of 1000 to 8000
// tokens, 8 x 128 heads of 64: 61 -> 68 us; of 32: 57 -> 71).
// Each tile's O^T is added to FP32 registers with proper rounding: only 128
// keys are summed inside the tensor core.
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

constexpr float kLift = 0x1p7f, kLowLift = 0x1p11f;  // the factors of P's parts, see above

// HC: query heads computed (4, 8 or 16, at least the group's share).
template <int D, int HC>
struct PagedCfg {
    static constexpr int THREADS = 384;
    // Tiles a step: the roles wait for one another once a step.  Tiles of
    // small heads are short, so two make a step.
    static constexpr int U = D <= 64 ? 2 : 1;
    static constexpr int NS = 16;                                    // N of the S^T MMA (the least there is)
    static constexpr int NP = HC == 16 ? 32 : 16;                    // N of the O^T MMA: the low parts from NP / 2 on
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
    static constexpr int PROW = 2 * NP;                              // bytes of a key's P row (= swizzle)
    static constexpr uint32_t PSW = PROW == 32 ? ptx::kSwizzle32B : ptx::kSwizzle64B;
    // Tensor Memory columns
    static constexpr int S_COL = 0;                                  // [2][U][NS]
    static constexpr int O_COL = 2 * U * NS;                         // [2][MT][NP]
    static constexpr int SFA_COL = O_COL + 2 * MT * NP;
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
    static constexpr int OFF_P = 0;                                  // [2][U][128 keys][PROW]
    static constexpr int P_BYTES = kPagedTile * PROW;
    static constexpr int OFF_Q = OFF_P + 2 * U * P_BYTES;            // [2 warpgroups][NS rows][KROW]
    static constexpr int Q_BYTES = align1k(NS * KROW);
    static constexpr int OFF_QSF = OFF_Q + 2 * Q_BYTES;              // [2][ATOMS][512]
    static constexpr int OFF_KSF = OFF_QSF + 2 * ATOMS * 512;        // [2][U][ATOMS][512]
    static constexpr int OFF_STAGE = align1k(OFF_KSF + 2 * U * ATOMS * 512);
    // The O^T MMA reads 128 rows (head-dim columns) of V: past head_dim it
    // reads on into what follows; those rows of O^T are not used.
    static constexpr int V_OVER = (MT * 128 - D) / CHE * kPagedTile * CB;
    static constexpr int MISC = 3 * 1024;                            // barriers, reductions
    static constexpr int kBudget = 227 * 1024 - 1024 - OFF_STAGE - MISC - V_OVER;
    static constexpr int STAGES = kBudget / STAGE < 8 ? kBudget / STAGE : 8;
    static_assert(STAGES >= 2, "shared memory budget exceeded");
    static constexpr int OFF_MISC = OFF_STAGE + STAGES * STAGE + V_OVER;
    static constexpr int SMEM_BYTES = OFF_MISC + MISC + 1024;
};

// The partial results of an item that spans blocks: slot 2 * block for a range
// that began inside the item, 2 * block + 1 for the item begun in the range.
struct PagedPartials {
    float* o;        // [2 * kPagedBlocks][HC][D]
    float2* ml;      // [2 * kPagedBlocks][HC]  reference (log2 domain), sum
    int4* items;     // [kPagedBlocks]  sequence, head group, last block, first slot; sequence -1: none begun here goes on
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
    const int len = a.seq_lens[b];
    const int64_t most = static_cast<int64_t>(a.t.max_pages) << a.c.page_shift;
    return len < 0 ? 0 : len > most ? static_cast<int>(most) : len;
}

// Tiles of a sequence; an empty one has one (without keys), which writes its zeros.
__device__ __forceinline__ int paged_tiles(int len) { return len <= 0 ? 1 : (len + kPagedTile - 1) / kPagedTile; }

// First tile of a block's range, and the block whose range holds a tile:
// `total` tiles dealt to `blocks` blocks (at most `total`), the first
// total % blocks of which have one more.
__device__ __forceinline__ int paged_first(int total, int block, int blocks)
{
    return block * (total / blocks) + min(block, total % blocks);
}
__device__ __forceinline__ int paged_block(int total, int tile, int blocks)
{
    const int base = total / blocks, more = total % blocks, head = more * (base + 1);
    return tile < head ? tile / (base + 1) : more + (tile - head) / base;
}

// The walk over the items, or parts of items, in a block's range; every role
// makes its own.
struct ItemWalk {
    int b, head, split, tile, n, left;  // the part: its first tile and number of tiles; tiles left in the range, its own included
    int len, tiles;                     // the sequence's
    __device__ __forceinline__ void begin(const PagedArgs& a, const int4& start, int count)
    {
        b = start.x;
        head = start.y / a.splits;  // (the only division: later ones would be on the way from item to item)
        split = start.y % a.splits;
        tile = start.z;
        left = count;
        n = 0;
        if (left > 0) {
            len = paged_length(a, b);
            tiles = paged_tiles(len);
            n = min(left, tiles - tile);
        }
    }
    __device__ __forceinline__ void next(const PagedArgs& a)
    {
        left -= n;
        tile = 0;
        if (left > 0 && ++split == a.splits) {
            split = 0;
            if (++head == a.c.kv_heads) {
                head = 0;
                b++;
                len = paged_length(a, b);
                tiles = paged_tiles(len);
            }
        }
        n = min(left, tiles);
    }
    __device__ __forceinline__ bool first_of_sequence() const { return tile == 0 && head == 0 && split == 0; }
    // Keys of the part's i-th tile.
    __device__ __forceinline__ int keys(int i) const { return max(0, min(kPagedTile, len - (tile + i) * kPagedTile)); }
};

// A position in a ring of N stages and the parity of the stage's use.
template <int N>
struct Ring {
    int s = 0;
    uint32_t parity = 0;
    __device__ __forceinline__ void next()
    {
        if (++s == N) {
            s = 0;
            parity ^= 1u;
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

// This block's range, by a scan of the lengths with the first 256 threads
// (every thread of the block calls it).
__device__ __forceinline__ void find_range(const PagedArgs& a, PagedRange* range, int* scratch)
{
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
    const bool scans = tid < 256;
    // With up to 256 sequences one scan gives the total as well; with more, a
    // sum over all of them comes first.
    int sum = 0;
    if (a.batch > 256) {
        if (scans) {
            for (int b = tid; b < a.batch; b += 256) sum += paged_tiles(paged_length(a, b));
            sum = __reduce_add_sync(~0u, sum);
            if (lane == 0) scratch[warp] = sum;
        }
        __syncthreads();
        sum = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) sum += scratch[i];
    }
    int carry = 0;  // tiles (of one head group) of the sequences before this chunk
    for (int b0 = 0; b0 < a.batch; b0 += 256) {
        const int mine = scans && b0 + tid < a.batch ? paged_tiles(paged_length(a, b0 + tid)) : 0;
        int inc = mine;
#pragma unroll
        for (int i = 1; i < 32; i <<= 1) {
            const int v = __shfl_up_sync(~0u, inc, i);
            if (lane >= i) inc += v;
        }
        if (a.batch > 256) __syncthreads();  // (the last chunk's sums have been read)
        if (scans && lane == 31) scratch[warp] = inc;
        __syncthreads();
        int before = carry, all = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            if (i < warp) before += scratch[i];
            all += scratch[i];
        }
        if (a.batch <= 256) sum = all;
        const int total = sum * a.head_groups, blocks = min(total, static_cast<int>(gridDim.x));
        const bool idle = static_cast<int>(blockIdx.x) >= blocks;
        const int t0 = idle ? 0 : paged_first(total, blockIdx.x, blocks);
        const int at = (before + inc - mine) * a.head_groups;
        if (scans && !idle && t0 >= at && t0 < at + mine * a.head_groups) {
            const int in = t0 - at;
            range->start = make_int4(b0 + tid, in / mine, in % mine, 0);
        }
        if (tid == 0) {
            range->first = t0;
            range->count = idle ? 0 : paged_first(total, blockIdx.x + 1, blocks) - t0;
            range->total = total;
            range->blocks = blocks;
        }
        carry += all;
    }
}

// Of four values per lane: the warp's `op` of the q-th, in the lanes with
// (lane >> 3) == q.  Six shuffles (each pair of them halves what a lane holds).
template <typename Op>
__device__ __forceinline__ float warp_reduce4(const float (&v)[4], int lane, Op op)
{
    const bool up = lane & 16, up2 = lane & 8;
    const float k0 = op(up ? v[2] : v[0], __shfl_xor_sync(~0u, up ? v[0] : v[2], 16));
    const float k1 = op(up ? v[3] : v[1], __shfl_xor_sync(~0u, up ? v[1] : v[3], 16));
    float k = op(up2 ? k1 : k0, __shfl_xor_sync(~0u, up2 ? k0 : k1, 8));
    k = op(k, __shfl_xor_sync(~0u, k, 4));
    k = op(k, __shfl_xor_sync(~0u, k, 2));
    return op(k, __shfl_xor_sync(~0u, k, 1));
}

// What runs once an item or less is out of line: the roles' loops together just
// about fill the SM's instruction cache, and with the rest between them they
// took up to a quarter longer.

// Eight elements of a query row, quantised with those of the three neighbouring
// lanes: their codes, and the block's scale byte.  (encode8<float> is exact for
// FP16 too.)
static __device__ __noinline__ uint2 quantize_query8(const void* q, int64_t at, int half, int ocp)
{
    float v[8];
    if (half) load8v(static_cast<const __half*>(q) + at, v);
    else load8v(static_cast<const float*>(q) + at, v);
    float amax = 0.f;
#pragma unroll
    for (int e = 0; e < 8; e++) amax = fmaxf(amax, fabsf(v[e]));
    const uint32_t quad = 0xFu << ((threadIdx.x & 31) & ~3);
    amax = fmaxf(amax, __shfl_xor_sync(quad, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(quad, amax, 2));
    const uint32_t sb = scale_byte(amax, ocp);
    return make_uint2(encode8<float>(v, sb), sb == 255u ? 254u : sb);
}

// Zeroes V of keys [keys, end) of a stage's tile: thread `row` of 128.
template <int D, int CB>
__device__ __noinline__ void zero_keys(uint8_t* v, int keys, int end, int page, int shift, int row)
{
    for (int k = row; k < (end - keys) * (D / 8); k += 128) {
        const int key = keys + k / (D / 8), c = k % (D / 8);
        *reinterpret_cast<uint4*>(v + (key >> shift) * page * D * 2 + c / (CB / 16) * page * CB + (key & (page - 1)) * CB +
                                  c % (CB / 16) * 16) = make_uint4(0u, 0u, 0u, 0u);
    }
}

// copy(p, id[p]) for pages 0 .. n - 1 of a tile (at most 8), by one elected
// thread, in runs of 8, 4, 2 and 1.  With a condition on each copy, one took 85
// cycles to issue instead of 20.
template <typename F>
__device__ __forceinline__ void each_page(int n, const int (&id)[8], F copy)
{
    if (n == 8) {
#pragma unroll
        for (int p = 0; p < 8; p++) copy(p, id[p]);
        return;
    }
    const bool four = n & 4;
    if (four) {
#pragma unroll
        for (int p = 0; p < 4; p++) copy(p, id[p]);
    }
    if (n & 2) {
        copy(four ? 4 : 0, four ? id[4] : id[0]);
        copy(four ? 5 : 1, four ? id[5] : id[1]);
    }
    const int last = n & 6;
    if (n & 1) copy(last, last == 0 ? id[0] : last == 2 ? id[2] : last == 4 ? id[4] : id[6]);
}

// kWithhold (test instantiation only, fp4attn_selftest_paged_abort): one thread
// of block 0 never reports its first weights, so the O^T issuer's wait runs out.
template <typename OutT, int D, int HC, bool kWithhold = false>
__global__ void __launch_bounds__(384, 1)
    paged_attention_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                           const __grid_constant__ PagedArgs a)
{
    using C = PagedCfg<D, HC>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_MISC);
    uint64_t* k_full = bars;               // [8] codes and scales of a stage landed
    uint64_t* v_full = k_full + 8;         // [8] values landed
    uint64_t* empty = v_full + 8;          // [8] the stage's MMAs are done (commit)
    uint64_t* q_full = empty + 8;          // [2] an item's query codes and scales written (128), by warpgroup
    // (these by step)
    uint64_t* s_full = q_full + 2;        // [2][2] S^T computed (commit); by warpgroup, see below
    uint64_t* s_free = s_full + 4;         // [2] S^T in registers (128)
    uint64_t* p_full = s_free + 2;         // [2] P written (128)
    uint64_t* o_full = p_full + 2;         // [2] O^T computed, P read (commit)
    uint64_t* o_free = o_full + 2;         // [2] O^T in registers (128)
    uint64_t* drain = o_free + 2;          // [2] everything an issuer issued is done (exit)
    float* red_all = reinterpret_cast<float*>(smem + C::OFF_MISC + 512);  // [2 warpgroups][maxima, sums][4][HC]
    int* scratch = reinterpret_cast<int*>(smem + C::OFF_MISC + 2560);     // [8]
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
            ptx::mbar_init(&q_full[i], 128);
            ptx::mbar_init(&s_full[i], 1);
            ptx::mbar_init(&s_full[2 + i], 1);
            ptx::mbar_init(&s_free[i], 128);
            ptx::mbar_init(&p_full[i], 128);
            ptx::mbar_init(&o_full[i], 1);
            ptx::mbar_init(&o_free[i], 128);
            ptx::mbar_init(&drain[i], 1);
        }
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
    for (int i = threadIdx.x; i < 2 * C::Q_BYTES / 16; i += C::THREADS)
        reinterpret_cast<uint4*>(smem + C::OFF_Q)[i] = make_uint4(0u, 0u, 0u, 0u);
    for (int i = threadIdx.x; i < 2 * C::ATOMS * 32; i += C::THREADS)
        reinterpret_cast<uint4*>(smem + C::OFF_QSF)[i] = make_uint4(0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu);
    ptx::fence_proxy_async_smem();
    // Everything before this overlaps the grid before this one in the stream.
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    // Nothing to join, until this block's last item says otherwise: the join reads
    // this word even when a wait here runs out and the items are not finished.
    if (threadIdx.x == 0) a.p.items[blockIdx.x] = make_int4(-1, 0, 0, 0);
    find_range(a, range, scratch);
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = *tmem_sh;
    const int count = range->count;
    const ServingWait w{abort_sh, a.timeout_ns};
    uint8_t* const stages = smem + C::OFF_STAGE;
    const int page = a.c.page_size, shift = a.c.page_shift;
    ItemWalk t;
    t.begin(a, range->start, count);

    if (warp <= 1) {
        // ------------------------------------------------------------ producers
        const bool keys_role = warp == 0;
        Ring<C::STAGES> ring;
        int g = 0;
        bool ok = true;
        for (; ok && t.left > 0; t.next(a)) {
            const int head = t.head;
            const uint8_t* scales = a.c.k_scales + static_cast<int64_t>(head) * page * C::NB;
            const int32_t* row = a.t.pages + t.b * a.t.stride + ((t.tile * kPagedTile) >> shift) + lane;
            const int step = kPagedTile >> shift;  // pages of a tile; lane p has the p-th
            int left = lane < step ? (t.len - t.tile * kPagedTile + page - 1) >> shift : 0;  // pages from this tile on
            int id = lane < left ? *row : 0;
            for (int i = 0; i < t.n; i++, g++, ring.next()) {
                row += step;
                left -= step;
                const int next_id = i + 1 < t.n && lane < left ? *row : 0;
                if (id < 0 || id >= a.c.pages) {
                    record_index_error(kIndexPage, id);
                    id = 0;
                }
                int pid[8];
#pragma unroll
                for (int p = 0; p < 8; p++) pid[p] = __shfl_sync(~0u, id, p);
                const int n = (t.keys(i) + page - 1) >> shift;
                uint8_t* st = stages + ring.s * C::STAGE;
                if (g >= C::STAGES && !__all_sync(~0u, bounded_wait(&empty[ring.s], ring.parity ^ 1u, w, kPagedEmpty))) {
                    ok = false;
                    break;
                }
                if (ptx::elect_one()) {
                    if (keys_role) {
                        ptx::mbar_arrive_expect_tx(&k_full[ring.s], n * page * (C::KROW + C::NB));
                        each_page(n, pid, [&](int p, int at) {
                            ptx::tma_load_4d(st + p * page * C::KROW, &tm_k, &k_full[ring.s], 0, head, at);
                            ptx::bulk_load(st + C::K_BYTES + C::V_BYTES + p * page * C::NB, scales + at * a.c.k_scales_stride,
                                           page * C::NB, &k_full[ring.s]);
                        });
                    } else {
                        ptx::mbar_arrive_expect_tx(&v_full[ring.s], n * page * D * 2);
                        each_page(n, pid, [&](int p, int at) {
                            ptx::tma_load_5d(st + C::K_BYTES + p * page * D * 2, &tm_v, &v_full[ring.s], 0, 0, head, at);
                        });
                    }
                }
                __syncwarp();
                id = next_id;
            }
        }
        // Every copy issued lands before the block exits.
        if (lane == 0)
            for (int i = max(0, g - C::STAGES); i < g; i++)
                bounded_drain(keys_role ? &k_full[i % C::STAGES] : &v_full[i % C::STAGES],
                              static_cast<uint32_t>(i / C::STAGES) & 1u, 2 * a.timeout_ns);
        __syncwarp();
    } else if (warp == 2) {
        // ------------------------------------------------------------ S^T issuer
        constexpr uint32_t qk_sw = ptx::swizzle_mode_for_bytes(C::KROW);
        const uint64_t kd0 = ptx::make_sdesc(ptx::smem_u32(stages), 16, 8 * C::KROW, qk_sw);
        const uint64_t qd0 = ptx::make_sdesc(ptx::smem_u32(smem + C::OFF_Q), 16, 8 * C::KROW, qk_sw);
        const uint64_t sfa0 = ptx::make_sdesc(ptx::smem_u32(smem + C::OFF_KSF), 0, 128, ptx::kSwizzleNone);
        const uint64_t sfb0 = ptx::make_sdesc(ptx::smem_u32(smem + C::OFF_QSF), 0, 128, ptx::kSwizzleNone);
        Ring<C::STAGES> ring;
        // A warpgroup waits for its own tiles only, and a barrier's parity tells
        // a phase from the one before it alone: so each has its own barriers,
        // used in the order of its tiles.
        int g = 0, own[2] = {0, 0};
        bool ok = true;
        for (int item = 0; ok && t.left > 0; t.next(a), item++) {
            const int wg = item & 1;
            int j = own[wg];
            const int n_steps = (t.n + C::U - 1) / C::U;
            own[wg] += n_steps;
            for (int i = 0; i < n_steps; i++, g++, j++) {
                const int buf = g & 1;
                // S^T and the scale atoms of step g - 2 have been read.
                bool go = g < 2 || bounded_wait(&s_free[buf], static_cast<uint32_t>((g - 2) / 2) & 1u, w, kPagedSFree);
                if (i == 0) go = bounded_wait(&q_full[wg], static_cast<uint32_t>(item / 2) & 1u, w, kPagedQFull) && go;
#pragma unroll
                for (int u = 0; u < C::U; u++) {
                    if (u > 0 && i * C::U + u >= t.n) break;
                    go = bounded_wait(&k_full[ring.s], ring.parity, w, kPagedKFull) && go;
                    if (!__all_sync(~0u, go)) {
                        ok = false;
                        break;
                    }
                    // Lane l writes row l of each atom: the scales of keys l, 32 + l, 64 + l, 96 + l.
                    const uint8_t* raw = stages + ring.s * C::STAGE + C::K_BYTES + C::V_BYTES;
#pragma unroll
                    for (int k = 0; k < C::ATOMS; k++) {
                        uint32_t word[4];
#pragma unroll
                        for (int c = 0; c < 4; c++) {
                            const uint8_t* p = raw + (c * 32 + lane) * C::NB + 4 * k;
                            if constexpr (C::NB % 4 == 0) {
                                word[c] = *reinterpret_cast<const uint32_t*>(p);
                            } else {
                                word[c] = 0u;
#pragma unroll
                                for (int e = 0; e < 4; e++) word[c] |= (4 * k + e < C::NB ? p[e] : 127u) << (8 * e);
                            }
                        }
                        *reinterpret_cast<uint4*>(smem + C::OFF_KSF + ((buf * C::U + u) * C::ATOMS + k) * 512 + lane * 16) =
                            make_uint4(word[0], word[1], word[2], word[3]);
                    }
                    ptx::fence_proxy_async_smem();
                    __syncwarp();
                    if (ptx::elect_one()) {
                        ptx::tc_fence_after();
                        if (i == 0 && u == 0)
#pragma unroll
                            for (int k = 0; k < C::ATOMS; k++)
                                ptx::tc_cp_32x128b_warpx4(tmem + C::SFB_COL + 4 * k, sfb0 + (wg * C::ATOMS + k) * (512 / 16));
#pragma unroll
                        for (int k = 0; k < C::ATOMS; k++)
                            ptx::tc_cp_32x128b_warpx4(tmem + C::SFA_COL + 4 * k, sfa0 + ((buf * C::U + u) * C::ATOMS + k) * (512 / 16));
                        const uint64_t kd = kd0 + static_cast<uint64_t>(ring.s * (C::STAGE / 16)), qd = qd0 + wg * (C::Q_BYTES / 16);
#pragma unroll
                        for (int kk = 0; kk < C::KSTEPS; kk++) {
                            const uint32_t id = 2u * (kk & 1);
                            ptx::mma_mxf4(tmem + C::S_COL + (buf * C::U + u) * C::NS, kd + 2 * kk, qd + 2 * kk,
                                          ptx::idesc_mxf4(128, C::NS, id, id), (tmem + C::SFA_COL + 4 * (kk / 2)) | (id << 30),
                                          (tmem + C::SFB_COL + 4 * (kk / 2)) | (id << 30), kk > 0 ? 1u : 0u);
                        }
                    }
                    __syncwarp();
                    ring.next();
                }
                if (!ok) break;
                if (ptx::elect_one()) ptx::tc_commit(&s_full[2 * wg + (j & 1)]);
            }
        }
        if (ptx::elect_one()) {  // everything issued completes before Tensor Memory is freed
            ptx::tc_commit(&drain[0]);
            bounded_drain(&drain[0], 0, 2 * a.timeout_ns);
        }
        __syncwarp();
    } else if (warp == 3) {
        // ------------------------------------------------------------ O^T issuer
        // (elect.sync, not a lane number: the compiler then knows that one
        // thread runs this, and an MMA takes 47 cycles to issue instead of 105)
        if (ptx::elect_one()) {
            constexpr uint32_t idesc_o = ptx::idesc_f16x(128, C::NP, 0, true, true);
            // V's 16-key steps within a stage, in 16-byte units: rows within a page, page by page.
            const int page_shift = shift - 4, page_mask = (1 << page_shift) - 1, page_step = page * D * 2 / 16;
            const uint64_t vd0 = ptx::make_sdesc(ptx::smem_u32(stages + C::K_BYTES), page * C::CB, 8 * C::CB, C::VSW);
            const uint64_t pd0 = ptx::make_sdesc(ptx::smem_u32(smem + C::OFF_P), C::P_BYTES, 8 * C::PROW, C::PSW);
            const uint32_t m_step = static_cast<uint32_t>((128 / C::CHE) * page * C::CB / 16);
            Ring<C::STAGES> ring;
            int g = 0;
            bool ok = true;
            for (; ok && t.left > 0; t.next(a)) {
                const int n_steps = (t.n + C::U - 1) / C::U;
                for (int i = 0; ok && i < n_steps; i++, g++) {
                    const int buf = g & 1;
                    ok = (g < 2 || bounded_wait(&o_free[buf], static_cast<uint32_t>((g - 2) / 2) & 1u, w, kPagedOFree)) &&
                         bounded_wait(&p_full[buf], static_cast<uint32_t>(g / 2) & 1u, w, kPagedPFull);
#pragma unroll
                    for (int u = 0; u < C::U; u++) {
                        const int ti = i * C::U + u;
                        if (u > 0 && ti >= t.n) break;
                        ok = ok && bounded_wait(&v_full[ring.s], ring.parity, w, kPagedVFull);
                        if (!ok) break;
                        ptx::tc_fence_after();
                        const uint64_t vd = vd0 + static_cast<uint64_t>(ring.s * (C::STAGE / 16));
                        const uint64_t pd = pd0 + static_cast<uint64_t>((buf * C::U + u) * C::P_BYTES / 16);
                        const uint32_t od = tmem + C::O_COL + buf * C::MT * C::NP;
                        const int keys = t.keys(ti);
                        const int steps = max(1, (keys + 15) / 16);
#pragma unroll 1
                        for (int kk = 0; kk < steps; kk++) {
                            // 16 keys further within a page, or to the next page.
                            const uint32_t v = (kk & page_mask) * (16 * C::CB / 16) + (kk >> page_shift) * page_step;
#pragma unroll
                            for (int m = 0; m < C::MT; m++)
                                ptx::mma_f16_ss(od + m * C::NP, vd + (v + m * m_step), pd + kk * C::PROW, idesc_o,
                                                (kk > 0 || u > 0) ? 1u : 0u);
                        }
                        ptx::tc_commit(&empty[ring.s]);
                        ring.next();
                    }
                    if (ok) ptx::tc_commit(&o_full[buf]);
                }
            }
            ptx::tc_commit(&drain[1]);
            bounded_drain(&drain[1], 0, 2 * a.timeout_ns);
        }
        __syncwarp();
    } else {
        // ------------------------------------------------------------ softmax
        const int wg = (warp - 4) / 4, wq = warp % 4, row = wq * 32 + lane;  // key of the tile; head-dim row of O^T
        const uint32_t lanes = tmem + (static_cast<uint32_t>(wq * 32) << 16);
        const int bar_id = 1 + wg;
        // (A warp writes sums only after all 128 threads have read the maxima, and
        // the other way round: an item's O^T needs the P of every thread.)
        float* red = red_all + wg * 8 * HC;
        float* red_sum = red + 4 * HC;
        constexpr float kGrowth = 8.f;  // how far (log2) a score may exceed the reference
        float nm[HC], l[HC], o[C::MT][HC];  // minus the reference, this thread's sums, O^T
        bool ok = true;  // no wait of this thread has run out
        auto load_cols = [&](uint32_t col, uint32_t (&r)[HC]) {
            if constexpr (HC == 4) ptx::tmem_ld4(lanes + col, r);
            else if constexpr (HC == 8) ptx::tmem_ld8(lanes + col, r);
            else ptx::tmem_ld16(lanes + col, r);
        };
        auto max_of = [](float x, float y) { return fmaxf(x, y); };
        auto sum_of = [](float x, float y) { return x + y; };
        Ring<C::STAGES> ring;
        int g = 0, j = 0;  // step of the block, step of this warpgroup
        for (int item = 0; t.left > 0; t.next(a), item++) {
            const int n_steps = (t.n + C::U - 1) / C::U;
            if ((item & 1) != wg) {  // the other warpgroup's
                g += n_steps;
                for (int i = t.n % C::STAGES; i > 0; i--) ring.next();
                ring.parity ^= static_cast<uint32_t>(t.n / C::STAGES) & 1u;
                continue;
            }
            const int h0 = t.split * a.heads_per_group, nh = min(a.heads_per_group, a.group - h0);
            // This item's queries, while the other warpgroup has the item before.
            // (S^T of this warpgroup's last item, the buffer's last use, is computed.)
            {
                const int64_t q0 = t.b * a.qb + (static_cast<int64_t>(t.head) * a.group + h0) * a.qh;
                for (int k = row; k < nh * C::NB * 4; k += 128) {  // a thread per eight elements
                    const int r = k / (C::NB * 4), blk = k / 4 % C::NB, quarter = k % 4;
                    const uint2 q8 = quantize_query8(a.q, q0 + r * a.qh + blk * 32 + quarter * 8, a.q_half, a.ocp);
                    const int sw = C::KROW == 32 ? (r >> 2) & 1 : C::KROW == 64 ? (r >> 1) & 3 : r & 7;
                    *reinterpret_cast<uint32_t*>(smem + C::OFF_Q + wg * C::Q_BYTES + r * C::KROW + ((blk ^ sw) * 16) + quarter * 4) = q8.x;
                    if (quarter == 0) smem[C::OFF_QSF + (wg * C::ATOMS + blk / 4) * 512 + r * 16 + blk % 4] = static_cast<uint8_t>(q8.y);
                }
                ptx::fence_proxy_async_smem();
                ptx::mbar_arrive(&q_full[wg]);
                if (row == 127 && t.first_of_sequence()) {
                    const int len = a.seq_lens[t.b];
                    if (len != t.len) record_index_error(kIndexLength, len);
                }
            }
            bool out_of_time = false;
            // Step i: P, then the O^T of step i - 1 is added (the last has no P).
            for (int i = 0; i <= n_steps; i++) {
                float beta[HC];  // what moves step i - 1's O^T to the present reference
#pragma unroll
                for (int h = 0; h < HC; h++) beta[h] = 1.f;
                if (i < n_steps) {
                    const int buf = g & 1;
                    ok = bounded_wait(&s_full[2 * wg + (j & 1)], static_cast<uint32_t>(j / 2) & 1u, w, kPagedSFull) && ok;
                    __syncwarp();
                    ptx::tc_fence_after();
                    uint32_t sr[C::U][HC];
#pragma unroll
                    for (int u = 0; u < C::U; u++) load_cols(C::S_COL + (buf * C::U + u) * C::NS, sr[u]);
                    ptx::tc_wait_ld();
                    ptx::tc_fence_before();
                    ptx::mbar_arrive(&s_free[buf]);
                    float x[C::U][HC];  // the scores, log2 domain, less the reference
                    bool over = !ok;
#pragma unroll
                    for (int u = 0; u < C::U; u++) {
                        const int keys = i * C::U + u < t.n ? t.keys(i * C::U + u) : 0;
                        if (row >= keys)
#pragma unroll
                            for (int h = 0; h < HC; h++) sr[u][h] = 0xFF800000u;  // -inf
#pragma unroll
                        for (int h = 0; h < HC; h++) {
                            if (i == 0) nm[h] = 0.f;
                            x[u][h] = fmaf(__uint_as_float(sr[u][h]), a.scale_log2, nm[h]);
                            over |= x[u][h] > kGrowth;
                        }
                    }
                    if (i == 0 || ptx::named_bar_any(bar_id, 128, over)) {
                        // A new item, or, rarely, a score that outgrew the reference or
                        // a wait that ran out.  All 128 threads come here together.
#pragma unroll
                        for (int c = 0; c < HC / 4; c++) {
                            float v[4];
#pragma unroll
                            for (int q = 0; q < 4; q++) v[q] = C::U == 2 ? fmaxf(x[0][4 * c + q], x[C::U - 1][4 * c + q]) : x[0][4 * c + q];
                            const float top = warp_reduce4(v, lane, max_of);
                            if ((lane & 7) == 0) red[wq * HC + 4 * c + (lane >> 3)] = top;
                        }
                        if (ptx::named_bar_any(bar_id, 128, !ok)) {
                            out_of_time = true;
                            break;
                        }
#pragma unroll
                        for (int h = 0; h < HC; h++) {
                            const float top = fmaxf(fmaxf(red[h], red[HC + h]), fmaxf(red[2 * HC + h], red[3 * HC + h]));
                            // How far the reference moves: up, or at an item's start to the
                            // maximum (0 when there is no key at all).
                            const float up = i > 0 ? fmaxf(top, 0.f) : top == -INFINITY ? 0.f : top;
                            beta[h] = i > 0 ? ptx::ex2_approx(-up) : 0.f;
                            nm[h] -= up;
#pragma unroll
                            for (int u = 0; u < C::U; u++) x[u][h] -= up;
                            l[h] = i > 0 ? l[h] * beta[h] : 0.f;
#pragma unroll
                            for (int m = 0; m < C::MT; m++) o[m][h] = i > 0 ? o[m][h] * beta[h] : 0.f;
                        }
                    }
                    // P of these keys.  Its buffer was last read by step g - 2's O^T:
                    // added already, unless the other warpgroup had it.  (Step g - 4's
                    // is complete then, so the parity is unambiguous: if it was the
                    // other warpgroup's, that added it before it read S^T of g - 2.)
                    if (i < 2 && g >= 2)
                        ok = bounded_wait(&o_full[buf], static_cast<uint32_t>((g - 2) / 2) & 1u, w, kPagedOFull) && ok;
#pragma unroll
                    for (int u = 0; u < C::U; u++) {
                        if (u > 0 && i * C::U + u >= t.n) break;
                        uint32_t hi[HC / 2], lo[HC / 2];
#pragma unroll
                        for (int h = 0; h < HC; h += 2) {
                            const float p0 = ptx::ex2_approx(x[u][h]), p1 = ptx::ex2_approx(x[u][h + 1]);
                            l[h] += p0;
                            l[h + 1] += p1;
                            const float2 p = make_float2(p0, p1), lifted = ptx::fmul2(p, make_float2(kLift, kLift));
                            hi[h / 2] = ptx::pack_half2(lifted.x, lifted.y);
                            // 2^11 (2^7 p - hi), which is exact
                            const float2 rest = ptx::ffma2(__half22float2(*reinterpret_cast<const __half2*>(&hi[h / 2])),
                                                           make_float2(-kLowLift, -kLowLift),
                                                           ptx::fmul2(p, make_float2(kLift * kLowLift, kLift * kLowLift)));
                            lo[h / 2] = ptx::pack_half2(rest.x, rest.y);
                        }
                        uint8_t* p = smem + C::OFF_P + (buf * C::U + u) * C::P_BYTES + row * C::PROW;
                        const int sw = C::PROW == 32 ? (row >> 2) & 1 : (row >> 1) & 3;
                        auto put = [&](int column, const uint32_t (&v)[HC / 2]) {  // HC columns from `column` on
                            if constexpr (HC == 4) {
                                *reinterpret_cast<uint2*>(p + (((column / 8) ^ sw) * 16)) = make_uint2(v[0], v[1]);
                            } else {
#pragma unroll
                                for (int c = 0; c < HC / 8; c++)
                                    *reinterpret_cast<uint4*>(p + (((column / 8 + c) ^ sw) * 16)) =
                                        make_uint4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
                            }
                        };
                        put(0, hi);
                        put(C::NP / 2, lo);
                        const int keys = t.keys(i * C::U + u);
                        if (keys % 16 != 0 || keys == 0) {
                            // Keys behind the last, up to the end of its MMA step:
                            // whatever lies in their places of V (NaN included) must
                            // not meet their weights of zero.
                            ok = bounded_wait(&v_full[ring.s], ring.parity, w, kPagedVFull) && ok;
                            zero_keys<D, C::CB>(stages + ring.s * C::STAGE + C::K_BYTES, keys, max(16, (keys + 15) / 16 * 16), page, shift, row);
                        }
                        ring.next();
                    }
                    __syncwarp();
                    ptx::fence_proxy_async_smem();
                    if (!kWithhold || blockIdx.x > 0 || g > 0 || row > 0) ptx::mbar_arrive(&p_full[buf]);
                    g++;
                    j++;
                }
                if (i > 0) {
                    const int done = g - (i < n_steps ? 2 : 1), buf = done & 1;  // step i - 1
                    ok = bounded_wait(&o_full[buf], static_cast<uint32_t>(done / 2) & 1u, w, kPagedOFull) && ok;
                    __syncwarp();
                    ptx::tc_fence_after();
                    // (One M at a time: two of 16 heads at once spilled registers.)
#pragma unroll
                    for (int m = 0; m < C::MT; m++) {
                        uint32_t hi[HC], lo[HC];
                        load_cols(C::O_COL + (buf * C::MT + m) * C::NP, hi);
                        load_cols(C::O_COL + (buf * C::MT + m) * C::NP + C::NP / 2, lo);
                        ptx::tc_wait_ld();
                        if (m == C::MT - 1) {
                            ptx::tc_fence_before();
                            ptx::mbar_arrive(&o_free[buf]);
                        }
#pragma unroll
                        for (int h = 0; h < HC; h += 2) {
                            const float2 v = ptx::ffma2(make_float2(__uint_as_float(lo[h]), __uint_as_float(lo[h + 1])),
                                                        make_float2(1.f / kLowLift, 1.f / kLowLift),
                                                        make_float2(__uint_as_float(hi[h]), __uint_as_float(hi[h + 1])));
                            const float2 sum = ptx::ffma2(v, make_float2(beta[h], beta[h + 1]), make_float2(o[m][h], o[m][h + 1]));
                            o[m][h] = sum.x;
                            o[m][h + 1] = sum.y;
                        }
                    }
                }
            }
            if (out_of_time) break;
            // The item's end in this block.
#pragma unroll
            for (int c = 0; c < HC / 4; c++) {
                const float v[4] = {l[4 * c], l[4 * c + 1], l[4 * c + 2], l[4 * c + 3]};
                const float sum = warp_reduce4(v, lane, sum_of);
                if ((lane & 7) == 0) red_sum[wq * HC + 4 * c + (lane >> 3)] = sum;
            }
            ptx::named_bar_sync(bar_id, 128);
            const bool begun = t.tile == 0;  // the item's first tile is in the range
            const bool whole = begun && t.n == t.tiles;
            const int slot = 2 * blockIdx.x + (t.left < count ? 1 : 0);
            const int64_t o0 = static_cast<int64_t>(t.b) * a.q_heads + t.head * a.group + h0;
#pragma unroll
            for (int h = 0; h < HC; h++) {
                if (h >= nh) break;
                const float sum = (red_sum[h] + red_sum[HC + h]) + (red_sum[2 * HC + h] + red_sum[3 * HC + h]);
                if (whole) {
                    const float inv = sum > 0.f ? __fdividef(1.f / kLift, sum) : 0.f;
#pragma unroll
                    for (int m = 0; m < C::MT; m++)
                        if (m * 128 + row < D)
                            static_cast<OutT*>(a.out)[(o0 + h) * D + m * 128 + row] = from_float<OutT>(o[m][h] * inv);
                    if (a.lse && row == h)
                        a.lse[o0 + h] = sum > 0.f ? (__log2f(sum) - nm[h]) * 0.6931471805599453f : INFINITY;
                } else {
#pragma unroll
                    for (int m = 0; m < C::MT; m++)
                        if (m * 128 + row < D)
                            a.p.o[(static_cast<int64_t>(slot) * HC + h) * D + m * 128 + row] = o[m][h] * (1.f / kLift);
                    if (row == h) a.p.ml[slot * HC + h] = make_float2(-nm[h], sum);
                }
            }
            // What the join has to do for this block: the item begun here that goes on, to
            // the block of its last tile.
            if (row == 0 && t.left == t.n && begun && !whole)
                a.p.items[blockIdx.x] = make_int4(t.b, t.head * a.splits + t.split,
                                                  paged_block(range->total, range->first + count - t.n + t.tiles - 1, range->blocks), slot);
        }
    }

    ptx::tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem, C::TMEM_COLS);
    }
}

// Block (j, h): head h of the item that attention block j began and others
// continued: their partial results, in the blocks' order.  A chain of three
// loads from memory (what to join, the weights, the parts), so the parts are
// read by as many threads as there are: kRows of them at once, 16 bytes a
// thread, and added in shared memory.
template <typename OutT, int D, int HC>
__global__ void __launch_bounds__(256) paged_join_kernel(const __grid_constant__ PagedArgs a)
{
    constexpr int kRows = 256 / (D / 4) < 8 ? 256 / (D / 4) : 8;
    __shared__ float weight[kPagedBlocks];
    __shared__ float red[16];
    __shared__ float4 sums[kRows][D / 4];
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32, h = blockIdx.y;
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    const int4 it = a.p.items[blockIdx.x];
    if (it.x < 0) return;
    const int h0 = (it.y % a.splits) * a.heads_per_group;
    if (h >= min(a.heads_per_group, a.group - h0)) return;
    const int parts = it.z - blockIdx.x + 1;
    auto slot = [&](int p) { return p == 0 ? it.w : 2 * (static_cast<int>(blockIdx.x) + p); };
    // The first rows of parts are on their way while the weights are formed.
    const int r = tid / (D / 4), c = tid % (D / 4);
    auto part = [&](int p) {
        return reinterpret_cast<const float4*>(a.p.o + (static_cast<int64_t>(slot(p)) * HC + h) * D)[c];
    };
    float4 first = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r < kRows && r < parts) first = part(r);
    const float2 ml = tid < parts ? a.p.ml[slot(tid) * HC + h] : make_float2(-INFINITY, 0.f);  // parts <= 148
    const float wtop = ptx::warp_max(ml.x);
    if (lane == 0) red[warp] = wtop;
    __syncthreads();
    float top = red[0];
#pragma unroll
    for (int i = 1; i < 8; i++) top = fmaxf(top, red[i]);
    const float wgt = ptx::ex2_approx(ml.x - top);  // 0 for no part
    if (tid < parts) weight[tid] = wgt;
    float sum = wgt * ml.y;
#pragma unroll
    for (int i = 16; i; i >>= 1) sum += __shfl_xor_sync(~0u, sum, i);
    if (lane == 0) red[8 + warp] = sum;
    __syncthreads();
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) sum += red[8 + i];
    if (r < kRows) {
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int p = r; p < parts; p += kRows) {
            const float4 v = p == r ? first : part(p);
            const float k = weight[p];
            o.x = fmaf(k, v.x, o.x);
            o.y = fmaf(k, v.y, o.y);
            o.z = fmaf(k, v.z, o.z);
            o.w = fmaf(k, v.w, o.w);
        }
        sums[r][c] = o;
    }
    __syncthreads();
    const int64_t at = static_cast<int64_t>(it.x) * a.q_heads + (it.y / a.splits) * a.group + h0 + h;
    if (tid < D) {
        float o = 0.f;
#pragma unroll
        for (int i = 0; i < kRows; i++) o += reinterpret_cast<const float*>(sums[i])[tid];
        static_cast<OutT*>(a.out)[at * D + tid] = from_float<OutT>(__fdividef(o, sum));
    }
    if (a.lse && tid == 0) a.lse[at] = (top + __log2f(sum)) * 0.6931471805599453f;
}

}  // namespace fp4attn
