// paged.cuh -- the paged FP4 key / FP16 value cache (sm_100a): appending
// tokens (keys rotated and quantised on the way in), reading tokens back, and
// copying pages.
//
// One cache holds, per page and key/value head, page_size tokens:
//   k_codes  [pages][kv_heads][page_size][head_dim / 2]   two E2M1 codes a byte
//   k_scales [pages][kv_heads][page_size][head_dim / 32]  UE8M0 bytes
//   v        [pages][kv_heads][page_size][head_dim]       FP16
// in the row-major forms of fp4attn_quantize, except that a scale of 255
// (only ever with all-zero codes) is stored as 254, which the tensor core
// reads as a finite factor.
#pragma once

#include <cuda_fp16.h>
#include <cstdint>

#include "device_status.cuh"
#include "quantize.cuh"
#include "rotary.cuh"

namespace fp4attn {

struct CacheView {
    uint8_t* k_codes;
    uint8_t* k_scales;
    __half* v;
    int64_t k_codes_stride, k_scales_stride, v_stride;  // bytes from one page to the next
    int pages, page_size, page_shift, kv_heads, head_dim;
};

struct TableView {
    const int32_t* pages;  // [seqs][stride]
    int64_t stride;
    int seqs, max_pages;
};

// The page of a sequence's position, or -1 (recorded) when there is none.
__device__ __forceinline__ int page_of(const CacheView& c, const TableView& t, int seq, int pos)
{
    if (seq < 0 || seq >= t.seqs) {
        record_index_error(kIndexSequence, seq);
        return -1;
    }
    const int slot = pos >> c.page_shift;
    if (slot >= t.max_pages) {
        record_index_error(kIndexLength, pos);
        return -1;
    }
    const int page = t.pages[seq * t.stride + slot];
    if (page < 0 || page >= c.pages) {
        record_index_error(kIndexPage, page);
        return -1;
    }
    return page;
}

// Eight elements of a block of 32 whose scale byte is sb, encoded as
// encode32 of quantize.cuh does (see there for the ties).
template <typename T>
__device__ __forceinline__ uint32_t encode8(const float (&v)[8], uint32_t sb)
{
    const int s = static_cast<int>(sb) - 127;
    if (s == 128) return 0u;
    const float inv = exact_pow2_neg(s);
    float q[8];
    bool exact = false;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        q[i] = v[i] * inv;
        if constexpr (sizeof(T) == 2) {
            exact |= isnan(v[i]);
        } else {
            const uint32_t b = __float_as_uint(q[i]);
            exact |= ((b << 11) == 0u && b != 0u) || isnan(q[i]);
        }
    }
    if (exact) {
        uint32_t w = 0u;
#pragma unroll
        for (int i = 0; i < 8; i++) w |= encode_e2m1(q[i]) << (4 * i);
        return w;
    }
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < 8; i++) q[i] = __fmaf_rn(q[i], 1.0f + 0x1p-12f, 0.f);
    }
    return ptx::cvt_e2m1x8(q);
}

struct AppendArgs {
    const void *k, *v, *q;
    void* q_out;                       // [tokens][q_heads][head_dim], contiguous
    int64_t kt, kh, vt, vh, qt, qh;    // element strides of token and head
    int tokens, q_heads;
    CacheView c;
    TableView t;
    const int32_t* seq_ids;            // [tokens] or null: token i belongs to sequence i
    const int32_t* positions;          // [tokens]; negative: the token is padding
    const float2* table;               // rotary table or null
    int rot;
    int64_t max_positions;
    int interleaved, ocp;
};

// Quantises eight elements of a key (as a separate rotation would have left
// them) that share a block of 32 with those of the three neighbouring lanes,
// and stores their codes and the block's scale.  `place`: the head's token in
// its page.
template <typename T>
__device__ __forceinline__ void put_key(const CacheView& c, int page, int64_t place, int e0, float (&v)[8], int ocp)
{
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        v[i] = to_float(from_float<T>(v[i]));
        amax = fmaxf(amax, fabsf(v[i]));
    }
    const uint32_t quad = 0xFu << ((threadIdx.x & 31) & ~3);
    amax = fmaxf(amax, __shfl_xor_sync(quad, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(quad, amax, 2));
    const uint32_t sb = scale_byte(amax, ocp);
    *reinterpret_cast<uint32_t*>(c.k_codes + page * c.k_codes_stride + place * (c.head_dim / 2) + e0 / 2) = encode8<T>(v, sb);
    if (e0 % 32 == 0)
        c.k_scales[page * c.k_scales_stride + place * (c.head_dim / 32) + e0 / 32] = static_cast<uint8_t>(sb == 255u ? 254u : sb);
}

// Eight elements as they lie in memory, and as floats.
__device__ __forceinline__ void load_raw8(const __half* p, uint4 (&r)[1]) { r[0] = *reinterpret_cast<const uint4*>(p); }
__device__ __forceinline__ void load_raw8(const float* p, uint4 (&r)[2])
{
    r[0] = reinterpret_cast<const uint4*>(p)[0];
    r[1] = reinterpret_cast<const uint4*>(p)[1];
}

// A block has one token and a set of its heads.  A thread has eight elements
// of a row and (halves) the eight they are paired with, or eight interleaved
// ones, or eight that are not turned.  Bound by memory: a token's K, V and Q
// in, Q out, 17/32 + 2 bytes an element into the cache.  What there is to wait
// for -- the position, then the angles and the page -- is waited for while the
// row is on its way, once, and 32 registers leave room for all the warps that an
// SM holds: 17,600 tokens of 32 + 2 x 8 heads of 128 take 95 us, 0.67 of their
// 63 us at the copy rate.  (With 50 registers 114 us; with three heads a
// thread, their angles kept, and 78 registers 156; interleaved 101 us, with one
// eight a thread 137.)  Needs 16-byte aligned rows and, for halves, a rotary
// dimension of whole 64s, so that a block of 32 is four neighbouring lanes'.
constexpr int kAppendThreads = 128;

// Threads of a row: two eights each where that leaves whole blocks of 32 to four
// neighbouring lanes (interleaved: head dimensions of whole 64s).
__host__ __device__ inline int append_units(int head_dim, int rot, bool interleaved)
{
    if (interleaved) return head_dim % 64 == 0 ? head_dim / 16 : head_dim / 8;
    return rot / 16 + (head_dim - rot) / 8;
}

// Eight interleaved elements from e0 on, of which those below 2 * half are
// turned.  cs: the position's angles.
__device__ __forceinline__ void turn_interleaved(float (&v)[8], const float2* cs, int e0, int half)
{
    if (e0 >= 2 * half) return;
    cs += e0 / 2;
    if (half % 4 == 0) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const float4 f = reinterpret_cast<const float4*>(cs)[i];
            turn(v[4 * i], v[4 * i + 1], f.x, f.y, v[4 * i], v[4 * i + 1]);
            turn(v[4 * i + 2], v[4 * i + 3], f.z, f.w, v[4 * i + 2], v[4 * i + 3]);
        }
    } else {  // the last eight may be turned in part
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (e0 / 2 + i >= half) break;
            const float2 f = cs[i];
            turn(v[2 * i], v[2 * i + 1], f.x, f.y, v[2 * i], v[2 * i + 1]);
        }
    }
}

// kTwo: interleaved, two eights a thread (head dimensions of whole 64s).
template <typename T, bool kInter, bool kTwo>
__global__ void __launch_bounds__(kAppendThreads, kTwo ? 12 : 16) cache_append_kernel(const __grid_constant__ AppendArgs a)
{
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    const int D = a.c.head_dim, half = a.rot / 2, units = append_units(D, a.rot, kInter), at_once = kAppendThreads / units;
    const int second = kInter ? D / 2 : half, pairs = kInter ? D / 16 : half / 8;
    const int hs = threadIdx.x / units, u = threadIdx.x % units;
    const int tok = blockIdx.x, kv = a.c.kv_heads, h = blockIdx.y * at_once + hs;  // K, V, Q
    if (hs >= at_once || h >= 2 * kv + a.q_heads) return;
    const bool pair = (!kInter || kTwo) && u < pairs, is_v = h >= kv && h < 2 * kv, is_q = h >= 2 * kv;
    const int e0 = kInter || pair ? 8 * u : a.rot + 8 * (u - pairs);
    const T* x = (is_q   ? static_cast<const T*>(a.q) + tok * a.qt + (h - 2 * kv) * a.qh
                  : is_v ? static_cast<const T*>(a.v) + tok * a.vt + (h - kv) * a.vh
                         : static_cast<const T*>(a.k) + tok * a.kt + h * a.kh) + e0;
    uint4 ra[sizeof(T) / 2], rb[sizeof(T) / 2];
    load_raw8(x, ra);
    if (pair) load_raw8(x + second, rb);
    const int pos = a.positions[tok];
    const bool valid = pos >= 0 && (!a.rot || pos < a.max_positions);
    int page = -1;
    if (valid && !is_q) page = page_of(a.c, a.t, a.seq_ids ? a.seq_ids[tok] : tok, pos);
    if (!valid && pos >= 0 && u == 0 && h == 0) record_index_error(kIndexPosition, pos);
    if (!is_q && page < 0) return;
    const int64_t place = static_cast<int64_t>(is_v ? h - kv : h) * a.c.page_size + (pos & (a.c.page_size - 1));
    if (is_v) {
        __half* dst = reinterpret_cast<__half*>(reinterpret_cast<uint8_t*>(a.c.v) + page * a.c.v_stride) + place * D + e0;
        if constexpr (sizeof(T) == 2) {  // FP16 values keep their bits
            *reinterpret_cast<uint4*>(dst) = ra[0];
            if (pair) *reinterpret_cast<uint4*>(dst + second) = rb[0];
        } else {
            float v[8];
            load8v(reinterpret_cast<const T*>(ra), v);
            store8v(dst, v);
            if (pair) {
                load8v(reinterpret_cast<const T*>(rb), v);
                store8v(dst + second, v);
            }
        }
        return;
    }
    float v[8], w[8];
    load8v(reinterpret_cast<const T*>(ra), v);
    if (pair) load8v(reinterpret_cast<const T*>(rb), w);
    if (!valid) {  // padding, and angles that are not there: a row of zeros
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = w[i] = 0.f;
    } else if constexpr (kInter) {
        const float2* cs = a.table + static_cast<int64_t>(pos) * half;
        turn_interleaved(v, cs, e0, half);
        if (pair) turn_interleaved(w, cs, e0 + second, half);
    } else if (pair) {
        const float4* cs = reinterpret_cast<const float4*>(a.table + static_cast<int64_t>(pos) * half + e0);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float4 f = cs[i];
            turn(v[2 * i], w[2 * i], f.x, f.y, v[2 * i], w[2 * i]);
            turn(v[2 * i + 1], w[2 * i + 1], f.z, f.w, v[2 * i + 1], w[2 * i + 1]);
        }
    }
    if (is_q) {
        T* dst = static_cast<T*>(a.q_out) + (static_cast<int64_t>(tok) * a.q_heads + h - 2 * kv) * D + e0;
        store8v(dst, v);
        if (pair) store8v(dst + second, w);
    } else {
        put_key<T>(a.c, page, place, e0, v, a.ocp);
        if (pair) put_key<T>(a.c, page, place, e0 + second, w, a.ocp);
    }
}

// Aligned rows in halves that are not whole 32s (a rotary dimension of 50 or 96):
// a thread has eight elements of a row, and a block's keys and queries pass through
// shared memory, for the elements that they are paired with lie across eights and
// blocks.  The token's angles are laid out in shared memory, one for each element.
// The 17,600 tokens above with 50 of 128 elements turned: 164 us (the angles from
// the table by each thread: 216; element by element, as below: 260).
template <typename T>
__global__ void __launch_bounds__(kAppendThreads) cache_append_rows_kernel(const __grid_constant__ AppendArgs a)
{
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    __shared__ __align__(16) T rows[kAppendThreads * 8];
    __shared__ __align__(16) float2 angles[256];  // of every element, the sine signed as its own sum needs it
    const int D = a.c.head_dim, half = a.rot / 2, units = D / 8, at_once = kAppendThreads / units;
    const int hs = threadIdx.x / units, e0 = threadIdx.x % units * 8;
    const int tok = blockIdx.x, kv = a.c.kv_heads, h = blockIdx.y * at_once + hs;  // K, V, Q
    const bool mine = hs < at_once && h < 2 * kv + a.q_heads;
    const bool is_v = h >= kv && h < 2 * kv, is_q = h >= 2 * kv;
    T* row = rows + hs * D;
    const int pos = a.positions[tok];
    const bool valid = pos >= 0 && pos < a.max_positions;
    uint4 raw[sizeof(T) / 2];
    if (mine) {
        const T* x = (is_q   ? static_cast<const T*>(a.q) + tok * a.qt + (h - 2 * kv) * a.qh
                      : is_v ? static_cast<const T*>(a.v) + tok * a.vt + (h - kv) * a.vh
                             : static_cast<const T*>(a.k) + tok * a.kt + h * a.kh) + e0;
        load_raw8(x, raw);
    }
    if (valid)
        for (int e = threadIdx.x; e < a.rot; e += kAppendThreads) {
            const float2 f = a.table[static_cast<int64_t>(pos) * half + (e < half ? e : e - half)];
            angles[e] = make_float2(f.x, e < half ? -f.y : f.y);
        }
    if (mine) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; i++) reinterpret_cast<uint4*>(row + e0)[i] = raw[i];
    }
    __syncthreads();
    if (!mine) return;
    int page = -1;
    if (valid && !is_q) page = page_of(a.c, a.t, a.seq_ids ? a.seq_ids[tok] : tok, pos);
    if (!valid && pos >= 0 && e0 == 0 && h == 0) record_index_error(kIndexPosition, pos);
    if (!is_q && page < 0) return;
    const int64_t place = static_cast<int64_t>(is_v ? h - kv : h) * a.c.page_size + (pos & (a.c.page_size - 1));
    float v[8];
    load8v(reinterpret_cast<const T*>(raw), v);
    if (is_v) {
        __half* dst = reinterpret_cast<__half*>(reinterpret_cast<uint8_t*>(a.c.v) + page * a.c.v_stride) + place * D + e0;
        if constexpr (sizeof(T) == 2) *reinterpret_cast<uint4*>(dst) = raw[0];  // FP16 values keep their bits
        else store8v(dst, v);
        return;
    }
    if (!valid) {  // padding, and angles that are not there: a row of zeros
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = 0.f;
    } else if (e0 < a.rot) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int e = e0 + i;
            if (e >= a.rot) break;
            const float2 f = angles[e];
            const float other = to_float(row[e < half ? e + half : e - half]);
            v[i] = __fadd_rn(__fmul_rn(v[i], f.x), __fmul_rn(other, f.y));  // (turn()'s bits)
        }
    }
    if (is_q) store8v(static_cast<T*>(a.q_out) + (static_cast<int64_t>(tok) * a.q_heads + h - 2 * kv) * D + e0, v);
    else put_key<T>(a.c, page, place, e0, v, a.ocp);
}

// Eight elements e0 .. e0 + 7 of a row, rotated one by one (FP32, not yet
// rounded).
template <typename T>
__device__ __forceinline__ void rotated8(const T* row, int e0, const float2* cs, int rot, int interleaved, float (&v)[8])
{
    const int half = rot / 2;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int e = e0 + i;
        if (e >= rot) {
            v[i] = to_float(row[e]);
            continue;
        }
        const int j = interleaved ? e / 2 : (e < half ? e : e - half);
        const int ia = interleaved ? 2 * j : j, ib = interleaved ? 2 * j + 1 : j + half;
        float ra, rb;
        turn(to_float(row[ia]), to_float(row[ib]), cs[j].x, cs[j].y, ra, rb);
        v[i] = e == ia ? ra : rb;
    }
}

// Rows that are not 16-byte aligned: one thread per eight elements of
// a token's K, V or Q, four neighbouring lanes to a block of 32, every element
// loaded by itself.
template <typename T>
__global__ void __launch_bounds__(256) cache_append_any_kernel(const __grid_constant__ AppendArgs a)
{
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    const int D = a.c.head_dim, row8 = D / 8;
    const int kv_units = a.c.kv_heads * row8, units = 2 * kv_units + a.q_heads * row8;
    const int64_t n = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (n >= static_cast<int64_t>(a.tokens) * units) return;
    const int tok = static_cast<int>(n / units);
    int u = static_cast<int>(n % units);
    const int pos = a.positions[tok];
    const bool is_q = u >= 2 * kv_units;
    const bool is_v = !is_q && u >= kv_units;
    u -= is_q ? 2 * kv_units : is_v ? kv_units : 0;
    const int head = u / row8, e0 = (u % row8) * 8;
    const bool valid = pos >= 0 && (!a.rot || pos < a.max_positions);
    if (pos >= 0 && !valid) record_index_error(kIndexPosition, pos);
    const float2* cs = a.rot ? a.table + (valid ? pos : 0) * static_cast<int64_t>(a.rot / 2) : nullptr;
    float v[8];
    if (is_q) {
        rotated8(static_cast<const T*>(a.q) + tok * a.qt + head * a.qh, e0, cs, a.rot, a.interleaved, v);
        if (!valid) {  // padding, and angles that are not there: a row of zeros
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = 0.f;
        }
        store8v(static_cast<T*>(a.q_out) + (static_cast<int64_t>(tok) * a.q_heads + head) * D + e0, v);
        return;
    }
    if (!valid) return;
    const int page = page_of(a.c, a.t, a.seq_ids ? a.seq_ids[tok] : tok, pos);
    if (page < 0) return;
    const int64_t place = static_cast<int64_t>(head) * a.c.page_size + (pos & (a.c.page_size - 1));
    if (is_v) {
        const T* row = static_cast<const T*>(a.v) + tok * a.vt + head * a.vh + e0;
        __half* dst = reinterpret_cast<__half*>(reinterpret_cast<uint8_t*>(a.c.v) + page * a.c.v_stride) + place * D + e0;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            if constexpr (sizeof(T) == 2) dst[i] = row[i];
            else dst[i] = __float2half_rn(row[i]);
        }
        return;
    }
    rotated8(static_cast<const T*>(a.k) + tok * a.kt + head * a.kh, e0, cs, a.rot, a.interleaved, v);
    put_key<T>(a.c, page, place, e0, v, a.ocp);
}

// Exactly 2^(sb - 127).
__device__ __forceinline__ float scale_value(uint32_t sb)
{
    return sb ? __uint_as_float(sb << 23) : __uint_as_float(1u << 22);
}

// The value of E2M1 code n (sign in bit 3), unscaled.
__device__ __forceinline__ float e2m1_value(uint32_t n)
{
    // Twice the magnitudes 0, 1, 2, 3, 4, 6, 8, 12 of bits 0-2, a nibble each.
    const float m = static_cast<float>((0xC8643210u >> (4u * (n & 7u))) & 15u) * 0.5f;
    return n & 8u ? -m : m;
}

struct GatherArgs {
    CacheView c;
    TableView t;
    const int32_t *starts, *lengths;  // [seqs]; starts may be null (0)
    int max_length, repeat;           // every key/value head is written `repeat` times
    void *k, *v;                      // [seqs][kv_heads * repeat][max_length][head_dim]
};

// Thread: eight elements of the K and V of kGatherRows tokens of one head, the
// block's rows apart, all of them loaded before the first is stored.  Rows past
// a sequence's length are written as zeros.  Bound by memory, most of it the
// writes: 8 sequences of 300 to 4096 tokens, 8 heads of 128, padded to 4096 rows of FP16, in 36 us,
// 0.78 of the copy rate (one row a thread, the page looked up for each: 49).
constexpr int kGatherRows = 4;

template <typename T, int D>
__global__ void __launch_bounds__(256) cache_gather_kernel(const __grid_constant__ GatherArgs a)
{
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    constexpr int ROW8 = D / 8, ROWS = 256 / ROW8;  // rows of a block at once
    const int tid = threadIdx.x, e0 = tid % ROW8 * 8, r = tid / ROW8;
    if (r >= ROWS) return;
    const int head = blockIdx.y, seq = blockIdx.z;
    const int start = a.starts ? a.starts[seq] : 0;
    int length = a.lengths[seq];
    if (start < 0 || length < 0 || length > a.max_length) {
        if (blockIdx.x == 0 && head == 0 && tid == 0) record_index_error(kIndexLength, start < 0 ? start : length);
        length = 0;
    }
    uint32_t code[kGatherRows];
    float scale[kGatherRows];
    uint4 value[kGatherRows];
#pragma unroll
    for (int k = 0; k < kGatherRows; k++) {
        const int i = (blockIdx.x * kGatherRows + k) * ROWS + r;
        code[k] = 0u;
        scale[k] = 0.f;
        value[k] = make_uint4(0u, 0u, 0u, 0u);
        if (i >= length) continue;
        const int64_t pos = static_cast<int64_t>(start) + i;
        if (pos > 0x7FFFFFFF) {
            record_index_error(kIndexLength, pos);
            continue;
        }
        const int page = page_of(a.c, a.t, seq, static_cast<int>(pos));
        if (page < 0) continue;
        const int64_t in_page = static_cast<int64_t>(head) * a.c.page_size + (pos & (a.c.page_size - 1));
        code[k] = *reinterpret_cast<const uint32_t*>(a.c.k_codes + page * a.c.k_codes_stride + in_page * (D / 2) + e0 / 2);
        scale[k] = scale_value(a.c.k_scales[page * a.c.k_scales_stride + in_page * (D / 32) + e0 / 32]);
        value[k] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(a.c.v) + page * a.c.v_stride +
                                                   (in_page * D + e0) * 2);
    }
#pragma unroll
    for (int k = 0; k < kGatherRows; k++) {
        const int i = (blockIdx.x * kGatherRows + k) * ROWS + r;
        if (i >= a.max_length) return;
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = e2m1_value((code[k] >> (4 * j)) & 15u) * scale[k];
        for (int q = 0; q < a.repeat; q++) {
            const int64_t at = ((static_cast<int64_t>(seq) * a.c.kv_heads + head) * a.repeat + q) * a.max_length + i;
            store8v(static_cast<T*>(a.k) + at * D + e0, x);
            T* v = static_cast<T*>(a.v) + at * D + e0;
            if constexpr (sizeof(T) == 2) {
                *reinterpret_cast<uint4*>(v) = value[k];
            } else {
                float f[8];
                load8v(reinterpret_cast<const __half*>(&value[k]), f);
                store8v(v, f);
            }
        }
    }
}

// ---------------------------------------------------------------- page copies
constexpr int kCopyChunk = 16384;  // bytes a block copies: 256 threads, four 16-byte words each

struct CopyArray {
    uint8_t* base;
    int64_t page_stride;
    int page_bytes;
    int first_chunk;  // chunks of the arrays before this one
};

// The arrays and page pairs of one launch, by value: the pairs are the host's
// and are checked there, and a captured launch carries them with it.
template <int kArrays, int kPairs>
struct CopyArgs {
    CopyArray arrays[kArrays];
    int2 pairs[kPairs];  // source, destination
    int n_arrays;
};

// Block (x, y): chunk x of pair y.  1500 pages of 64 tokens, 8 heads of 128
// (249 MB in, 249 MB out) take 78 us, 0.99 of the copy rate.
template <int kArrays, int kPairs>
__global__ void __launch_bounds__(256) copy_pages_kernel(const __grid_constant__ CopyArgs<kArrays, kPairs> a)
{
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    int i = 0;
    while (i + 1 < a.n_arrays && a.arrays[i + 1].first_chunk <= static_cast<int>(blockIdx.x)) i++;
    const CopyArray& ar = a.arrays[i];
    const int2 p = a.pairs[blockIdx.y];
    const uint4* src = reinterpret_cast<const uint4*>(ar.base + p.x * ar.page_stride);
    uint4* dst = reinterpret_cast<uint4*>(ar.base + p.y * ar.page_stride);
    const int words = ar.page_bytes / 16;
    const int w0 = (static_cast<int>(blockIdx.x) - ar.first_chunk) * (kCopyChunk / 16) + threadIdx.x;
    uint4 v[4];
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (w0 + 256 * j < words) v[j] = src[w0 + 256 * j];
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (w0 + 256 * j < words) dst[w0 + 256 * j] = v[j];
}

}  // namespace fp4attn
