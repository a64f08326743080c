// rotary.cuh -- rotary positions (sm_100a): the table of cosines and sines,
// and the rotation of a [batch, heads, seq, head_dim] tensor.
//
// Pair j of a row at position p is turned by the angle p * freq[j]:
//     (a, b) -> (a cos - b sin, a sin + b cos),
// pairs (2j, 2j + 1) (interleaved) or (j, j + r/2) (halves) of the first r
// elements; the rest of the row is copied.  The rotation is orthogonal up to
// the table's factor, so its gradient is the same with sin negated.
// The products and the sum are rounded one by one (no fused multiply-add), so
// that the same expression in any FP32 arithmetic gives the same bits, and
// the result once to the tensor's type.
#pragma once

#include <cuda_fp16.h>
#include <cstdint>

#include "device_status.cuh"

namespace fp4attn {

__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(float v) { return v; }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }

// a cos - b sin and a sin + b cos, each operation rounded.
__device__ __forceinline__ void turn(float a, float b, float c, float s, float& ra, float& rb)
{
    ra = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
    rb = __fadd_rn(__fmul_rn(a, s), __fmul_rn(b, c));
}

// Eight consecutive elements, 16-byte aligned.
__device__ __forceinline__ void load8v(const __half* p, float (&v)[8])
{
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const __half2* h = reinterpret_cast<const __half2*>(&u);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = __half22float2(h[i]);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void load8v(const float* p, float (&v)[8])
{
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void store8v(__half* p, const float (&v)[8])
{
    uint4 u;
    __half2* h = reinterpret_cast<__half2*>(&u);
#pragma unroll
    for (int i = 0; i < 4; i++) h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = u;
}
__device__ __forceinline__ void store8v(float* p, const float (&v)[8])
{
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}

// Frequencies of one table, by value (head_dim <= 256: at most 128 pairs).
struct RotaryFreqs {
    double f[128];
};

// table[p][j] = factor * (cos, sin)(p * freq[j]).  The angle is formed and
// reduced in 64 bits: at position 10^6 a 32-bit angle is off by 0.03 radians.
// Bound by the FP64 sine and cosine; made once per model, not per call.
__global__ void __launch_bounds__(256) rotary_table_kernel(const RotaryFreqs freqs, int pairs, int64_t positions,
                                                           double factor, float2* __restrict__ table)
{
    const int64_t total = positions * pairs;
    for (int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; i < total;
         i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
        double s, c;
        sincos(static_cast<double>(i / pairs) * freqs.f[i % pairs], &s, &c);
        table[i] = make_float2(static_cast<float>(factor * c), static_cast<float>(factor * s));
    }
}

struct RotaryArgs {
    const void* x;
    void* y;
    int64_t xb, xh, xs, yb, yh, ys;  // element strides of batch, head and position
    int heads, seq, head_dim, rot;
    const float2* table;             // [max_positions][rot / 2]
    const int32_t* positions;        // [batch][seq] or null: 0 .. seq - 1
    int64_t pos_stride;              // elements from a batch entry's positions to the next
    int64_t max_positions;
    float sign;                      // -1: the gradient's rotation
    int heads_per_thread;
};

// A thread owns a piece of a row at one position -- kVec (rows of 16-byte
// alignment): eight elements of each half of the rotated part (halves of whole
// eights), or eight interleaved ones, or eight of the rest; otherwise one pair
// or one element -- loads its cosines and sines
// once, and walks `heads_per_thread` heads.  One read and one write of x.
// Bound by memory; many warps with one head in flight each do better than
// fewer with two or four (8 x 32 x 4096 x 128 FP16, four heads a thread: 86 us,
// 0.96 of the measured copy rate, against 98 and 100; eight heads: 88).
template <typename T, bool kVec, bool kInter>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryArgs a)
{
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    constexpr int E = kVec ? 8 : 1;
    const int half = a.rot / 2;
    const int turned = kVec ? (kInter ? (a.rot + 7) / 8 : half / 8) : half;
    const int rest = kVec && kInter ? 8 * turned : a.rot;  // what is not turned, from here on
    const int units = turned + (a.head_dim - rest) / E;
    const int t = blockIdx.x * blockDim.x + threadIdx.x;
    if (t >= a.seq * units) return;
    const int s = t / units, u = t % units;
    const int64_t b = blockIdx.z;
    const int h0 = blockIdx.y * a.heads_per_thread, h1 = min(a.heads, h0 + a.heads_per_thread);
    const T* x = static_cast<const T*>(a.x) + b * a.xb + s * a.xs;
    T* y = static_cast<T*>(a.y) + b * a.yb + s * a.ys;
    const int64_t pos = a.positions ? a.positions[b * a.pos_stride + s] : s;
    const bool ok = pos >= 0 && pos < a.max_positions;
    if (!ok && u == 0 && h0 == 0) record_index_error(kIndexPosition, pos);
    if (u >= turned) {  // the part that is not rotated
        const int e = rest + (u - turned) * E;
        for (int h = h0; h < h1; h++) {
            if constexpr (kVec) {
                float v[8];
                load8v(x + h * a.xh + e, v);
                if (!ok)
                    for (int i = 0; i < 8; i++) v[i] = 0.f;
                store8v(y + h * a.yh + e, v);
            } else {
                y[h * a.yh + e] = ok ? x[h * a.xh + e] : from_float<T>(0.f);
            }
        }
        return;
    }
    constexpr int P = kVec ? (kInter ? 4 : 8) : 1;  // pairs of this thread
    const int pairs = kVec && kInter ? min(P, half - u * P) : P;  // (a last eight may be turned in part)
    float2 cs[P];
    {
        const float2* row = a.table + (ok ? pos : 0) * half + u * P;
        if (kVec && kInter && half % 4 != 0) {
#pragma unroll
            for (int i = 0; i < P; i++) {
                cs[i] = i < pairs ? row[i] : make_float2(0.f, 0.f);
                cs[i].y *= a.sign;
            }
        } else if constexpr (kVec) {
#pragma unroll
            for (int i = 0; i < P; i += 2) {
                const float4 f = *reinterpret_cast<const float4*>(row + i);
                cs[i] = make_float2(f.x, a.sign * f.y);
                cs[i + 1] = make_float2(f.z, a.sign * f.w);
            }
        } else {
            cs[0] = row[0];
            cs[0].y *= a.sign;
        }
        if (!ok)
            for (int i = 0; i < P; i++) cs[i] = make_float2(0.f, 0.f);
    }
#pragma unroll 1
    for (int h = h0; h < h1; h++) {
        const T* xr = x + h * a.xh;
        T* yr = y + h * a.yh;
        if constexpr (!kVec) {
            const int ia = kInter ? 2 * u : u, ib = kInter ? 2 * u + 1 : u + half;
            float ra, rb;
            turn(to_float(xr[ia]), to_float(xr[ib]), cs[0].x, cs[0].y, ra, rb);
            yr[ia] = from_float<T>(ok ? ra : 0.f);
            yr[ib] = from_float<T>(ok ? rb : 0.f);
        } else if constexpr (kInter) {
            float v[8];
            load8v(xr + 8 * u, v);
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (i < pairs) turn(v[2 * i], v[2 * i + 1], cs[i].x, cs[i].y, v[2 * i], v[2 * i + 1]);
            if (!ok)
                for (int i = 0; i < 8; i++) v[i] = 0.f;
            store8v(yr + 8 * u, v);
        } else {
            float va[8], vb[8];
            load8v(xr + 8 * u, va);
            load8v(xr + half + 8 * u, vb);
#pragma unroll
            for (int i = 0; i < 8; i++) turn(va[i], vb[i], cs[i].x, cs[i].y, va[i], vb[i]);
            if (!ok)
                for (int i = 0; i < 8; i++) va[i] = vb[i] = 0.f;
            store8v(yr + 8 * u, va);
            store8v(yr + half + 8 * u, vb);
        }
    }
}

// Halves that are not whole eights: a thread has eight elements of a row, which
// the block passes around through shared memory, for the elements that they are
// paired with lie across eights.  (The block has whole rows, so y may be x.)
// 2 x 18 x 11394 x 128 FP16 with 50 elements turned: 71 us, 0.46 of the copy rate,
// for the eight 2-byte reads from shared memory (a pair a thread from memory: 146).
template <typename T>
__global__ void __launch_bounds__(256) rotary_rows_kernel(const RotaryArgs a)
{
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    __shared__ __align__(16) T rows[2][256 * 8];
    const int D = a.head_dim, half = a.rot / 2, units = D / 8, at_once = 256 / units;
    const int r = threadIdx.x / units, e0 = threadIdx.x % units * 8;
    const int s = blockIdx.x * at_once + r;
    const bool mine = r < at_once && s < a.seq;
    const int64_t b = blockIdx.z;
    const int h0 = blockIdx.y * a.heads_per_thread, h1 = min(a.heads, h0 + a.heads_per_thread);
    const int64_t pos = !mine ? 0 : a.positions ? a.positions[b * a.pos_stride + s] : s;
    const bool ok = pos >= 0 && pos < a.max_positions;
    if (!ok && e0 == 0 && h0 == 0) record_index_error(kIndexPosition, pos);
    float2 cs[8];
    const float2* angles = a.table + (ok ? pos : 0) * half;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int e = e0 + i;
        cs[i] = e < a.rot ? angles[e < half ? e : e - half] : make_float2(1.f, 0.f);
        cs[i].y *= e < half ? -a.sign : a.sign;  // as the element's own sum needs it
    }
    for (int h = h0; h < h1; h++) {
        T* row = rows[(h - h0) & 1] + r * D;
        float v[8];
        if (mine) {
            load8v(static_cast<const T*>(a.x) + b * a.xb + h * a.xh + s * a.xs + e0, v);
            store8v(row + e0, v);
        }
        __syncthreads();
        if (!mine) continue;
        if (e0 < a.rot) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int e = e0 + i;
                if (e >= a.rot) break;
                const float other = to_float(row[e < half ? e + half : e - half]);
                v[i] = __fadd_rn(__fmul_rn(v[i], cs[i].x), __fmul_rn(other, cs[i].y));  // (turn()'s bits)
            }
        }
        if (!ok)
            for (int i = 0; i < 8; i++) v[i] = 0.f;
        store8v(static_cast<T*>(a.y) + b * a.yb + h * a.yh + s * a.ys + e0, v);
    }
}

}  // namespace fp4attn
