// paged.cu -- the serving half of the C ABI (declared in include/fp4attn.h):
// rotary positions, the paged cache and the attention over it.
#include <cuda.h>
#include <cuda_runtime.h>

#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <mutex>
#include <new>
#include <type_traits>
#include <utility>
#include <vector>

#include "../../include/fp4attn.h"
#include "paged.cuh"
#include "paged_attention.cuh"
#include "rotary.cuh"

namespace fp4attn {
unsigned long long current_context_id();  // fp4attn.cu
namespace host {  // fp4attn.cu
int error(int code, const char* msg);
void clear_error();
int ready();
int sms();
unsigned long long timeout_ns();
bool pdl();

// The serving kernels' error word, read and cleared (for fp4attn_status_query).
int serving_status()
{
    int w[4] = {0, 0, 0, 0};
    cudaError_t e = cudaMemcpyFromSymbol(w, g_serving_error, sizeof w);
    if (e != cudaSuccess) return error(FP4ATTN_ECUDA, cudaGetErrorString(e));
    if (w[0] == 0) return FP4ATTN_OK;
    const int zero[4] = {0, 0, 0, 0};
    e = cudaMemcpyToSymbol(g_serving_error, zero, sizeof zero);
    if (e != cudaSuccess) return error(FP4ATTN_ECUDA, cudaGetErrorString(e));
    char buf[160];
    if (w[0] == FP4ATTN_EINDEX) {
        static const char* const kinds[] = {"index", "position", "page", "sequence", "length or position"};
        const long long value = (static_cast<long long>(w[3]) << 32) | static_cast<unsigned>(w[2]);
        snprintf(buf, sizeof buf, "%s %lld out of range", kinds[w[1] >= 1 && w[1] <= 4 ? w[1] : 0], value);
    } else {
        snprintf(buf, sizeof buf, "device wait expired at serving site %d (block %d)", w[1], w[2]);
    }
    return error(w[0], buf);
}
}  // namespace host
}  // namespace fp4attn

namespace {

using namespace fp4attn;

int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int fail(int code, const char* fmt, ...)
{
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    return host::error(code, buf);
}

#define PAGED_CUDA(call)                                                                            \
    do {                                                                                            \
        cudaError_t e_ = (call);                                                                    \
        if (e_ != cudaSuccess) return fail(FP4ATTN_ECUDA, "%s: %s", #call, cudaGetErrorString(e_)); \
    } while (0)

bool aligned(const void* p, int n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
bool bad_dtype(int t) { return t != FP4ATTN_F32 && t != FP4ATTN_F16; }
int bytes_of(int dtype) { return dtype == FP4ATTN_F16 ? 2 : 4; }
bool supported_dim(int d) { return d == 32 || d == 64 || d == 96 || d == 128 || d == 160 || d == 256; }

int check_cache(const fp4attn_cache* c)
{
    if (!c || !c->k_codes || !c->k_scales || !c->v) return fail(FP4ATTN_EINVAL, "null cache pointer");
    if (!supported_dim(c->head_dim))
        return fail(FP4ATTN_EUNSUPPORTED, "head_dim %d is not one of 32/64/96/128/160/256", c->head_dim);
    if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128)
        return fail(FP4ATTN_EUNSUPPORTED, "page_size %d is not one of 16/32/64/128", c->page_size);
    if (c->pages < 1 || c->kv_heads < 1 || c->kv_heads > 65535)
        return fail(FP4ATTN_EINVAL, "pages %d >= 1, kv_heads %d in [1, 65535]", c->pages, c->kv_heads);
    const int64_t rows = static_cast<int64_t>(c->kv_heads) * c->page_size;
    if (rows * c->head_dim * 2 > 0x7FFFFFFF) return fail(FP4ATTN_EINVAL, "a page of 2 GiB or more");
    if (c->k_codes_stride < rows * c->head_dim / 2 || c->k_scales_stride < rows * c->head_dim / 32 ||
        c->v_stride < rows * c->head_dim * 2)
        return fail(FP4ATTN_EINVAL, "page strides smaller than a page");
    if (!aligned(c->k_codes, 16) || !aligned(c->k_scales, 16) || !aligned(c->v, 16) ||
        ((c->k_codes_stride | c->k_scales_stride | c->v_stride) & 15))
        return fail(FP4ATTN_EINVAL, "cache pointers and page strides must be multiples of 16 bytes");
    return FP4ATTN_OK;
}

int check_table(const int32_t* block_table, int64_t stride, int seqs, int max_pages)
{
    if (!block_table && seqs != 0) return fail(FP4ATTN_EINVAL, "null block table");
    if (seqs < 0 || max_pages < 1 || stride < 0 || (seqs > 1 && stride < max_pages))
        return fail(FP4ATTN_EINVAL, "block table of %d sequences, %d pages, stride %lld", seqs, max_pages,
                    static_cast<long long>(stride));
    return FP4ATTN_OK;
}

CacheView view_of(const fp4attn_cache& c)
{
    CacheView v{c.k_codes, c.k_scales, static_cast<__half*>(c.v), c.k_codes_stride, c.k_scales_stride, c.v_stride,
                c.pages, c.page_size, 0, c.kv_heads, c.head_dim};
    while ((1 << v.page_shift) < c.page_size) v.page_shift++;
    return v;
}

int check_rotary(const float* table, int rotary_dim, int64_t max_positions, int head_dim)
{
    if (!table || !aligned(table, 16)) return fail(FP4ATTN_EINVAL, "the rotary table must be a 16-byte aligned pointer");
    if (rotary_dim < 2 || rotary_dim % 2 || rotary_dim > head_dim)
        return fail(FP4ATTN_EINVAL, "rotary_dim %d must be even, in [2, head_dim %d]", rotary_dim, head_dim);
    if (max_positions < 1) return fail(FP4ATTN_EINVAL, "max_positions must be >= 1");
    return FP4ATTN_OK;
}

// f(std::integral_constant<int, head_dim>) for a supported head_dim.
template <typename F>
void with_dim(int d, F f)
{
    switch (d) {
        case 32: f(std::integral_constant<int, 32>{}); break;
        case 64: f(std::integral_constant<int, 64>{}); break;
        case 96: f(std::integral_constant<int, 96>{}); break;
        case 128: f(std::integral_constant<int, 128>{}); break;
        case 160: f(std::integral_constant<int, 160>{}); break;
        default: f(std::integral_constant<int, 256>{}); break;
    }
}

// Whether rows at these strides take 16-byte accesses.
bool wide(const void* p, int dtype, std::initializer_list<int64_t> strides)
{
    const int e = 16 / bytes_of(dtype);
    if (!aligned(p, 16)) return false;
    for (int64_t s : strides)
        if (s % e) return false;
    return true;
}

// Launches a kernel as the programmatic dependent of whatever precedes it in
// the stream: a step of serving is a chain of kernels of a few microseconds,
// each of which comes up while the one before drains and waits for its
// completion (griddepcontrol.wait) before it touches memory.
template <typename... KArgs, typename... Args>
int launch_after(void (*kern)(KArgs...), dim3 grid, unsigned block, size_t smem, cudaStream_t st, Args&&... args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = host::pdl() ? 1 : 0;
    PAGED_CUDA(cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...));
    return FP4ATTN_OK;
}

template <typename T>
int launch_rotary(dim3 grid, cudaStream_t st, const RotaryArgs& a, bool vec, bool inter)
{
    if (vec) return launch_after(inter ? rotary_kernel<T, true, true> : rotary_kernel<T, true, false>, grid, 256, 0, st, a);
    return launch_after(inter ? rotary_kernel<T, false, true> : rotary_kernel<T, false, false>, grid, 256, 0, st, a);
}

template <typename T>
int launch_append(dim3 grid, cudaStream_t st, const AppendArgs& a)
{
    auto kern = !a.interleaved               ? cache_append_kernel<T, false, false>
                : a.c.head_dim % 64 == 0 ? cache_append_kernel<T, true, true>
                                         : cache_append_kernel<T, true, false>;
    return launch_after(kern, grid, kAppendThreads, 0, st, a);
}

template <typename T>
int launch_gather(dim3 grid, cudaStream_t st, const GatherArgs& a)
{
    int rc = FP4ATTN_OK;
    with_dim(a.c.head_dim, [&](auto d) { rc = launch_after(cache_gather_kernel<T, d.value>, grid, 256, 0, st, a); });
    return rc;
}

PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder()
{
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    });
    return fn;
}

int encode_map(CUtensorMap* m, CUtensorMapDataType type, int rank, const void* base, const cuuint64_t* dims,
               const cuuint64_t* strides, const cuuint32_t* box, int swizzle_bytes)
{
    auto enc = tensor_map_encoder();
    if (!enc) return fail(FP4ATTN_ECUDA, "cuTensorMapEncodeTiled unavailable");
    const cuuint32_t ones[5] = {1, 1, 1, 1, 1};
    const CUtensorMapSwizzle sw = swizzle_bytes == 128  ? CU_TENSOR_MAP_SWIZZLE_128B
                                  : swizzle_bytes == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                                        : CU_TENSOR_MAP_SWIZZLE_32B;
    const CUresult r = enc(m, type, rank, const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           sw, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? FP4ATTN_OK : fail(FP4ATTN_ECUDA, "cuTensorMapEncodeTiled failed (%d)", static_cast<int>(r));
}

// Query heads of a group computed at once.  A larger group is split, and its
// keys and values are read again, from L2: for 32 sequences of 1000 to 8000
// tokens, 8 x 32 query heads of 128, two groups of 16 take 129 us; 32 heads at
// once, which spilled registers, took 144 when two groups took 131.
int heads_at_once(int group) { return group <= 4 ? 4 : group <= 8 ? 8 : 16; }

struct AttentionWorkspace {
    size_t items, ml, o, total;
};

AttentionWorkspace attention_workspace(int group, int head_dim)
{
    const size_t rows = static_cast<size_t>(2 * kPagedBlocks) * heads_at_once(group);
    AttentionWorkspace w{};
    w.ml = (kPagedBlocks * sizeof(int4) + 255) / 256 * 256;
    w.o = w.ml + rows * sizeof(float2);
    w.total = w.o + rows * head_dim * sizeof(float);
    return w;
}

template <typename OutT, int D, int HC, bool kWithhold = false>
int launch_attention(const PagedArgs& a, int blocks, bool join, cudaStream_t st)
{
    using C = PagedCfg<D, HC>;
    auto kern = paged_attention_kernel<OutT, D, HC, kWithhold>;
    // The shared memory limit is an attribute of the kernel in a context.
    static std::atomic<unsigned long long> done[64];
    int dev = 0;
    PAGED_CUDA(cudaGetDevice(&dev));
    const unsigned long long ctx = current_context_id();
    if (dev < 0 || dev >= 64) return fail(FP4ATTN_EUNSUPPORTED, "device index %d", dev);
    if (ctx == 0 || done[dev].load(std::memory_order_acquire) != ctx) {
        PAGED_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM_BYTES));
        done[dev].store(ctx, std::memory_order_release);
    }
    const CacheView& c = a.c;
    CUtensorMap tk, tv;
    {
        const cuuint64_t row = D / 2;
        const cuuint64_t dims[4] = {row, static_cast<cuuint64_t>(c.page_size), static_cast<cuuint64_t>(c.kv_heads),
                                    static_cast<cuuint64_t>(c.pages)};
        const cuuint64_t strides[3] = {row, row * c.page_size, static_cast<cuuint64_t>(c.k_codes_stride)};
        const cuuint32_t box[4] = {C::KROW, static_cast<cuuint32_t>(c.page_size), 1, 1};
        if (int rc = encode_map(&tk, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, c.k_codes, dims, strides, box, C::KROW)) return rc;
    }
    {
        const cuuint64_t row = D * 2;
        const cuuint64_t dims[5] = {C::CHE, static_cast<cuuint64_t>(c.page_size), C::DCH,
                                    static_cast<cuuint64_t>(c.kv_heads), static_cast<cuuint64_t>(c.pages)};
        const cuuint64_t strides[4] = {row, C::CB, row * c.page_size, static_cast<cuuint64_t>(c.v_stride)};
        const cuuint32_t box[5] = {C::CHE, static_cast<cuuint32_t>(c.page_size), C::DCH, 1, 1};
        if (int rc = encode_map(&tv, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5, c.v, dims, strides, box, C::CB)) return rc;
    }
    if (int rc = launch_after(kern, dim3(blocks), C::THREADS, C::SMEM_BYTES, st, tk, tv, a)) return rc;
    if (!join) return FP4ATTN_OK;
    return launch_after(paged_join_kernel<OutT, D, HC>, dim3(blocks, a.heads_per_group), 256, 0, st, a);
}

template <typename OutT, int D>
int launch_heads(const PagedArgs& a, int blocks, bool join, cudaStream_t st)
{
    switch (heads_at_once(a.group)) {
        case 4: return launch_attention<OutT, D, 4>(a, blocks, join, st);
        case 8: return launch_attention<OutT, D, 8>(a, blocks, join, st);
        default: return launch_attention<OutT, D, 16>(a, blocks, join, st);
    }
}

template <typename OutT>
int launch_dim(const PagedArgs& a, int blocks, bool join, cudaStream_t st)
{
    switch (a.c.head_dim) {
        case 32: return launch_heads<OutT, 32>(a, blocks, join, st);
        case 64: return launch_heads<OutT, 64>(a, blocks, join, st);
        case 96: return launch_heads<OutT, 96>(a, blocks, join, st);
        case 128: return launch_heads<OutT, 128>(a, blocks, join, st);
        case 160: return launch_heads<OutT, 160>(a, blocks, join, st);
        default: return launch_heads<OutT, 256>(a, blocks, join, st);
    }
}

// fp4attn_paged_attention.  test_timeout_ns > 0: its abort self-test, the FP32
// output kernel of up to four heads of 64 with one withheld arrival, waits
// bounded by that time.
int do_paged_attention(const fp4attn_cache* cache, const void* Q, void* Out, float* lse, int in_dtype, int out_dtype, int batch,
                       int q_heads, const int64_t* q_strides, const int32_t* block_table, int64_t table_stride, int max_pages,
                       const int32_t* seq_lens, float softmax_scale, int scale_mode, void* workspace, size_t workspace_bytes,
                       void* stream, unsigned long long test_timeout_ns = 0)
{
    if (int rc = check_cache(cache)) return rc;
    if (bad_dtype(in_dtype) || bad_dtype(out_dtype)) return fail(FP4ATTN_EINVAL, "dtype %d, %d", in_dtype, out_dtype);
    if (scale_mode != FP4ATTN_SCALE_REFERENCE && scale_mode != FP4ATTN_SCALE_OCP)
        return fail(FP4ATTN_EINVAL, "scale_mode %d", scale_mode);
    if (batch < 0 || batch > 65535) return fail(FP4ATTN_EINVAL, "batch %d in [0, 65535]", batch);
    if (q_heads < 1 || q_heads % cache->kv_heads)
        return fail(FP4ATTN_EINVAL, "q_heads %d is not a multiple of kv_heads %d", q_heads, cache->kv_heads);
    if (int rc = check_table(block_table, table_stride, batch, max_pages)) return rc;
    // (the device counts tokens and tiles in 32 bits)
    if (static_cast<int64_t>(max_pages) * cache->page_size > (1 << 30))
        return fail(FP4ATTN_EINVAL, "max_pages %d of %d tokens: more than 2^30", max_pages, cache->page_size);
    const int64_t longest = (static_cast<int64_t>(max_pages) * cache->page_size + kPagedTile - 1) / kPagedTile;
    const int64_t most_tiles = longest * q_heads * batch;
    if (most_tiles > 0x7FFFFFFF) return fail(FP4ATTN_EINVAL, "batch %d x heads %d x max_pages %d: more than 2^31 tiles", batch, q_heads, max_pages);
    if (batch == 0) return FP4ATTN_OK;
    if (!Q || !Out || !q_strides || !seq_lens) return fail(FP4ATTN_EINVAL, "null pointer");
    if (!wide(Q, in_dtype, {q_strides[0], q_strides[1]}) || !aligned(Out, 16) || !aligned(lse, 4) || !aligned(seq_lens, 4) ||
        !aligned(block_table, 4))
        return fail(FP4ATTN_EINVAL, "Q (and its strides) and Out must be 16-byte aligned");
    const size_t need = fp4attn_paged_attention_workspace_size(batch, q_heads, cache->kv_heads, cache->head_dim);
    if (!workspace || workspace_bytes < need)
        return fail(FP4ATTN_EWORKSPACE, "workspace of %zu bytes needed, %zu given", need, workspace ? workspace_bytes : 0);
    if (!aligned(workspace, 256)) return fail(FP4ATTN_EINVAL, "workspace must be 256-byte aligned");
    if (int rc = host::ready()) return rc;
    PagedArgs a{};
    a.q = Q;
    a.q_half = in_dtype == FP4ATTN_F16;
    a.qb = q_strides[0];
    a.qh = q_strides[1];
    a.batch = batch;
    a.q_heads = q_heads;
    a.group = q_heads / cache->kv_heads;
    a.c = view_of(*cache);
    a.t = TableView{block_table, table_stride, batch, max_pages};
    a.seq_lens = seq_lens;
    const float scale = softmax_scale > 0.f ? softmax_scale : 1.0f / std::sqrt(static_cast<float>(cache->head_dim));
    a.scale_log2 = scale * 1.4426950408889634f;
    a.ocp = scale_mode == FP4ATTN_SCALE_OCP;
    a.out = Out;
    a.lse = lse;
    const int nh = heads_at_once(a.group);
    a.splits = (a.group + nh - 1) / nh;
    a.heads_per_group = (a.group + a.splits - 1) / a.splits;
    a.head_groups = cache->kv_heads * a.splits;
    const AttentionWorkspace ws = attention_workspace(a.group, cache->head_dim);
    char* base = static_cast<char*>(workspace);
    a.p = PagedPartials{reinterpret_cast<float*>(base + ws.o), reinterpret_cast<float2*>(base + ws.ml),
                        reinterpret_cast<int4*>(base + ws.items)};
    a.timeout_ns = test_timeout_ns ? test_timeout_ns : host::timeout_ns();
    // The most tiles the block table allows; what there are is known on the device.
    const int64_t tiles = longest * a.head_groups * batch;
    const int blocks = static_cast<int>(std::min<int64_t>({kPagedBlocks, host::sms(), tiles}));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (test_timeout_ns) return launch_attention<float, 64, 4, true>(a, blocks, longest > 1, st);
    return out_dtype == FP4ATTN_F16 ? launch_dim<__half>(a, blocks, longest > 1, st) : launch_dim<float>(a, blocks, longest > 1, st);
}

template <int kArrays, int kPairs>
int launch_copies(const std::vector<CopyArray>& arrays, const int32_t* src, const int32_t* dst, int n, cudaStream_t st)
{
    CopyArgs<kArrays, kPairs> a;
    for (size_t first = 0; first < arrays.size(); first += kArrays) {
        a.n_arrays = static_cast<int>(std::min<size_t>(kArrays, arrays.size() - first));
        int chunks = 0;
        for (int i = 0; i < a.n_arrays; i++) {
            a.arrays[i] = arrays[first + i];
            a.arrays[i].first_chunk = chunks;
            chunks += (a.arrays[i].page_bytes + kCopyChunk - 1) / kCopyChunk;
        }
        for (int p0 = 0; p0 < n; p0 += kPairs) {
            const int m = std::min(kPairs, n - p0);
            for (int i = 0; i < m; i++) a.pairs[i] = make_int2(src[p0 + i], dst[p0 + i]);
            if (int rc = launch_after(copy_pages_kernel<kArrays, kPairs>, dim3(chunks, m), 256, 0, st, a)) return rc;
        }
    }
    return FP4ATTN_OK;
}

}  // namespace

extern "C" {

int fp4attn_rotary_table(const double* freqs, int pairs, int64_t max_positions, double factor, float* table, void* stream)
{
    host::clear_error();
    if (!freqs || !table || !aligned(table, 16)) return fail(FP4ATTN_EINVAL, "null or misaligned pointer");
    if (pairs < 1 || pairs > 128 || max_positions < 1) return fail(FP4ATTN_EINVAL, "pairs in [1, 128], max_positions >= 1");
    for (int i = 0; i < pairs; i++)
        if (!std::isfinite(freqs[i])) return fail(FP4ATTN_EINVAL, "freqs[%d] is not finite", i);
    if (!std::isfinite(factor)) return fail(FP4ATTN_EINVAL, "factor is not finite");
    if (int rc = host::ready()) return rc;
    RotaryFreqs f{};
    std::memcpy(f.f, freqs, pairs * sizeof(double));
    const int64_t blocks = std::min<int64_t>((max_positions * pairs + 255) / 256, 148 * 32);
    rotary_table_kernel<<<static_cast<unsigned>(blocks), 256, 0, static_cast<cudaStream_t>(stream)>>>(
        f, pairs, max_positions, factor, reinterpret_cast<float2*>(table));
    PAGED_CUDA(cudaGetLastError());
    return FP4ATTN_OK;
}

int fp4attn_rotary(const void* x, void* y, int dtype, int batch, int heads, int seq, int head_dim,
                   const int64_t* x_strides, const int64_t* y_strides, const float* table, int rotary_dim,
                   int64_t max_positions, const int32_t* positions, int64_t positions_stride, int interleaved, int inverse,
                   void* stream)
{
    host::clear_error();
    if (bad_dtype(dtype)) return fail(FP4ATTN_EINVAL, "dtype %d", dtype);
    if (batch < 0 || heads < 0 || seq < 0 || batch > 65535 || heads > 65535)
        return fail(FP4ATTN_EINVAL, "batch and heads in [0, 65535], seq >= 0");
    if (!supported_dim(head_dim))
        return fail(FP4ATTN_EUNSUPPORTED, "head_dim %d is not one of 32/64/96/128/160/256", head_dim);
    if (int rc = check_rotary(table, rotary_dim, max_positions, head_dim)) return rc;
    if (!positions && seq > max_positions) return fail(FP4ATTN_EINVAL, "seq %d exceeds the table's %lld positions", seq,
                                                       static_cast<long long>(max_positions));
    if (batch == 0 || heads == 0 || seq == 0) return FP4ATTN_OK;
    if (!x || !y || !x_strides || !y_strides) return fail(FP4ATTN_EINVAL, "null pointer");
    if (!aligned(x, bytes_of(dtype)) || !aligned(y, bytes_of(dtype)) || !aligned(positions, 4))
        return fail(FP4ATTN_EINVAL, "misaligned pointer");
    if (int rc = host::ready()) return rc;
    RotaryArgs a{x, y, x_strides[0], x_strides[1], x_strides[2], y_strides[0], y_strides[1], y_strides[2],
                 heads, seq, head_dim, rotary_dim, reinterpret_cast<const float2*>(table), positions, positions_stride,
                 max_positions, inverse ? -1.f : 1.f, 1};
    const bool in_eights = wide(x, dtype, {a.xb, a.xh, a.xs}) && wide(y, dtype, {a.yb, a.yh, a.ys});
    const bool vec = in_eights && (interleaved || rotary_dim % 16 == 0), by_rows = in_eights && !vec;
    const int64_t units = by_rows              ? head_dim / 8
                          : vec && interleaved ? head_dim / 8
                          : vec                ? rotary_dim / 16 + (head_dim - rotary_dim) / 8
                                               : head_dim - rotary_dim / 2;
    const int64_t work = seq * units;
    if (work > 0x7FFFFF00) return fail(FP4ATTN_EINVAL, "seq %d is too long", seq);
    // Several heads a thread where that leaves every SM its 2048 threads.
    while (a.heads_per_thread < (by_rows ? 16 : 4) && work * batch * (heads / (2 * a.heads_per_thread)) >= 148 * 2048) a.heads_per_thread *= 2;
    const int64_t blocks = by_rows ? (seq + 256 / units - 1) / (256 / units) : (work + 255) / 256;
    const dim3 grid(static_cast<unsigned>(blocks), (heads + a.heads_per_thread - 1) / a.heads_per_thread, batch);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (by_rows)
        return launch_after(dtype == FP4ATTN_F16 ? rotary_rows_kernel<__half> : rotary_rows_kernel<float>, grid, 256, 0, st, a);
    return dtype == FP4ATTN_F16 ? launch_rotary<__half>(grid, st, a, vec, interleaved != 0)
                                : launch_rotary<float>(grid, st, a, vec, interleaved != 0);
}

int fp4attn_cache_append(const fp4attn_cache* cache, const void* K, const void* V, const void* Q, void* Q_out, int dtype,
                         int tokens, int q_heads, const int64_t* k_strides, const int64_t* v_strides,
                         const int64_t* q_strides, const int32_t* block_table, int64_t table_stride, int seqs,
                         int max_pages, const int32_t* seq_ids, const int32_t* positions, const float* table,
                         int rotary_dim, int64_t max_positions, int interleaved, int scale_mode, void* stream)
{
    host::clear_error();
    if (int rc = check_cache(cache)) return rc;
    if (bad_dtype(dtype)) return fail(FP4ATTN_EINVAL, "dtype %d", dtype);
    if (scale_mode != FP4ATTN_SCALE_REFERENCE && scale_mode != FP4ATTN_SCALE_OCP)
        return fail(FP4ATTN_EINVAL, "scale_mode %d", scale_mode);
    if (tokens < 0) return fail(FP4ATTN_EINVAL, "tokens must be >= 0");
    if (int rc = check_table(block_table, table_stride, seqs, max_pages)) return rc;
    if (!seq_ids && tokens != seqs) return fail(FP4ATTN_EINVAL, "without seq_ids there is one token per sequence");
    if (table)
        if (int rc = check_rotary(table, rotary_dim, max_positions, cache->head_dim)) return rc;
    if (!Q != !Q_out || (Q && (q_heads < 1 || q_heads > 65535))) return fail(FP4ATTN_EINVAL, "Q and Q_out go together, with q_heads in [1, 65535]");
    if (tokens == 0) return FP4ATTN_OK;
    if (!K || !V || !positions || !k_strides || !v_strides || (Q && !q_strides)) return fail(FP4ATTN_EINVAL, "null pointer");
    const int es = bytes_of(dtype);
    if (!aligned(K, es) || !aligned(V, es) || !aligned(Q, es) || !aligned(Q_out, 16) || !aligned(positions, 4) ||
        !aligned(seq_ids, 4) || !aligned(block_table, 4))
        return fail(FP4ATTN_EINVAL, "misaligned pointer");
    if (int rc = host::ready()) return rc;
    AppendArgs a{};
    a.k = K; a.v = V; a.q = Q; a.q_out = Q_out;
    a.kt = k_strides[0]; a.kh = k_strides[1];
    a.vt = v_strides[0]; a.vh = v_strides[1];
    if (Q) { a.qt = q_strides[0]; a.qh = q_strides[1]; }
    a.tokens = tokens;
    a.q_heads = Q ? q_heads : 0;
    a.c = view_of(*cache);
    a.t = TableView{block_table, table_stride, seqs, max_pages};
    a.seq_ids = seq_ids;
    a.positions = positions;
    a.table = reinterpret_cast<const float2*>(table);
    a.rot = table ? rotary_dim : 0;
    a.max_positions = max_positions;
    a.interleaved = interleaved != 0;
    a.ocp = scale_mode == FP4ATTN_SCALE_OCP;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool f16 = dtype == FP4ATTN_F16;
    if (wide(K, dtype, {a.kt, a.kh}) && wide(V, dtype, {a.vt, a.vh}) && (!Q || wide(Q, dtype, {a.qt, a.qh}))) {
        const bool by_rows = !a.interleaved && a.rot % 64 != 0;
        const int units = by_rows ? a.c.head_dim / 8 : append_units(a.c.head_dim, a.rot, a.interleaved);
        const int at_once = kAppendThreads / units, sets = (2 * a.c.kv_heads + a.q_heads + at_once - 1) / at_once;
        if (sets > 65535) return fail(FP4ATTN_EINVAL, "%d heads are too many", 2 * a.c.kv_heads + a.q_heads);
        const dim3 grid(tokens, sets);
        if (by_rows)
            return launch_after(f16 ? cache_append_rows_kernel<__half> : cache_append_rows_kernel<float>, grid, kAppendThreads, 0, st, a);
        return f16 ? launch_append<__half>(grid, st, a) : launch_append<float>(grid, st, a);
    }
    const int64_t work = static_cast<int64_t>(tokens) * (2 * a.c.kv_heads + a.q_heads) * (a.c.head_dim / 8);
    if ((work + 255) / 256 > 0x7FFFFFFF) return fail(FP4ATTN_EINVAL, "%d tokens are too many", tokens);
    const unsigned grid = static_cast<unsigned>((work + 255) / 256);
    return launch_after(f16 ? cache_append_any_kernel<__half> : cache_append_any_kernel<float>, grid, 256, 0, st, a);
}

int fp4attn_cache_gather(const fp4attn_cache* cache, const int32_t* block_table, int64_t table_stride, int seqs,
                         int max_pages, const int32_t* starts, const int32_t* lengths, int max_length, int heads, void* K,
                         void* V, int dtype, void* stream)
{
    host::clear_error();
    if (int rc = check_cache(cache)) return rc;
    if (bad_dtype(dtype)) return fail(FP4ATTN_EINVAL, "dtype %d", dtype);
    if (int rc = check_table(block_table, table_stride, seqs, max_pages)) return rc;
    if (heads < 1 || heads % cache->kv_heads) return fail(FP4ATTN_EINVAL, "heads %d is not a multiple of kv_heads %d", heads, cache->kv_heads);
    if (max_length < 0 || max_length > (1 << 30) || seqs > 65535)
        return fail(FP4ATTN_EINVAL, "max_length in [0, 2^30], at most 65535 sequences");
    if (seqs == 0 || max_length == 0) return FP4ATTN_OK;
    if (!lengths || !K || !V || !aligned(K, 16) || !aligned(V, 16) || !aligned(lengths, 4) || !aligned(starts, 4) ||
        !aligned(block_table, 4))
        return fail(FP4ATTN_EINVAL, "null or misaligned pointer");
    if (int rc = host::ready()) return rc;
    const GatherArgs a{view_of(*cache), TableView{block_table, table_stride, seqs, max_pages}, starts, lengths,
                       max_length, heads / cache->kv_heads, K, V};
    const int rows = 256 / (cache->head_dim / 8) * kGatherRows;
    const dim3 grid(static_cast<unsigned>((static_cast<int64_t>(max_length) + rows - 1) / rows), cache->kv_heads, seqs);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return dtype == FP4ATTN_F16 ? launch_gather<__half>(grid, st, a) : launch_gather<float>(grid, st, a);
}

size_t fp4attn_paged_attention_workspace_size(int batch, int q_heads, int kv_heads, int head_dim)
{
    if (batch < 1 || kv_heads < 1 || q_heads < 1 || q_heads % kv_heads || !supported_dim(head_dim)) return 0;
    return attention_workspace(q_heads / kv_heads, head_dim).total;
}

int fp4attn_paged_attention(const fp4attn_cache* cache, const void* Q, void* Out, float* lse, int in_dtype, int out_dtype,
                            int batch, int q_heads, const int64_t* q_strides, const int32_t* block_table,
                            int64_t table_stride, int max_pages, const int32_t* seq_lens, float softmax_scale,
                            int scale_mode, void* workspace, size_t workspace_bytes, void* stream)
{
    host::clear_error();
    return do_paged_attention(cache, Q, Out, lse, in_dtype, out_dtype, batch, q_heads, q_strides, block_table, table_stride,
                              max_pages, seq_lens, softmax_scale, scale_mode, workspace, workspace_bytes, stream);
}

int fp4attn_selftest_paged_abort(const fp4attn_cache* cache, const void* Q, float* Out, int batch, int q_heads,
                                 const int32_t* block_table, int64_t table_stride, int max_pages, const int32_t* seq_lens,
                                 void* workspace, size_t workspace_bytes, unsigned timeout_us, void* stream)
{
    host::clear_error();
    if (timeout_us < 1 || timeout_us > 10000000u) return fail(FP4ATTN_EINVAL, "timeout_us in [1, 1e7]");
    if (int rc = check_cache(cache)) return rc;
    if (cache->head_dim != 64 || q_heads > 4 * static_cast<int64_t>(cache->kv_heads))
        return fail(FP4ATTN_EINVAL, "the self-test takes head_dim 64 and up to four query heads a key/value head");
    const int64_t strides[2] = {64 * static_cast<int64_t>(q_heads), 64};
    return do_paged_attention(cache, Q, Out, nullptr, FP4ATTN_F16, FP4ATTN_F32, batch, q_heads, strides, block_table, table_stride,
                              max_pages, seq_lens, 0.f, FP4ATTN_SCALE_REFERENCE, workspace, workspace_bytes, stream,
                              static_cast<unsigned long long>(timeout_us) * 1000ull);
}

int fp4attn_copy_pages(const fp4attn_cache* caches, int n_caches, const int32_t* src, const int32_t* dst, int n, void* stream)
{
    host::clear_error();
    if (n_caches < 0 || n < 0 || (n_caches && !caches) || (n && (!src || !dst))) return fail(FP4ATTN_EINVAL, "null pointer or negative count");
    try {
        std::vector<CopyArray> arrays;
        int pages = 0x7FFFFFFF;
        for (int i = 0; i < n_caches; i++) {
            const fp4attn_cache& c = caches[i];
            if (int rc = check_cache(&c)) return rc;
            const int rows = c.kv_heads * c.page_size;
            arrays.push_back({static_cast<uint8_t*>(c.v), c.v_stride, rows * c.head_dim * 2, 0});
            arrays.push_back({c.k_codes, c.k_codes_stride, rows * c.head_dim / 2, 0});
            arrays.push_back({c.k_scales, c.k_scales_stride, rows * c.head_dim / 32, 0});
            pages = std::min(pages, c.pages);
        }
        // Every copy reads what was there before the call: no page is written
        // twice, and none is both read and written.
        if (n_caches && n) {
            std::vector<uint8_t> seen(pages, 0);
            for (int i = 0; i < n; i++) {
                if (src[i] < 0 || src[i] >= pages || dst[i] < 0 || dst[i] >= pages)
                    return fail(FP4ATTN_EINVAL, "pair %d (%d to %d): page outside [0, %d)", i, src[i], dst[i], pages);
                if (seen[dst[i]]) return fail(FP4ATTN_EINVAL, "page %d is written twice", dst[i]);
                seen[dst[i]] = 1;
            }
            for (int i = 0; i < n; i++)
                if (seen[src[i]]) return fail(FP4ATTN_EINVAL, "page %d is both read and written", src[i]);
        }
        if (n_caches == 0 || n == 0) return FP4ATTN_OK;
        if (int rc = host::ready()) return rc;
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        if (arrays.size() <= 24 && n <= 64) return launch_copies<24, 64>(arrays, src, dst, n, st);
        return launch_copies<192, 2048>(arrays, src, dst, n, st);
    } catch (const std::bad_alloc&) {
        return fail(FP4ATTN_EINVAL, "out of host memory");
    }
}

}  // extern "C"
