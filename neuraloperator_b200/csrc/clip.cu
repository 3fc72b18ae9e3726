// Global norm over many tensors, and clipping by it (the step between loss.backward() and the optimizer).
//
//   norm = sqrt(sum over all tensors of sum |g|^2)   (or max |g|)
//   g'   = g * min(1, max_norm / (norm + 1e-6))
//
// Complex gradients (the spectral weights) are pairs of reals: the same sums and the same scaling.
// Both steps are bound by HBM: the norm reads every gradient once, the scaling reads and writes them once.
// Tensors come as a table in the kernel's parameters (up to kItems a launch), so a call copies nothing to the
// device and can be captured into a graph.  Every tensor is cut into chunks of kChunk values; CTA b takes the
// chunks b, b + grid, ... of the table, and each CTA leaves one partial sum.  The scaling kernel's CTAs add the
// partial sums up themselves, each in the same order, so there is no launch between the two, no atomic, and the
// result does not depend on scheduling.  The scaling walks the chunks backwards: the last chunks that the norm
// read are still in the 126 MB L2 (and are loaded with the wish to stay there).
// Measured on B200, 0.57 GB of fp32 gradients: norm 111 us (5.1 TB/s), scaling 180 us (6.3 TB/s).  A call with some tens
// of small tensors takes 7 us on the device and the host's time for its lists.
#include "l2_hints.cuh"
#include "nop_internal.cuh"

#include <cuda_fp16.h>

#include <algorithm>
#include <exception>

namespace nop {

int32_t current_device(int* dev, int* sms) {
    static std::atomic<int> known[64];
    NOP_CUDA_TRY(cudaGetDevice(dev));
    int n = *dev < 64 ? known[*dev].load(std::memory_order_relaxed) : 0;
    if (!n) {
        NOP_CUDA_TRY(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, *dev));
        if (*dev < 64) known[*dev].store(n, std::memory_order_relaxed);
    }
    *sms = n;
    return NOP_OK;
}

namespace clip {

constexpr int kItems = 256;         // tensors a launch (a 32-byte entry each in the kernel parameters)
constexpr int kChunk = 8192;        // values a chunk
constexpr int kThreads = 256;
constexpr uint32_t kKeep = 2560;    // chunks of a launch that L2 is asked to keep for the scaling: 80 MB in fp32
constexpr int kMaxGrid = 1024;      // partial sums a launch leaves at most

struct Item {
    const void* src;
    void* dst;
    int64_t n;          // reals
    uint32_t first;     // index of the first chunk
    int32_t dtype;
};

struct Table {
    Item it[kItems];
    int32_t count;
    uint32_t chunks;
};

__device__ __forceinline__ const Item& item_of(const Table& t, uint32_t chunk) {
    int lo = 0, hi = t.count - 1;  // the last item whose first chunk is <= chunk
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.it[mid].first <= chunk) lo = mid;
        else hi = mid - 1;
    }
    return t.it[lo];
}

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f(float* d, float v) { *d = v; }
__device__ __forceinline__ void from_f(__half* d, float v) { *d = __float2half_rn(v); }
__device__ __forceinline__ void from_f(__nv_bfloat16* d, float v) { *d = __float2bfloat16_rn(v); }

// the two norms as one running value: the sum of squares, or the largest magnitude (a NaN stays)
template <bool INF>
__device__ __forceinline__ float add_value(float s, float v) {
    if (!INF) return fmaf(v, v, s);
    const float a = fabsf(v);
    return (a > s || a != a) ? a : s;
}
template <bool INF>
__device__ __forceinline__ double join(double a, double b) {
    if (!INF) return a + b;
    return (b > a || b != b) ? b : a;
}

template <bool INF>
__device__ double block_join(double v) {
    __shared__ double part[kThreads / 32];
    __shared__ double total;
#pragma unroll
    for (int o = 16; o; o >>= 1) v = join<INF>(v, __shfl_down_sync(0xffffffffu, v, o));
    __syncthreads();  // an earlier call's total has been read
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = v;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < kThreads / 32; ++i) v = join<INF>(v, part[i]);
        total = v;
    }
    __syncthreads();
    return total;
}

// A thread's part of one chunk: at most kChunk / kThreads = 32 squares in fp32 before they join the running
// sum in 64 bits, so the sum over any number of values keeps fp32's precision.
template <bool INF, class T>
__device__ float chunk_value(const T* __restrict__ src, int len, uint64_t pol) {
    float s = 0.f;
    constexpr int V = 16 / (int)sizeof(T);
    if ((reinterpret_cast<uintptr_t>(src) & 15) == 0) {
        const uint4* v4 = reinterpret_cast<const uint4*>(src);
        const int nv = len / V;
#pragma unroll 4
        for (int i = threadIdx.x; i < nv; i += kThreads) {
            const float4 q = l2::ld4(v4 + i, pol);
            const T* e = reinterpret_cast<const T*>(&q);
#pragma unroll
            for (int j = 0; j < V; ++j) s = add_value<INF>(s, to_f(e[j]));
        }
        for (int i = nv * V + threadIdx.x; i < len; i += kThreads) s = add_value<INF>(s, to_f(src[i]));
    } else {
#pragma unroll 8
        for (int i = threadIdx.x; i < len; i += kThreads) s = add_value<INF>(s, to_f(src[i]));
    }
    return s;
}

template <bool INF>
__global__ void __launch_bounds__(kThreads) k_norm(const __grid_constant__ Table t, double* __restrict__ partial) {
    const uint64_t keep = l2::evict_last(), pass = l2::evict_first();
    double acc = 0.0;
    for (uint32_t c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const Item& it = item_of(t, c);
        const int64_t at = (int64_t)(c - it.first) * kChunk;
        const int len = (int)(it.n - at < kChunk ? it.n - at : kChunk);
        const uint64_t pol = t.chunks - c <= kKeep ? keep : pass;
        float s;
        if (it.dtype == NOP_DTYPE_FP32) s = chunk_value<INF>(static_cast<const float*>(it.src) + at, len, pol);
        else if (it.dtype == NOP_DTYPE_BF16) s = chunk_value<INF>(static_cast<const __nv_bfloat16*>(it.src) + at, len, pol);
        else s = chunk_value<INF>(static_cast<const __half*>(it.src) + at, len, pol);
        acc = join<INF>(acc, (double)s);
    }
    acc = block_join<INF>(acc);
    if (threadIdx.x == 0) partial[blockIdx.x] = acc;
}

// the norm from the partial sums, the same value in every CTA
template <bool INF>
__device__ float norm_of(const double* __restrict__ partial, int parts) {
    double acc = 0.0;
    for (int i = threadIdx.x; i < parts; i += kThreads) acc = join<INF>(acc, partial[i]);
    acc = block_join<INF>(acc);
    return (float)(INF ? acc : sqrt(acc));
}

template <class T>
__device__ void scale_chunk(const T* src, T* dst, int len, float coef) {
    constexpr int V = 16 / (int)sizeof(T);
    if (((reinterpret_cast<uintptr_t>(src) | reinterpret_cast<uintptr_t>(dst)) & 15) == 0) {
        const uint4* s4 = reinterpret_cast<const uint4*>(src);
        uint4* d4 = reinterpret_cast<uint4*>(dst);
        const int nv = len / V;
#pragma unroll 4
        for (int i = threadIdx.x; i < nv; i += kThreads) {
            uint4 q = __ldcs(s4 + i);
            T* e = reinterpret_cast<T*>(&q);
#pragma unroll
            for (int j = 0; j < V; ++j) from_f(&e[j], to_f(e[j]) * coef);
            __stcs(d4 + i, q);
        }
        for (int i = nv * V + threadIdx.x; i < len; i += kThreads) from_f(&dst[i], to_f(src[i]) * coef);
    } else {
#pragma unroll 8
        for (int i = threadIdx.x; i < len; i += kThreads) from_f(&dst[i], to_f(src[i]) * coef);
    }
}

template <bool INF>
__global__ void __launch_bounds__(kThreads)
k_scale(const __grid_constant__ Table t, const double* __restrict__ partial, int parts, double max_norm,
        float* __restrict__ norm) {
    const float n = norm_of<INF>(partial, parts);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = n;
    const double ratio = max_norm / ((double)n + 1e-6);
    const float coef = ratio > 1.0 ? 1.f : (float)ratio;  // a NaN norm gives NaN gradients
    for (uint32_t k = blockIdx.x; k < t.chunks; k += gridDim.x) {
        const uint32_t c = t.chunks - 1 - k;
        const Item& it = item_of(t, c);
        if (coef == 1.f && it.src == it.dst) continue;  // in place and under the limit: nothing to write
        const int64_t at = (int64_t)(c - it.first) * kChunk;
        const int len = (int)(it.n - at < kChunk ? it.n - at : kChunk);
        if (it.dtype == NOP_DTYPE_FP32)
            scale_chunk(static_cast<const float*>(it.src) + at, static_cast<float*>(it.dst) + at, len, coef);
        else if (it.dtype == NOP_DTYPE_BF16)
            scale_chunk(static_cast<const __nv_bfloat16*>(it.src) + at, static_cast<__nv_bfloat16*>(it.dst) + at, len,
                        coef);
        else
            scale_chunk(static_cast<const __half*>(it.src) + at, static_cast<__half*>(it.dst) + at, len, coef);
    }
}

template <bool INF>
__global__ void __launch_bounds__(kThreads)
k_norm_only(const double* __restrict__ partial, int parts, float* __restrict__ norm) {
    const float n = norm_of<INF>(partial, parts);
    if (threadIdx.x == 0) *norm = n;
}

template <bool INF>
int32_t run(const std::vector<Table>& tables, bool scale, double max_norm, float* norm, double* partial, int sms,
            cudaStream_t s) {
    int parts = 0;
    for (const Table& t : tables) {
        const unsigned grid = (unsigned)std::min<uint32_t>(t.chunks, (uint32_t)std::min(4 * sms, kMaxGrid));
        k_norm<INF><<<grid, kThreads, 0, s>>>(t, partial + parts);
        NOP_CUDA_TRY(cudaGetLastError());
        parts += (int)grid;
    }
    if (!scale || tables.empty()) {
        if (norm) k_norm_only<INF><<<1, kThreads, 0, s>>>(partial, parts, norm);
        NOP_CUDA_TRY(cudaGetLastError());
        return NOP_OK;
    }
    for (size_t i = tables.size(); i-- > 0;) {
        const Table& t = tables[i];
        const unsigned grid = (unsigned)std::min<uint32_t>(t.chunks, (uint32_t)(8 * sms));
        k_scale<INF><<<grid, kThreads, 0, s>>>(t, partial, parts, max_norm, i == 0 ? norm : nullptr);
        NOP_CUDA_TRY(cudaGetLastError());
    }
    return NOP_OK;
}

}  // namespace clip
}  // namespace nop

using namespace nop;

extern "C" {

int32_t nop_clip_workspace_size(int32_t n, size_t* bytes) {
    if (n < 0 || !bytes) return fail(NOP_E_INVALID, "the number of tensors must be >= 0 and bytes non-NULL");
    *bytes = (size_t)(ceil_div(n, clip::kItems) + 1) * clip::kMaxGrid * sizeof(double);
    return NOP_OK;
}

int32_t nop_clip_by_norm(int32_t n, const void* const* src, void* const* dst, const int64_t* numel,
                         const int32_t* dtypes, int32_t norm_type, double max_norm, float* norm, void* workspace,
                         size_t workspace_bytes, void* stream) try {
    size_t need = 0;
    const int32_t rc = nop_clip_workspace_size(n, &need);
    if (rc != NOP_OK) return rc;
    if (n && (!src || !numel || !dtypes)) return fail(NOP_E_INVALID, "src, numel and dtypes must be non-NULL");
    if (norm_type != NOP_NORM_L2 && norm_type != NOP_NORM_INF)
        return fail(NOP_E_INVALID, "norm_type must be NOP_NORM_L2 or NOP_NORM_INF");
    if (dst && !(max_norm >= 0.0)) return fail(NOP_E_INVALID, "max_norm must be a number >= 0");
    if (!dst && !norm) return fail(NOP_E_INVALID, "neither dst nor norm is given");
    if (!workspace || workspace_bytes < need) return fail(NOP_E_WORKSPACE, "workspace missing or too small");
    if ((uintptr_t)workspace % 8) return fail(NOP_E_ALIGNMENT, "the workspace must be 8-byte aligned");
    std::vector<clip::Table> tables;
    for (int32_t i = 0; i < n; ++i) {
        if (numel[i] < 0) return fail(NOP_E_INVALID, "numel must be >= 0");
        if (dtypes[i] < NOP_DTYPE_FP32 || dtypes[i] > NOP_DTYPE_FP16) return fail(NOP_E_INVALID, "unknown dtype");
        if (numel[i] == 0) continue;
        if (!src[i] || (dst && !dst[i])) return fail(NOP_E_INVALID, "a tensor's pointer is NULL");
        const uintptr_t size = dtypes[i] == NOP_DTYPE_FP32 ? 4 : 2;
        if ((uintptr_t)src[i] % size || (dst && (uintptr_t)dst[i] % size))
            return fail(NOP_E_ALIGNMENT, "a tensor's pointer is not aligned to its type");
        const int64_t chunks = ceil_div(numel[i], clip::kChunk);
        if (chunks > 0x3fffffffLL) return fail(NOP_E_UNSUPPORTED, "a tensor has more than 2^43 values");
        if (tables.empty() || tables.back().count == clip::kItems || tables.back().chunks + chunks > 0x7fffffffLL) {
            tables.emplace_back();
            tables.back().count = 0;
            tables.back().chunks = 0;
        }
        clip::Table& t = tables.back();
        t.it[t.count++] = {src[i], dst ? dst[i] : nullptr, numel[i], t.chunks, dtypes[i]};
        t.chunks += (uint32_t)chunks;
    }
    if (tables.size() * clip::kMaxGrid * sizeof(double) > workspace_bytes)
        return fail(NOP_E_WORKSPACE, "workspace too small");
    int dev = 0, sms = 148;
    const int32_t dc = current_device(&dev, &sms);
    if (dc != NOP_OK) return dc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    double* partial = static_cast<double*>(workspace);
    return norm_type == NOP_NORM_INF ? clip::run<true>(tables, dst != nullptr, max_norm, norm, partial, sms, s)
                                     : clip::run<false>(tables, dst != nullptr, max_norm, norm, partial, sms, s);
} catch (const std::exception& e) {
    return fail(NOP_E_NOMEM, std::string("nop_clip_by_norm: ") + e.what());
}

}  // extern "C"
