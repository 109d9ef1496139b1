// grad_norm.hip -- global gradient norm over many tensors, and clipping (include/rlipv2_gradnorm.h).
//
// Bound by HBM: one pass over the gradients for the norm, one more and a write for the clipped ones (nothing is known before the
// norm is).  The tensor lists travel as kernel arguments (240 / 160 tensors fit 4 KB), so there is no table to build on the device
// and nothing to keep in step with the caller's tensors.
//
// A workgroup takes one chunk of one tensor and finds it by bisection over the chunks' first numbers (scalar loads, the same for
// the whole group).  The chunk size grows with the model so that there are at most 8192 + n partial sums, which one workgroup joins
// (212.7 M gradients in 754 tensors, norm and clip: 387 us with 4096, 366 with 8192, 362 with 16384 and a longer join).
// Elements are moved 16 bytes at a time (flat gradient buffers put tensors at odd offsets: a chunk starts with the few elements in
// front of a 16-byte boundary; where only one side can be aligned the memory unit takes the other's unaligned vectors).  The clipped
// gradients are stored non-temporally: they are larger than the caches, and what the norm pass read last stays there for the clip pass,
// which starts with it (436 -> 387 us).
//
// The sums are float64 from the first product on: an element's square neither overflows nor vanishes, and the order of 10^8 terms
// does not show in the float32 result.  The conversions and float64 multiply-adds take less time than the loads.
//
// Measured: bf16 -> float32 clip of 212.7 M gradients 366 us (425 MB read twice, 851 MB written: 4.65 TB/s, a large copy's rate; the
// plain form 2405); largest element of 44.5 M float32 36 us (5 TB/s, in part from the memory-side cache); 3.7 M bf16 clipped 14 us;
// norm of 0.13 M 8.7 us, the two launches.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/rlipv2_gradnorm.h"
#include "../../include/rlipv2_msda.h"
#include "msda_device.h"

namespace {

using namespace msda;

constexpr int THREADS = 256, JOIN = 1024, GRAIN = 2048, CHUNKS = 8192;
constexpr int NORM_LIST = 240, CLIP_LIST = 160;
constexpr uint32_t SRC_F32 = 1u << 30, DST_F32 = 1u << 29, COUNT = DST_F32 - 1;

struct Entry { uint32_t first, last; };              // number of its first chunk in this launch; elements of its last chunk | types
struct NormList { const void *src[NORM_LIST]; Entry at[NORM_LIST]; int n; uint32_t chunk, chunks; };
struct ClipList { const void *src[CLIP_LIST]; void *dst[CLIP_LIST]; Entry at[CLIP_LIST]; int n; uint32_t chunk, chunks; };
static_assert(sizeof(NormList) <= 3900 && sizeof(ClipList) <= 3900, "kernel arguments");

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x2 u32x2_at2 __attribute__((aligned(2)));
typedef u32x4 u32x4_at2 __attribute__((aligned(2)));
typedef u32x4 u32x4_at4 __attribute__((aligned(4)));

// N consecutive elements: 8 or 16 bytes at any alignment the type has
template <typename T, int N> struct Run;
template <> struct Run<bf16_t, 8> {
    static __device__ __forceinline__ void load(const bf16_t *p, float (&v)[8])
    {
        const u32x4 w = *reinterpret_cast<const u32x4_at2 *>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[2 * i] = bf16_lo(w[i]); v[2 * i + 1] = bf16_hi(w[i]); }
    }
    static __device__ __forceinline__ void store(bf16_t *p, const float (&v)[8])
    {
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
        __builtin_nontemporal_store(w, reinterpret_cast<u32x4_at2 *>(p));
    }
};
template <> struct Run<bf16_t, 4> {
    static __device__ __forceinline__ void load(const bf16_t *p, float (&v)[4])
    {
        const u32x2 w = *reinterpret_cast<const u32x2_at2 *>(p);
#pragma unroll
        for (int i = 0; i < 2; ++i) { v[2 * i] = bf16_lo(w[i]); v[2 * i + 1] = bf16_hi(w[i]); }
    }
    static __device__ __forceinline__ void store(bf16_t *p, const float (&v)[4])
    {
        u32x2 w;
#pragma unroll
        for (int i = 0; i < 2; ++i) w[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
        __builtin_nontemporal_store(w, reinterpret_cast<u32x2_at2 *>(p));
    }
};
template <> struct Run<float, 4> {
    static __device__ __forceinline__ void load(const float *p, float (&v)[4])
    {
        const u32x4 w = *reinterpret_cast<const u32x4_at4 *>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(w[i]);
    }
    static __device__ __forceinline__ void store(float *p, const float (&v)[4])
    {
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(v[i]);
        __builtin_nontemporal_store(w, reinterpret_cast<u32x4_at4 *>(p));
    }
};
__device__ __forceinline__ float load_one(const bf16_t *p) { return bf16_to_float(*p); }
__device__ __forceinline__ float load_one(const float *p) { return *p; }
__device__ __forceinline__ void store_one(bf16_t *p, float v) { *p = (bf16_t)float_to_bf16_bits(v); }
__device__ __forceinline__ void store_one(float *p, float v) { *p = v; }

// elements in front of the first 16-byte boundary, at most n
template <typename T> __device__ __forceinline__ int lead_of(const T *p, int n)
{
    const int lead = (int)((16u - ((uint32_t)reinterpret_cast<uintptr_t>(p) & 15u)) & 15u) / (int)sizeof(T);
    return lead < n ? lead : n;
}

// the tensor that chunk `c` of this launch belongs to
template <typename L> __device__ __forceinline__ int tensor_of(const L &list, uint32_t c)
{
    int lo = 0, hi = list.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (list.at[mid].first <= c) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}
template <typename L> __device__ __forceinline__ int chunk_length(const L &list, int t, uint32_t c)
{
    const uint32_t end = t + 1 < list.n ? list.at[t + 1].first : list.chunks;
    return c + 1 == end ? (int)(list.at[t].last & COUNT) : (int)list.chunk;
}

// One value of the running sum / maximum.  The maximum compares the bits of |g|: among non-negative numbers they order as the
// numbers do, and a NaN is above infinity.
template <int ORDER> struct Sum {
    double s = 0.0;
    __device__ __forceinline__ void add(float g)
    {
        if (ORDER == GRAD_NORM_L2) s = fma((double)g, (double)g, s);
        else s += (double)fabsf(g);
    }
    __device__ __forceinline__ void join(const Sum &o) { s += o.s; }
    __device__ __forceinline__ void across(int mask) { s += __shfl_xor(s, mask, 64); }
    __device__ __forceinline__ double value() const { return s; }
    __device__ __forceinline__ void set(double v) { s = v; }
};
template <> struct Sum<GRAD_NORM_INF> {
    uint32_t m = 0;
    __device__ __forceinline__ void add(float g) { m = max(m, __float_as_uint(g) & 0x7fffffffu); }
    __device__ __forceinline__ void join(const Sum &o) { m = max(m, o.m); }
    __device__ __forceinline__ void across(int mask) { m = max(m, (uint32_t)__shfl_xor((int)m, mask, 64)); }
    __device__ __forceinline__ double value() const { return (double)__uint_as_float(m); }
    __device__ __forceinline__ void set(double v) { m = __float_as_uint((float)v); }
};

template <int ORDER, int N> __device__ __forceinline__ double group_total(Sum<ORDER> s)
{
    __shared__ double part[N / 64];
#pragma unroll
    for (int mask = 32; mask >= 1; mask >>= 1) s.across(mask);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s.value();
    __syncthreads();
    Sum<ORDER> all, one;
    all.set(part[0]);
    for (int i = 1; i < N / 64; ++i) { one.set(part[i]); all.join(one); }
    return all.value();
}

template <int ORDER, typename T> __device__ __forceinline__ Sum<ORDER> chunk_sum(const T *p, int n)
{
    constexpr int VEC = 16 / (int)sizeof(T), STEP = THREADS * VEC, DEEP = 4;
    Sum<ORDER> a[DEEP];                                    // independent sums: four loads in flight per thread
    const int lead = lead_of(p, n);
    if ((int)threadIdx.x < lead) a[0].add(load_one(p + threadIdx.x));
    p += lead;
    n -= lead;
    int i = threadIdx.x * VEC;
    for (; i + (DEEP - 1) * STEP + VEC <= n; i += DEEP * STEP) {
        float v[DEEP][VEC];
#pragma unroll
        for (int j = 0; j < DEEP; ++j) Run<T, VEC>::load(p + i + j * STEP, v[j]);
#pragma unroll
        for (int j = 0; j < DEEP; ++j)
#pragma unroll
            for (int e = 0; e < VEC; ++e) a[j].add(v[j][e]);
    }
    for (; i + VEC <= n; i += STEP) {
        float v[VEC];
        Run<T, VEC>::load(p + i, v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) a[0].add(v[e]);
    }
    const int rest = n & ~(VEC - 1);
    if (rest + (int)threadIdx.x < n) a[0].add(load_one(p + rest + threadIdx.x));
#pragma unroll
    for (int j = 1; j < DEEP; ++j) a[0].join(a[j]);
    return a[0];
}

template <int ORDER> __global__ __launch_bounds__(THREADS) void norm_kernel(NormList list, double *partial)
{
    const uint32_t c = blockIdx.x;
    const int t = tensor_of(list, c), n = chunk_length(list, t, c);
    const int64_t begin = (int64_t)(c - list.at[t].first) * list.chunk;
    const Sum<ORDER> s = list.at[t].last & SRC_F32 ? chunk_sum<ORDER>(static_cast<const float *>(list.src[t]) + begin, n)
                                                   : chunk_sum<ORDER>(static_cast<const bf16_t *>(list.src[t]) + begin, n);
    const double total = group_total<ORDER, THREADS>(s);
    if (threadIdx.x == 0) partial[c] = total;
}

// joins the partial sums in a fixed order; total[0] = the norm in float64 (what grad_clip reads)
template <int ORDER> __global__ __launch_bounds__(JOIN) void join_kernel(const double *partial, int count, double scale, double *total, float *norm)
{
    Sum<ORDER> s, one;
    for (int i = threadIdx.x; i < count; i += JOIN) { one.set(partial[i]); s.join(one); }
    double v = group_total<ORDER, JOIN>(s);
    if (ORDER == GRAD_NORM_L2) v = sqrt(v);
    v *= scale;
    if (threadIdx.x == 0) { *total = v; *norm = (float)v; }
}

// (the stores are 16 bytes on 16-byte boundaries, consecutive over the lanes; the loads take what alignment is left)
template <typename S, typename D> __device__ __forceinline__ void scale_chunk(const S *src, D *dst, int n, float coef)
{
    constexpr int WIDE = sizeof(S) > sizeof(D) ? (int)sizeof(S) : (int)sizeof(D), VEC = 16 / WIDE, STEP = THREADS * VEC, DEEP = 4;
    const int lead = lead_of(dst, n);
    if ((int)threadIdx.x < lead) store_one(dst + threadIdx.x, load_one(src + threadIdx.x) * coef);
    src += lead;
    dst += lead;
    n -= lead;
    int i = threadIdx.x * VEC;
    for (; i + (DEEP - 1) * STEP + VEC <= n; i += DEEP * STEP) {
        float v[DEEP][VEC];
#pragma unroll
        for (int j = 0; j < DEEP; ++j) Run<S, VEC>::load(src + i + j * STEP, v[j]);
#pragma unroll
        for (int j = 0; j < DEEP; ++j) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[j][e] *= coef;
            Run<D, VEC>::store(dst + i + j * STEP, v[j]);
        }
    }
    for (; i + VEC <= n; i += STEP) {
        float v[VEC];
        Run<S, VEC>::load(src + i, v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] *= coef;
        Run<D, VEC>::store(dst + i, v);
    }
    const int rest = n & ~(VEC - 1);
    if (rest + (int)threadIdx.x < n) store_one(dst + rest + threadIdx.x, load_one(src + rest + threadIdx.x) * coef);
}

__global__ __launch_bounds__(THREADS) void clip_kernel(ClipList list, const double *total, double max_norm, double scale)
{
    const double ratio = max_norm / (*total + 1e-6);
    const float coef = (float)(scale * (ratio >= 1.0 ? 1.0 : ratio));           // (a NaN ratio stays)
    const uint32_t c = list.chunks - 1 - blockIdx.x;                            // (last chunk first: see grad_clip)
    const int t = tensor_of(list, c), n = chunk_length(list, t, c);
    const uint32_t types = list.at[t].last;
    const bool sf = types & SRC_F32, df = types & DST_F32;
    if (coef == 1.f && list.src[t] == list.dst[t] && sf == df) return;          // in place, nothing to clip
    const int64_t begin = (int64_t)(c - list.at[t].first) * list.chunk;
    if (sf) {
        const float *src = static_cast<const float *>(list.src[t]) + begin;
        if (df) scale_chunk(src, static_cast<float *>(list.dst[t]) + begin, n, coef);
        else scale_chunk(src, static_cast<bf16_t *>(list.dst[t]) + begin, n, coef);
    } else {
        const bf16_t *src = static_cast<const bf16_t *>(list.src[t]) + begin;
        if (df) scale_chunk(src, static_cast<float *>(list.dst[t]) + begin, n, coef);
        else scale_chunk(src, static_cast<bf16_t *>(list.dst[t]) + begin, n, coef);
    }
}

// elements per chunk: at most CHUNKS chunks and one per tensor
int64_t chunk_of(int64_t total)
{
    return (total / CHUNKS + GRAIN) / GRAIN * GRAIN;
}

int check(const void *const *src, const int64_t *numel, const uint8_t *types, int n, int64_t &total)
{
    total = 0;
    if (n < 0 || n > (1 << 20)) return MSDA_ERR_BAD_SHAPE;
    if (n == 0) return MSDA_OK;
    if (!src || !numel || !types) return MSDA_ERR_NULL_POINTER;
    for (int i = 0; i < n; ++i) {
        if (numel[i] < 0 || numel[i] > ((int64_t)1 << 40) - total) return MSDA_ERR_BAD_SHAPE;
        if (types[i] != MSDA_F32 && types[i] != MSDA_BF16) return MSDA_ERR_BAD_DTYPE;
        if (numel[i] > 0) {
            if (!src[i]) return MSDA_ERR_NULL_POINTER;
            if (reinterpret_cast<uintptr_t>(src[i]) % (types[i] == MSDA_F32 ? 4 : 2)) return MSDA_ERR_ALIGNMENT;
        }
        total += numel[i];
    }
    return MSDA_OK;
}

}  // namespace

extern "C" size_t grad_norm_workspace_bytes(int n) { return n > 0 ? ((size_t)CHUNKS + n + 2) * sizeof(double) : 2 * sizeof(double); }

extern "C" int grad_norm(const void *const *src, const uint8_t *src_types, const int64_t *numel, int n, int order, double grad_scale,
                         void *workspace, size_t workspace_bytes, float *norm, void *stream_)
{
    int64_t total;
    if (const int st = check(src, numel, src_types, n, total)) return st;
    if (order != GRAD_NORM_L1 && order != GRAD_NORM_L2 && order != GRAD_NORM_INF) return MSDA_ERR_BAD_VARIANT;
    if (!(grad_scale > 0.0) || !(grad_scale < __builtin_inf())) return MSDA_ERR_BAD_SHAPE;
    if (!workspace || !norm || workspace_bytes < grad_norm_workspace_bytes(n)) return MSDA_ERR_NULL_POINTER;
    if (reinterpret_cast<uintptr_t>(workspace) % 8) return MSDA_ERR_ALIGNMENT;
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    (void)hipGetLastError();                  // (an error that an earlier call left is not this one's)
    double *joined = static_cast<double *>(workspace), *partial = joined + 1;
    const int64_t chunk = chunk_of(total);
    NormList list;
    list.n = 0;
    list.chunk = (uint32_t)chunk;
    list.chunks = 0;
    int count = 0;
    const auto flush = [&] {
        if (list.n == 0) return;
        double *at = partial + count;
        const dim3 grid(list.chunks);
        if (order == GRAD_NORM_L1) hipLaunchKernelGGL(norm_kernel<GRAD_NORM_L1>, grid, dim3(THREADS), 0, stream, list, at);
        else if (order == GRAD_NORM_L2) hipLaunchKernelGGL(norm_kernel<GRAD_NORM_L2>, grid, dim3(THREADS), 0, stream, list, at);
        else hipLaunchKernelGGL(norm_kernel<GRAD_NORM_INF>, grid, dim3(THREADS), 0, stream, list, at);
        count += (int)list.chunks;
        list.n = 0;
        list.chunks = 0;
    };
    for (int i = 0; i < n; ++i) {
        if (numel[i] == 0) continue;
        const int64_t chunks = (numel[i] + chunk - 1) / chunk;
        list.src[list.n] = src[i];
        list.at[list.n] = {list.chunks, (uint32_t)(numel[i] - (chunks - 1) * chunk) | (src_types[i] == MSDA_F32 ? SRC_F32 : 0)};
        list.chunks += (uint32_t)chunks;
        if (++list.n == NORM_LIST) flush();
    }
    flush();
    if (order == GRAD_NORM_L1) hipLaunchKernelGGL(join_kernel<GRAD_NORM_L1>, dim3(1), dim3(JOIN), 0, stream, partial, count, grad_scale, joined, norm);
    else if (order == GRAD_NORM_L2) hipLaunchKernelGGL(join_kernel<GRAD_NORM_L2>, dim3(1), dim3(JOIN), 0, stream, partial, count, grad_scale, joined, norm);
    else hipLaunchKernelGGL(join_kernel<GRAD_NORM_INF>, dim3(1), dim3(JOIN), 0, stream, partial, count, grad_scale, joined, norm);
    return hipGetLastError() == hipSuccess ? MSDA_OK : MSDA_ERR_LAUNCH;
}

extern "C" int grad_clip(const void *const *src, const uint8_t *src_types, void *const *dst, const uint8_t *dst_types,
                         const int64_t *numel, int n, double max_norm, double grad_scale, const void *workspace, void *stream_)
{
    int64_t total;
    if (int st = check(src, numel, src_types, n, total)) return st;
    if (int st = check(const_cast<const void *const *>(dst), numel, dst_types, n, total)) return st;
    if (!(max_norm >= 0.0) || !(grad_scale > 0.0) || !(grad_scale < __builtin_inf())) return MSDA_ERR_BAD_SHAPE;
    if (!workspace) return MSDA_ERR_NULL_POINTER;
    if (reinterpret_cast<uintptr_t>(workspace) % 8) return MSDA_ERR_ALIGNMENT;
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    (void)hipGetLastError();                  // (an error that an earlier call left is not this one's)
    const double *joined = static_cast<const double *>(workspace);
    const int64_t chunk = chunk_of(total);
    ClipList list;
    list.n = 0;
    list.chunk = (uint32_t)chunk;
    list.chunks = 0;
    const auto flush = [&] {
        if (list.n) hipLaunchKernelGGL(clip_kernel, dim3(list.chunks), dim3(THREADS), 0, stream, list, joined, max_norm, grad_scale);
        list.n = 0;
        list.chunks = 0;
    };
    // From the last tensor to the first: what the norm pass read last is still in the memory-side cache (256 MB).
    for (int end = n; end > 0;) {
        int begin = end, taken = 0;
        while (begin > 0 && taken < CLIP_LIST) taken += numel[--begin] != 0;
        for (int i = begin; i < end; ++i) {
            if (numel[i] == 0) continue;
            const int64_t chunks = (numel[i] + chunk - 1) / chunk;
            list.src[list.n] = src[i];
            list.dst[list.n] = dst[i];
            list.at[list.n++] = {list.chunks, (uint32_t)(numel[i] - (chunks - 1) * chunk) | (src_types[i] == MSDA_F32 ? SRC_F32 : 0) |
                                                  (dst_types[i] == MSDA_F32 ? DST_F32 : 0)};
            list.chunks += (uint32_t)chunks;
        }
        flush();
        end = begin;
    }
    return hipGetLastError() == hipSuccess ? MSDA_OK : MSDA_ERR_LAUNCH;
}
