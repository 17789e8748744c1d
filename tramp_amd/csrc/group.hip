// group.hip - norms over many arrays at once: the global norm of an instance over all arrays of a list, clipping to it, and the
// bounded step new <- old + min(1, max / |new - old|) (new - old) of a whole set of EP messages.
//
// The arrays of a list have lengths of their own, [batch, n_i] each; an instance b owns row b of every array.  The list is laid
// out once as chunks of 32 KiB that never straddle two arrays; workgroup p of instance b walks the chunks p, p + P, ... and
// leaves one partial sum of squares, the second launch adds the P partials of its instance in a fixed order (every workgroup
// for itself: P <= 2048 doubles out of the L2) and applies the factor, from the last chunk to the first: what the first pass
// read last is still in the 256 MB of cache before memory.  Sums are held in double: no overflow below 1e154, no loss in long
// sums, and the same bits every time.
#include "common.h"

#include <algorithm>
#include <new>
#include <vector>

namespace {
constexpr size_t kChunkBytes = 32768;                // 8 pieces of 16 bytes per thread
constexpr int kPieces = kChunkBytes / 16 / kBlock;
constexpr int kMaxPartials = 2048;
}  // namespace

// one chunk: everything a workgroup needs in one scalar load, the next one's is on its way while this one is worked on
struct GroupChunk {
    unsigned long long addr;     // of its first element, instance 0
    unsigned long long stride;   // bytes from one instance to the next
    unsigned long long len;      // elements
};

struct tramp_group {
    int device;
    int dtype;
    int k;
    size_t batch;
    size_t nchunk;
    void* mem;
    const GroupChunk* chunks;    // [nchunk]; lists of the same lengths have the same chunks
    void** ptr_h;                // host copies (checks between lists)
    size_t* len_h;
};

// 16-byte pieces at any element boundary
template <typename T> struct GVec;
template <> struct GVec<float> {
    typedef float U __attribute__((ext_vector_type(4), aligned(4)));
    static constexpr int N = 4;
};
template <> struct GVec<double> {
    typedef double U __attribute__((ext_vector_type(2), aligned(8)));
    static constexpr int N = 2;
};

// partial sums of squares of x (STEP = false) or of x - prev
template <typename T, bool STEP>
__global__ __launch_bounds__(kBlock) void group_squares_kernel(unsigned nchunk, const GroupChunk* __restrict__ xs, const GroupChunk* __restrict__ ps,
                                                               double* __restrict__ partials) {
    using U = typename GVec<T>::U;
    constexpr int N = GVec<T>::N;
    constexpr size_t CH = kChunkBytes / sizeof(T);
    __shared__ double smem[kBlock / kWave];
    const size_t b = blockIdx.y;
    double acc = 0.0;
    for (unsigned c = blockIdx.x; c < nchunk; c += gridDim.x) {
        const T* x = reinterpret_cast<const T*>(xs[c].addr + b * xs[c].stride);
        const T* p = STEP ? reinterpret_cast<const T*>(ps[c].addr + b * ps[c].stride) : nullptr;
        const size_t len = xs[c].len;
        if (len == CH) {
            U v[kPieces], w[kPieces];
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                v[i] = reinterpret_cast<const U*>(x)[i * kBlock + threadIdx.x];
                if (STEP) w[i] = reinterpret_cast<const U*>(p)[i * kBlock + threadIdx.x];
            }
#pragma unroll
            for (int i = 0; i < kPieces; ++i)
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    const double d = STEP ? (double)v[i][e] - (double)w[i][e] : (double)v[i][e];
                    acc = fma(d, d, acc);
                }
        } else {
            for (size_t j = threadIdx.x; j < len; j += kBlock) {
                const double d = STEP ? (double)x[j] - (double)p[j] : (double)x[j];
                acc = fma(d, d, acc);
            }
        }
    }
    acc = block_sum(acc, smem);
    if (threadIdx.x == 0) partials[b * gridDim.x + blockIdx.x] = acc;
}

__device__ __forceinline__ double fold_norm(const double* __restrict__ partials, int P, size_t b, double* smem) {
    double acc = 0.0;
    for (int i = threadIdx.x; i < P; i += kBlock) acc += partials[b * (size_t)P + i];
    return sqrt(block_sum(acc, smem));
}

// min(1, max / norm); a norm that is zero or not finite leaves the instance alone (its NaN guard sees it)
__device__ __forceinline__ double clip_factor(double norm, double bound) {
    return (norm > bound && norm <= 1.7976931348623157e308) ? bound / norm : 1.0;
}

__global__ __launch_bounds__(kBlock) void group_norm_kernel(const double* __restrict__ partials, int P, double* __restrict__ norm_out) {
    __shared__ double smem[kBlock / kWave];
    const double n = fold_norm(partials, P, blockIdx.x, smem);
    if (threadIdx.x == 0) norm_out[blockIdx.x] = n;
}

template <typename T, bool STEP> __device__ __forceinline__ T bounded(T x, T p, double c) {
    if (c == 1.0) return x;
    return STEP ? T((double)p + c * ((double)x - (double)p)) : T(c * (double)x);
}

// out = c x, or out = prev + c (x - prev) with the precisions a moved by the same factor; refresh: the result over prev too
template <typename T, bool STEP>
__global__ __launch_bounds__(kBlock) void group_apply_kernel(unsigned nchunk, const GroupChunk* __restrict__ xs, const GroupChunk* __restrict__ ps,
                                                             const GroupChunk* __restrict__ os, int refresh, double bound,
                                                             const double* __restrict__ partials, int P, size_t n_a, size_t B, double* a,
                                                             double* a_prev, double* __restrict__ norm_out) {
    using U = typename GVec<T>::U;
    constexpr int N = GVec<T>::N;
    constexpr size_t CH = kChunkBytes / sizeof(T);
    __shared__ double smem[kBlock / kWave];
    const size_t b = blockIdx.y;
    const double norm = fold_norm(partials, P, b, smem), c = clip_factor(norm, bound);
    if (blockIdx.x == 0) {
        if (threadIdx.x == 0 && norm_out) norm_out[b] = norm;
        if (STEP)
            for (size_t i = threadIdx.x; i < n_a; i += kBlock) {
                const double o = a_prev[i * B + b];
                const double r = c < 1.0 ? o + c * (a[i * B + b] - o) : a[i * B + b];
                a[i * B + b] = r;
                if (refresh) a_prev[i * B + b] = r;
            }
    }
    for (unsigned k = blockIdx.x; k < nchunk; k += gridDim.x) {
        const unsigned ch = nchunk - 1 - k;
        const T* x = reinterpret_cast<const T*>(xs[ch].addr + b * xs[ch].stride);
        T* p = STEP ? reinterpret_cast<T*>(ps[ch].addr + b * ps[ch].stride) : nullptr;
        T* o = reinterpret_cast<T*>(os[ch].addr + b * os[ch].stride);
        const size_t len = xs[ch].len;
        if (c == 1.0 && o == x && !(STEP && refresh)) continue;
        if (len == CH) {
            U v[kPieces], w[kPieces];
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                v[i] = reinterpret_cast<const U*>(x)[i * kBlock + threadIdx.x];
                if (STEP) w[i] = reinterpret_cast<const U*>(p)[i * kBlock + threadIdx.x];
            }
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
#pragma unroll
                for (int e = 0; e < N; ++e) v[i][e] = bounded<T, STEP>(v[i][e], STEP ? w[i][e] : T(0), c);
                reinterpret_cast<U*>(o)[i * kBlock + threadIdx.x] = v[i];
                if (STEP && refresh) reinterpret_cast<U*>(p)[i * kBlock + threadIdx.x] = v[i];
            }
        } else {
            for (size_t j = threadIdx.x; j < len; j += kBlock) {
                const T r = bounded<T, STEP>(x[j], STEP ? p[j] : T(0), c);
                o[j] = r;
                if (STEP && refresh) p[j] = r;
            }
        }
    }
}

// ---------------------------------------------------------------- handle
static size_t elem_size(const tramp_group* g) { return dtype_size(g->dtype); }

extern "C" int tramp_group_create(tramp_ctx* ctx, int dtype, int k, void* const* arrays_d, const size_t* n, size_t batch, tramp_group** out) {
    if (!ctx || !out) return TRAMP_EINVAL;
    *out = nullptr;
    TRAMP_REQUIRE(ctx, dtype == TRAMP_F32 || dtype == TRAMP_F64);
    TRAMP_REQUIRE(ctx, k >= 1 && arrays_d && n && batch >= 1 && batch <= 65535);
    TRAMP_REQUIRE(ctx, !ctx->capturing);
    const size_t e = dtype_size(dtype), per = kChunkBytes / e;
    try {
        size_t nchunk = 0;
        std::vector<std::pair<uintptr_t, uintptr_t>> span;
        for (int i = 0; i < k; ++i) {
            TRAMP_REQUIRE(ctx, arrays_d[i] || !n[i]);
            TRAMP_REQUIRE(ctx, n[i] <= ((size_t)1 << 40) / batch);
            nchunk += (n[i] + per - 1) / per;
            const uintptr_t a = (uintptr_t)arrays_d[i];
            if (n[i]) span.emplace_back(a, a + n[i] * batch * e);
        }
        TRAMP_REQUIRE(ctx, nchunk < 0x7fffffffu);
        std::sort(span.begin(), span.end());
        for (size_t i = 1; i < span.size(); ++i)
            if (span[i].first < span[i - 1].second)
                return tramp_fail(ctx, TRAMP_EINVAL, "tramp_group_create", "two arrays of the list overlap");
        std::vector<GroupChunk> chunks;
        chunks.reserve(nchunk);
        for (int i = 0; i < k; ++i)
            for (size_t lo = 0; lo < n[i]; lo += per)
                chunks.push_back(GroupChunk{(unsigned long long)(uintptr_t)arrays_d[i] + lo * e, (unsigned long long)(n[i] * e),
                                            (unsigned long long)std::min(per, n[i] - lo)});
        const size_t total = std::max(nchunk, (size_t)1) * sizeof(GroupChunk);
        chunks.resize(std::max(nchunk, (size_t)1));
        tramp_group* g = new tramp_group();
        *g = tramp_group{};
        g->ptr_h = static_cast<void**>(malloc((size_t)k * 8));
        g->len_h = static_cast<size_t*>(malloc((size_t)k * 8));
        (void)hipSetDevice(ctx->device);
        if (!g->ptr_h || !g->len_h || hipMalloc(&g->mem, total) != hipSuccess) {
            (void)hipGetLastError();
            free(g->ptr_h);
            free(g->len_h);
            delete g;
            return tramp_fail(ctx, TRAMP_ENOMEM, "tramp_group_create", "out of memory");
        }
        hipError_t err = hipMemcpyAsync(g->mem, chunks.data(), total, hipMemcpyHostToDevice, ctx->stream);
        if (err == hipSuccess) err = hipStreamSynchronize(ctx->stream);
        if (err != hipSuccess) {
            (void)hipFree(g->mem);
            free(g->ptr_h);
            free(g->len_h);
            delete g;
            return tramp_fail(ctx, TRAMP_EHIP, "tramp_group_create", hipGetErrorString(err));
        }
        memcpy(g->ptr_h, arrays_d, (size_t)k * 8);
        memcpy(g->len_h, n, (size_t)k * 8);
        g->device = ctx->device;
        g->dtype = dtype;
        g->k = k;
        g->batch = batch;
        g->nchunk = nchunk;
        g->chunks = static_cast<const GroupChunk*>(g->mem);
        *out = g;
        return TRAMP_OK;
    } catch (const std::bad_alloc&) {
        return tramp_fail(ctx, TRAMP_ENOMEM, "tramp_group_create", "host memory");
    }
}

extern "C" int tramp_group_destroy(tramp_ctx* ctx, tramp_group* g) {
    if (!ctx || !g) return TRAMP_EINVAL;
    (void)hipStreamSynchronize(ctx->stream);
    (void)hipFree(g->mem);
    free(g->ptr_h);
    free(g->len_h);
    delete g;
    return TRAMP_OK;
}

// the same shapes, and every array of `o` either in the place of the same one of `g` (if `same` allows it) or clear of all of them
static int check_pair(tramp_ctx* ctx, const tramp_group* g, const tramp_group* o, bool same, const char* what) {
    if (o->device != g->device || o->dtype != g->dtype || o->k != g->k || o->batch != g->batch)
        return tramp_fail(ctx, TRAMP_EINVAL, what, "lists of different lengths, types, instances or devices");
    const size_t e = elem_size(g);
    for (int i = 0; i < g->k; ++i)
        if (o->len_h[i] != g->len_h[i]) return tramp_fail(ctx, TRAMP_EINVAL, what, "arrays of different lengths");
    if (g == o) return same ? TRAMP_OK : tramp_fail(ctx, TRAMP_EINVAL, what, "the same list twice");
    try {
        std::vector<std::pair<uintptr_t, uintptr_t>> span;
        for (int i = 0; i < g->k; ++i)
            if (g->len_h[i]) span.emplace_back((uintptr_t)g->ptr_h[i], (uintptr_t)g->ptr_h[i] + g->len_h[i] * g->batch * e);
        std::sort(span.begin(), span.end());
        for (int i = 0; i < g->k; ++i) {
            if (!g->len_h[i] || (same && o->ptr_h[i] == g->ptr_h[i])) continue;
            const uintptr_t lo = (uintptr_t)o->ptr_h[i], hi = lo + g->len_h[i] * g->batch * e;
            auto it = std::upper_bound(span.begin(), span.end(), std::make_pair(hi - 1, (uintptr_t)-1));
            if (it != span.begin() && std::prev(it)->second > lo)
                return tramp_fail(ctx, TRAMP_EINVAL, what, "the arrays of the two lists overlap");
        }
    } catch (const std::bad_alloc&) {
        return tramp_fail(ctx, TRAMP_ENOMEM, what, "host memory");
    }
    return TRAMP_OK;
}

static int partials_of(const tramp_group* g) {
    return (int)(g->nchunk < 1 ? 1 : g->nchunk > (size_t)kMaxPartials ? (size_t)kMaxPartials : g->nchunk);
}

template <typename T, bool STEP>
static int group_run(tramp_ctx* ctx, const tramp_group* g, const tramp_group* prev, const tramp_group* out, int refresh, double bound,
                     size_t n_a, double* a, double* a_prev, double* norm_d) {
    const int P = partials_of(g);
    int rc = tramp_ws_reserve(ctx, g->batch * (size_t)P * sizeof(double));
    if (rc) return rc;
    dim3 grid((unsigned)P, (unsigned)g->batch);
    hipLaunchKernelGGL((group_squares_kernel<T, STEP>), grid, dim3(kBlock), 0, ctx->stream, (unsigned)g->nchunk, g->chunks,
                       STEP ? prev->chunks : nullptr, ctx->ws);
    if (!out)
        hipLaunchKernelGGL(group_norm_kernel, dim3((unsigned)g->batch), dim3(kBlock), 0, ctx->stream, ctx->ws, P, norm_d);
    else
        hipLaunchKernelGGL((group_apply_kernel<T, STEP>), grid, dim3(kBlock), 0, ctx->stream, (unsigned)g->nchunk, g->chunks,
                           STEP ? prev->chunks : nullptr, out->chunks, refresh, bound, ctx->ws, P, n_a, g->batch, a, a_prev, norm_d);
    TRAMP_LAUNCH_CHECK(ctx);
    return TRAMP_OK;
}

extern "C" int tramp_group_norm(tramp_ctx* ctx, const tramp_group* g, double* norm_d) {
    if (!ctx) return TRAMP_EINVAL;
    TRAMP_REQUIRE(ctx, g && norm_d && g->device == ctx->device);
    return g->dtype == TRAMP_F64 ? group_run<double, false>(ctx, g, nullptr, nullptr, 0, 0.0, 0, nullptr, nullptr, norm_d)
                                 : group_run<float, false>(ctx, g, nullptr, nullptr, 0, 0.0, 0, nullptr, nullptr, norm_d);
}

extern "C" int tramp_group_clip(tramp_ctx* ctx, const tramp_group* g, double max_norm, const tramp_group* out, double* norm_d) {
    if (!ctx) return TRAMP_EINVAL;
    TRAMP_REQUIRE(ctx, g && out && g->device == ctx->device);
    TRAMP_REQUIRE(ctx, max_norm > 0.0);
    int rc = check_pair(ctx, g, out, true, "tramp_group_clip");
    if (rc) return rc;
    return g->dtype == TRAMP_F64 ? group_run<double, false>(ctx, g, nullptr, out, 0, max_norm, 0, nullptr, nullptr, norm_d)
                                 : group_run<float, false>(ctx, g, nullptr, out, 0, max_norm, 0, nullptr, nullptr, norm_d);
}

extern "C" int tramp_group_limit_step(tramp_ctx* ctx, const tramp_group* g, const tramp_group* prev, double max_step,
                                      const tramp_group* out, int refresh, size_t n_a, double* a_d, double* a_prev_d, double* norm_d) {
    if (!ctx) return TRAMP_EINVAL;
    TRAMP_REQUIRE(ctx, g && prev && out && g->device == ctx->device);
    TRAMP_REQUIRE(ctx, max_step > 0.0);
    TRAMP_REQUIRE(ctx, n_a == 0 || (a_d && a_prev_d));
    TRAMP_REQUIRE(ctx, n_a == 0 || a_d + n_a * g->batch <= a_prev_d || a_prev_d + n_a * g->batch <= a_d);
    int rc = check_pair(ctx, g, prev, false, "tramp_group_limit_step");
    if (!rc) rc = check_pair(ctx, g, out, true, "tramp_group_limit_step");
    if (!rc) rc = check_pair(ctx, prev, out, false, "tramp_group_limit_step");
    if (rc) return rc;
    return g->dtype == TRAMP_F64 ? group_run<double, true>(ctx, g, prev, out, refresh, max_step, n_a, a_d, a_prev_d, norm_d)
                                 : group_run<float, true>(ctx, g, prev, out, refresh, max_step, n_a, a_d, a_prev_d, norm_d);
}
