// group.hip - norms over many arrays at once: the global norm of an instance over all arrays of a list, clipping to it, and the
// bounded step new <- old + min(1, max / |new - old|) (new - old) of a whole set of EP messages.
//
// The arrays of a list have lengths of their own, [batch, n_i] each; an instance b owns row b of every array.  The list is laid
// out once as chunks of kChunk elements that never straddle two arrays; workgroup p of instance b walks the chunks p, p + P, ...
// and leaves one partial sum of squares, the second launch adds the P partials of its instance in a fixed order (every
// workgroup for itself: P <= 1024 doubles out of the L2) and applies the factor.  Sums are held in double: no overflow below
// 1e154, no loss in long sums, and the same bits every time.
#include "common.h"

#include <algorithm>
#include <new>
#include <vector>

namespace {
constexpr size_t kChunk = 4096;
constexpr int kMaxPartials = 1024;
}  // namespace

struct tramp_group {
    int device;
    int dtype;
    int k;
    size_t batch;
    size_t nchunk;
    void* mem;
    void* const* ptr;            // [k] device pointers
    const size_t* len;           // [k]
    const int* chunk_array;      // [nchunk] the array a chunk belongs to
    const unsigned* first;       // [k] the first chunk of every array
    void** ptr_h;                // host copies (checks between lists)
    size_t* len_h;
};

struct GroupDev {
    void* const* ptr;
    const size_t* len;
    const int* chunk_array;
    const unsigned* first;
    unsigned nchunk;
};

static GroupDev dev_of(const tramp_group* g) { return GroupDev{g->ptr, g->len, g->chunk_array, g->first, (unsigned)g->nchunk}; }

// partial sums of squares of x (STEP = false) or of x - prev
template <typename T, bool STEP>
__global__ __launch_bounds__(kBlock) void group_squares_kernel(GroupDev g, void* const* __restrict__ prev, double* __restrict__ partials) {
    __shared__ double smem[kBlock / kWave];
    const size_t b = blockIdx.y;
    double acc = 0.0;
    for (unsigned c = blockIdx.x; c < g.nchunk; c += gridDim.x) {
        const int i = g.chunk_array[c];
        const size_t n = g.len[i], lo = (size_t)(c - g.first[i]) * kChunk, hi = lo + kChunk < n ? lo + kChunk : n;
        const T* x = static_cast<const T*>(g.ptr[i]) + b * n;
        const T* p = STEP ? static_cast<const T*>(prev[i]) + b * n : nullptr;
        for (size_t j = lo + threadIdx.x; j < hi; j += kBlock) {
            const double d = STEP ? (double)x[j] - (double)p[j] : (double)x[j];
            acc += d * d;
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

// out = c x, or out = prev + c (x - prev) with the precisions a moved by the same factor; REFRESH writes the result over prev too
template <typename T, bool STEP>
__global__ __launch_bounds__(kBlock) void group_apply_kernel(GroupDev g, void* const* prev, void* const* out, int refresh, double bound,
                                                             const double* __restrict__ partials, int P, size_t n_a, size_t B, double* a,
                                                             double* a_prev, double* __restrict__ norm_out) {
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
    for (unsigned ch = blockIdx.x; ch < g.nchunk; ch += gridDim.x) {
        const int i = g.chunk_array[ch];
        const size_t n = g.len[i], lo = (size_t)(ch - g.first[i]) * kChunk, hi = lo + kChunk < n ? lo + kChunk : n;
        const T* x = static_cast<const T*>(g.ptr[i]) + b * n;
        T* p = STEP ? static_cast<T*>(prev[i]) + b * n : nullptr;
        T* o = static_cast<T*>(out[i]) + b * n;
        if (c == 1.0 && o == x && !(STEP && refresh)) continue;
        for (size_t j = lo + threadIdx.x; j < hi; j += kBlock) {
            T r = x[j];
            if (c < 1.0) r = STEP ? T((double)p[j] + c * ((double)r - (double)p[j])) : T(c * (double)r);
            o[j] = r;
            if (STEP && refresh) p[j] = r;
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
    const size_t e = dtype_size(dtype);
    try {
        size_t nchunk = 0;
        std::vector<std::pair<uintptr_t, uintptr_t>> span;
        for (int i = 0; i < k; ++i) {
            TRAMP_REQUIRE(ctx, arrays_d[i] || !n[i]);
            TRAMP_REQUIRE(ctx, n[i] <= ((size_t)1 << 40) / batch);
            nchunk += (n[i] + kChunk - 1) / kChunk;
            const uintptr_t a = (uintptr_t)arrays_d[i];
            if (n[i]) span.emplace_back(a, a + n[i] * batch * e);
        }
        TRAMP_REQUIRE(ctx, nchunk < 0x7fffffffu);
        std::sort(span.begin(), span.end());
        for (size_t i = 1; i < span.size(); ++i)
            if (span[i].first < span[i - 1].second)
                return tramp_fail(ctx, TRAMP_EINVAL, "tramp_group_create", "two arrays of the list overlap");
        std::vector<int> chunk_array;
        std::vector<unsigned> first((size_t)k);
        chunk_array.reserve(nchunk);
        for (int i = 0; i < k; ++i) {
            first[(size_t)i] = (unsigned)chunk_array.size();
            chunk_array.insert(chunk_array.end(), (n[i] + kChunk - 1) / kChunk, i);
        }
        auto up = [](size_t bytes) { return (bytes + 255) & ~(size_t)255; };
        const size_t o_len = up((size_t)k * 8), o_first = o_len + up((size_t)k * 8), o_chunk = o_first + up((size_t)k * 4);
        const size_t total = o_chunk + up(nchunk * 4);
        std::vector<char> host(total, 0);
        memcpy(host.data(), arrays_d, (size_t)k * 8);
        memcpy(host.data() + o_len, n, (size_t)k * 8);
        memcpy(host.data() + o_first, first.data(), (size_t)k * 4);
        if (nchunk) memcpy(host.data() + o_chunk, chunk_array.data(), nchunk * 4);
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
        hipError_t err = hipMemcpyAsync(g->mem, host.data(), total, hipMemcpyHostToDevice, ctx->stream);
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
        char* m = static_cast<char*>(g->mem);
        g->device = ctx->device;
        g->dtype = dtype;
        g->k = k;
        g->batch = batch;
        g->nchunk = nchunk;
        g->ptr = reinterpret_cast<void* const*>(m);
        g->len = reinterpret_cast<const size_t*>(m + o_len);
        g->first = reinterpret_cast<const unsigned*>(m + o_first);
        g->chunk_array = reinterpret_cast<const int*>(m + o_chunk);
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
    hipLaunchKernelGGL((group_squares_kernel<T, STEP>), grid, dim3(kBlock), 0, ctx->stream, dev_of(g), STEP ? prev->ptr : nullptr, ctx->ws);
    if (!out)
        hipLaunchKernelGGL(group_norm_kernel, dim3((unsigned)g->batch), dim3(kBlock), 0, ctx->stream, ctx->ws, P, norm_d);
    else
        hipLaunchKernelGGL((group_apply_kernel<T, STEP>), grid, dim3(kBlock), 0, ctx->stream, dev_of(g), STEP ? prev->ptr : nullptr, out->ptr,
                           refresh, bound, ctx->ws, P, n_a, g->batch, a, a_prev, norm_d);
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
