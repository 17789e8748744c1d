// group.hip - norms over many arrays at once: the global norm of an instance over all arrays of a list, clipping to it, and the
// bounded step new <- old + min(1, max / |new - old|) (new - old) of a whole set of EP messages.
//
// The arrays of a list have lengths of their own, [batch, n_i] each; an instance b owns row b of every array.  The list is laid
// out once as chunks of 16 KiB that never straddle two arrays; workgroup p of instance b walks the chunks p, p + P, ... and
// leaves one partial sum of squares, the second launch adds the P partials of its instance in a fixed order (every workgroup
// for itself: P <= 2048 doubles out of the L2) and applies the factor, from the last chunk to the first: what the first pass
// read last is still in the 256 MB of cache before memory.  Sums are held in double: no loss in long sums, and the same bits every
// time.  Squares of f64 beyond 1e154 are infinite (such an instance stays as it is), below 1e-162 they are 0.
#include "common.h"

#include <algorithm>
#include <new>
#include <vector>

namespace {
constexpr size_t kChunkBytes = 16384;                // 4 pieces of 16 bytes per thread
constexpr int kPieces = kChunkBytes / 16 / kBlock;
// Up to this many chunks one workgroup does both passes of an instance, in one launch: 4 arrays of 1000 f64 together 5.4 against
// 7.6 us, of 3000 6.3 against 7.9 us; 12000 (six chunks) would be 11.8 against 7.6 us.  A chunk never straddles two arrays, so five
// arrays take two launches however short they are (not measured against one).
constexpr size_t kSmall = 4;
// workgroups of a pass: 8 per CU; 1280 and 4096 time the same within 4 % (24 arrays of 10^9 bytes), 1280 loses 20 % on 64
// instances
constexpr size_t kBlocks = 2048;
// Lists larger than this are gone from the cache before anyone reads the result: the second pass reads and writes past it.
// 10^9 bytes 559 -> 494 us, 64 instances x 300000 f64 with their previous values 140 -> 130 us, 16 x 3000000 f32 112 -> 101 us;
// 20 MB 14.4 -> 15.3 us.
constexpr size_t kOnce = (size_t)128 << 20;
// Slices of instances (group_run): 64 instances x 300000 f64 and their previous values, 307 MB, in slices of 80 MB 140 us, of
// 48 MB 151 us, of 128 MB 143 us, whole 152 us.
constexpr size_t kSlice = (size_t)80 << 20;
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
    // host copies for the checks between lists: the arrays in order, and where they lie, sorted
    void** ptr_h;
    size_t* len_h;
    struct Span { uintptr_t lo, hi; }* span;
    int n_span;
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

// ONCE: past the caches, for what will not be touched again before it is gone from them
template <typename T, bool ONCE> __device__ __forceinline__ typename GVec<T>::U g_load(const T* p, unsigned j) {
    using U = typename GVec<T>::U;
    return ONCE ? __builtin_nontemporal_load(reinterpret_cast<const U*>(p) + j) : reinterpret_cast<const U*>(p)[j];
}
template <typename T, bool ONCE> __device__ __forceinline__ void g_store(T* p, unsigned j, typename GVec<T>::U v) {
    using U = typename GVec<T>::U;
    if (ONCE)
        __builtin_nontemporal_store(v, reinterpret_cast<U*>(p) + j);
    else
        reinterpret_cast<U*>(p)[j] = v;
}

// sum of squares of a chunk of x (STEP = false) or of x - prev, this thread's share
template <typename T, bool STEP>
__device__ __forceinline__ double chunk_squares(const GroupChunk* __restrict__ xs, const GroupChunk* __restrict__ ps, size_t b) {
    using U = typename GVec<T>::U;
    constexpr int N = GVec<T>::N;
    const T* x = reinterpret_cast<const T*>(xs->addr + b * xs->stride);
    const T* p = STEP ? reinterpret_cast<const T*>(ps->addr + b * ps->stride) : nullptr;
    const unsigned len = xs->len, full = len / N;
    U v[kPieces], w[kPieces];
    double acc = 0.0;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        const unsigned j = i * kBlock + threadIdx.x;
        if (j < full) {
            v[i] = reinterpret_cast<const U*>(x)[j];
            if (STEP) w[i] = reinterpret_cast<const U*>(p)[j];
        }
    }
    const unsigned r = full * N + threadIdx.x;                     // fewer than N elements behind the whole pieces
    if (r < len) {
        const double d = STEP ? (double)x[r] - (double)p[r] : (double)x[r];
        acc = fma(d, d, acc);
    }
#pragma unroll
    for (int i = 0; i < kPieces; ++i)
        if (i * kBlock + threadIdx.x < full) {
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const double d = STEP ? (double)v[i][e] - (double)w[i][e] : (double)v[i][e];
                acc = fma(d, d, acc);
            }
        }
    return acc;
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

// one chunk of out = c x, or of out = prev + c (x - prev); refresh: the result over prev too
template <typename T, bool STEP, bool ONCE>
__device__ __forceinline__ void chunk_apply(const GroupChunk* __restrict__ xs, const GroupChunk* __restrict__ ps,
                                            const GroupChunk* __restrict__ os, size_t b, int refresh, double c) {
    using U = typename GVec<T>::U;
    constexpr int N = GVec<T>::N;
    const T* x = reinterpret_cast<const T*>(xs->addr + b * xs->stride);
    T* p = STEP ? reinterpret_cast<T*>(ps->addr + b * ps->stride) : nullptr;
    T* o = reinterpret_cast<T*>(os->addr + b * os->stride);
    if (c == 1.0 && o == x && !(STEP && refresh)) return;
    const unsigned len = xs->len, full = len / N;
    U v[kPieces], w[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        const unsigned j = i * kBlock + threadIdx.x;
        if (j < full) {
            v[i] = g_load<T, ONCE>(x, j);
            if (STEP) w[i] = g_load<T, ONCE>(p, j);
        }
    }
    const unsigned r = full * N + threadIdx.x;
    if (r < len) {
        const T t = bounded<T, STEP>(x[r], STEP ? p[r] : T(0), c);
        o[r] = t;
        if (STEP && refresh) p[r] = t;
    }
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        const unsigned j = i * kBlock + threadIdx.x;
        if (j < full) {
#pragma unroll
            for (int e = 0; e < N; ++e) v[i][e] = bounded<T, STEP>(v[i][e], STEP ? w[i][e] : T(0), c);
            g_store<T, ONCE>(o, j, v[i]);
            if (STEP && refresh) g_store<T, ONCE>(p, j, v[i]);
        }
    }
}

// what goes with the arrays: the norm, the precisions a moved by the same factor
struct GroupSide {
    double bound;
    double* norm_out;
    double* a;
    double* a_prev;
    size_t n_a, batch;
    int refresh;
};
template <bool STEP> __device__ __forceinline__ void group_side(const GroupSide& q, size_t b, double norm, double c) {
    if (threadIdx.x == 0 && q.norm_out) q.norm_out[b] = norm;
    if (!STEP) return;
    for (size_t i = threadIdx.x; i < q.n_a; i += kBlock) {
        const double o = q.a_prev[i * q.batch + b], x = q.a[i * q.batch + b], d = x - o;
        const double r = c < 1.0 && d - d == 0.0 ? o + c * d : x;          // a step that is infinite or NaN is taken whole
        q.a[i * q.batch + b] = r;
        if (q.refresh) q.a_prev[i * q.batch + b] = r;
    }
}

// The two passes.  Bound by memory: x (and prev) twice, the second time from the cache as far as it reaches, out once.
// 10^9 bytes of f32 in 24 arrays clipped in place 495 us (2 GB at a copy's 5.14 TB/s: 389 us), 64 instances of 300000 f64 with their
// previous values 130 us (461 MB: 90 us), 20 MB in 41 arrays 15 us (7.8 us).  Rows y of the grid: the instances [a0, a0 + n_apply), whose sums an earlier launch has left, are finished;
// of the following ones the sums are taken.
template <typename T, bool STEP, bool ONCE>
__global__ __launch_bounds__(kBlock) void group_pass_kernel(unsigned nchunk, const GroupChunk* __restrict__ xs, const GroupChunk* __restrict__ ps,
                                                            const GroupChunk* __restrict__ os, size_t a0, unsigned n_apply, GroupSide q,
                                                            double* __restrict__ partials) {
    __shared__ double smem[kBlock / kWave];
    const size_t b = a0 + blockIdx.y;
    if (blockIdx.y >= n_apply) {
        double acc = 0.0;
        for (unsigned c = blockIdx.x; c < nchunk; c += gridDim.x) acc += chunk_squares<T, STEP>(xs + c, ps + c, b);
        acc = block_sum(acc, smem);
        if (threadIdx.x == 0) partials[b * gridDim.x + blockIdx.x] = acc;
        return;
    }
    const double norm = fold_norm(partials, gridDim.x, b, smem), c = clip_factor(norm, q.bound);
    if (blockIdx.x == 0) group_side<STEP>(q, b, norm, c);
    for (unsigned k = blockIdx.x; k < nchunk; k += gridDim.x) {
        const unsigned ch = nchunk - 1 - k;
        chunk_apply<T, STEP, ONCE>(xs + ch, ps + ch, os + ch, b, q.refresh, c);
    }
}

// small instances: one workgroup each does both passes in one launch; bound by its latency (4 arrays, 3000 f64 in all: 6.2 us)
template <typename T, bool STEP>
__global__ __launch_bounds__(kBlock) void group_small_kernel(unsigned nchunk, const GroupChunk* __restrict__ xs, const GroupChunk* __restrict__ ps,
                                                             const GroupChunk* __restrict__ os, GroupSide q) {
    __shared__ double smem[kBlock / kWave];
    const size_t b = blockIdx.x;
    double acc = 0.0;
    for (unsigned c = 0; c < nchunk; ++c) acc += chunk_squares<T, STEP>(xs + c, ps + c, b);
    const double norm = sqrt(block_sum(acc, smem)), c = clip_factor(norm, q.bound);
    group_side<STEP>(q, b, norm, c);
    if (!os) return;
    for (unsigned k = 0; k < nchunk; ++k) chunk_apply<T, STEP, false>(xs + k, ps + k, os + k, b, q.refresh, c);
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
        std::vector<tramp_group::Span> span;
        for (int i = 0; i < k; ++i) {
            TRAMP_REQUIRE(ctx, arrays_d[i] || !n[i]);
            TRAMP_REQUIRE(ctx, n[i] <= ((size_t)1 << 40) / batch);
            nchunk += (n[i] + per - 1) / per;
            const uintptr_t a = (uintptr_t)arrays_d[i];
            if (n[i]) span.push_back({a, a + n[i] * batch * e});
        }
        TRAMP_REQUIRE(ctx, nchunk < 0x7fffffffu);
        std::sort(span.begin(), span.end(), [](const tramp_group::Span& a, const tramp_group::Span& b) { return a.lo < b.lo; });
        for (size_t i = 1; i < span.size(); ++i)
            if (span[i].lo < span[i - 1].hi)
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
        g->span = static_cast<tramp_group::Span*>(malloc((size_t)k * sizeof(tramp_group::Span)));
        (void)hipSetDevice(ctx->device);
        if (!g->ptr_h || !g->len_h || !g->span || hipMalloc(&g->mem, total) != hipSuccess) {
            (void)hipGetLastError();
            free(g->ptr_h);
            free(g->len_h);
            free(g->span);
            delete g;
            return tramp_fail(ctx, TRAMP_ENOMEM, "tramp_group_create", "out of memory");
        }
        hipError_t err = hipMemcpyAsync(g->mem, chunks.data(), total, hipMemcpyHostToDevice, ctx->stream);
        if (err == hipSuccess) err = hipStreamSynchronize(ctx->stream);
        if (err != hipSuccess) {
            (void)hipFree(g->mem);
            free(g->ptr_h);
            free(g->len_h);
            free(g->span);
            delete g;
            return tramp_fail(ctx, TRAMP_EHIP, "tramp_group_create", hipGetErrorString(err));
        }
        memcpy(g->ptr_h, arrays_d, (size_t)k * 8);
        memcpy(g->len_h, n, (size_t)k * 8);
        std::copy(span.begin(), span.end(), g->span);
        g->n_span = (int)span.size();
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
    free(g->span);
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
    for (int i = 0; i < g->k; ++i) {
        if (!g->len_h[i] || (same && o->ptr_h[i] == g->ptr_h[i])) continue;
        const uintptr_t lo = (uintptr_t)o->ptr_h[i], hi = lo + g->len_h[i] * g->batch * e;
        // the last array of g that starts before hi ends last of those
        const tramp_group::Span* it = std::lower_bound(g->span, g->span + g->n_span, hi, [](const tramp_group::Span& s, uintptr_t x) { return s.lo < x; });
        if (it != g->span && (it - 1)->hi > lo) return tramp_fail(ctx, TRAMP_EINVAL, what, "the arrays of the two lists overlap");
    }
    return TRAMP_OK;
}

// n doubles of the caller's (norms, precisions) that touch no array of g
static bool clear_of(const tramp_group* g, const double* p, size_t n) {
    const uintptr_t lo = (uintptr_t)p, hi = lo + n * sizeof(double);
    const tramp_group::Span* it = std::lower_bound(g->span, g->span + g->n_span, hi, [](const tramp_group::Span& s, uintptr_t x) { return s.lo < x; });
    return !p || it == g->span || (it - 1)->hi <= lo;
}
static bool apart(const double* p, size_t n, const double* q, size_t m) { return !p || !q || p + n <= q || q + m <= p; }

// workgroups per instance: about kBlocks in all, each with the same number of chunks
static int partials_of(const tramp_group* g, size_t batch) {
    if (g->nchunk < 1) return 1;
    const size_t want = std::max((size_t)1, kBlocks / batch), rounds = (g->nchunk + want - 1) / want;
    return (int)((g->nchunk + rounds - 1) / rounds);
}

template <typename T, bool STEP>
static int group_run(tramp_ctx* ctx, const tramp_group* g, const tramp_group* prev, const tramp_group* out, const GroupSide& q) {
    const GroupChunk* ps = STEP ? prev->chunks : nullptr;
    if (g->nchunk <= kSmall) {
        hipLaunchKernelGGL((group_small_kernel<T, STEP>), dim3((unsigned)g->batch), dim3(kBlock), 0, ctx->stream, (unsigned)g->nchunk, g->chunks,
                           ps, out ? out->chunks : nullptr, q);
        TRAMP_LAUNCH_CHECK(ctx);
        return TRAMP_OK;
    }
    // Instances in slices whose arrays stay in the 256 MB of cache from one pass to the other: every launch finishes one slice and
    // takes the sums of the next.
    const size_t bytes = g->nchunk * kChunkBytes * (STEP ? 2 : 1), most = kSlice;
    const size_t slice = !out || bytes * g->batch <= 2 * most || bytes > most ? g->batch : most / bytes;
    const int P = partials_of(g, slice);
    int rc = tramp_ws_reserve(ctx, g->batch * (size_t)P * sizeof(double));
    if (rc) return rc;
    size_t done = 0, summed = 0;
    while (done < g->batch) {
        const size_t n_apply = out ? summed - done : 0, n_sum = std::min(slice, g->batch - summed);
        const dim3 grid((unsigned)P, (unsigned)(n_apply + n_sum));
        const GroupChunk* os = out ? out->chunks : nullptr;
        if (bytes * g->batch > kOnce)
            hipLaunchKernelGGL((group_pass_kernel<T, STEP, true>), grid, dim3(kBlock), 0, ctx->stream, (unsigned)g->nchunk, g->chunks, ps, os,
                               done, (unsigned)n_apply, q, ctx->ws);
        else
            hipLaunchKernelGGL((group_pass_kernel<T, STEP, false>), grid, dim3(kBlock), 0, ctx->stream, (unsigned)g->nchunk, g->chunks, ps, os,
                               done, (unsigned)n_apply, q, ctx->ws);
        done = summed;
        summed += n_sum;
        if (!out) break;
    }
    if (!out)
        hipLaunchKernelGGL(group_norm_kernel, dim3((unsigned)g->batch), dim3(kBlock), 0, ctx->stream, ctx->ws, P, q.norm_out);
    TRAMP_LAUNCH_CHECK(ctx);
    return TRAMP_OK;
}

extern "C" int tramp_group_norm(tramp_ctx* ctx, const tramp_group* g, double* norm_d) {
    if (!ctx) return TRAMP_EINVAL;
    TRAMP_REQUIRE(ctx, g && norm_d && g->device == ctx->device);
    TRAMP_REQUIRE(ctx, clear_of(g, norm_d, g->batch));
    const GroupSide q{0.0, norm_d, nullptr, nullptr, 0, g->batch, 0};
    return g->dtype == TRAMP_F64 ? group_run<double, false>(ctx, g, nullptr, nullptr, q)
                                 : group_run<float, false>(ctx, g, nullptr, nullptr, q);
}

extern "C" int tramp_group_clip(tramp_ctx* ctx, const tramp_group* g, double max_norm, const tramp_group* out, double* norm_d) {
    if (!ctx) return TRAMP_EINVAL;
    TRAMP_REQUIRE(ctx, g && out && g->device == ctx->device);
    TRAMP_REQUIRE(ctx, max_norm > 0.0);
    int rc = check_pair(ctx, g, out, true, "tramp_group_clip");
    if (rc) return rc;
    TRAMP_REQUIRE(ctx, clear_of(g, norm_d, g->batch) && clear_of(out, norm_d, g->batch));
    const GroupSide q{max_norm, norm_d, nullptr, nullptr, 0, g->batch, 0};
    return g->dtype == TRAMP_F64 ? group_run<double, false>(ctx, g, nullptr, out, q)
                                 : group_run<float, false>(ctx, g, nullptr, out, q);
}

extern "C" int tramp_group_limit_step(tramp_ctx* ctx, const tramp_group* g, const tramp_group* prev, double max_step,
                                      const tramp_group* out, int refresh, size_t n_a, double* a_d, double* a_prev_d, double* norm_d) {
    if (!ctx) return TRAMP_EINVAL;
    TRAMP_REQUIRE(ctx, g && prev && out && g->device == ctx->device);
    TRAMP_REQUIRE(ctx, max_step > 0.0);
    TRAMP_REQUIRE(ctx, n_a == 0 || (a_d && a_prev_d));
    const size_t na = n_a * g->batch;
    if (!n_a) a_d = a_prev_d = nullptr;
    TRAMP_REQUIRE(ctx, apart(a_d, na, a_prev_d, na) && apart(a_d, na, norm_d, g->batch) && apart(a_prev_d, na, norm_d, g->batch));
    for (const tramp_group* l : {g, prev, out})
        TRAMP_REQUIRE(ctx, clear_of(l, norm_d, g->batch) && clear_of(l, a_d, na) && clear_of(l, a_prev_d, na));
    int rc = check_pair(ctx, g, prev, false, "tramp_group_limit_step");
    if (!rc) rc = check_pair(ctx, g, out, true, "tramp_group_limit_step");
    if (!rc) rc = check_pair(ctx, prev, out, false, "tramp_group_limit_step");
    if (rc) return rc;
    const GroupSide q{max_step, norm_d, a_d, a_prev_d, n_a, g->batch, refresh};
    return g->dtype == TRAMP_F64 ? group_run<double, true>(ctx, g, prev, out, q)
                                 : group_run<float, true>(ctx, g, prev, out, q);
}
