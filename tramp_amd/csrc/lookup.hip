// lookup.hip - lookup channel x_t = scale z[token_t] of a table z of V rows and D columns.
//
// The linear factor of categorical data: W [T D, V D] has one entry `scale` per row (none where the position is padded), so
// W^T W = scale^2 diag(count_v) (x) I_D and every quantity of LinearChannel (tramp/channels/linear/linear_channel.py:58-132)
// is closed form in the counts.  With  g_v = scale sum_{t: token_t = v} bx_t  (the adjoint),  lik_v = ax scale^2 count_v,
// prec_v = az + lik_v:
//     r_v  = (bz_v + g_v) / prec_v                                  posterior mean of the table
//     rx_t = scale r_{token_t}                                      posterior mean of the positions (0 where padded)
//     vz   = (1/V) sum_v 1 / prec_v            vx = (scale^2 / T) sum_v count_v / prec_v
// and the messages a' = clip(1/v - a), b' = r (a + a') - b (tramp/base.py:250-255).  Both ends of 1/v - a and of the b' to
// the table are sums without cancellation, which is how they are formed here:
//     1/vz - az = [(1/V) sum_v lik_v / prec_v] / vz
//     1/vx - ax = [padded / T + (1/T) sum_v count_v (az + ax scale^2 (count_v - 1)) / prec_v] / vx
//     b'_v = [g_v (az + a') + bz_v (a' - lik_v)] / prec_v
// (a table of 10^5 rows of which ten are read has a' of order 10^-4 az: the difference would lose the digits of f64).
//
// The positions are sorted by token once, at creation (perm, off): the adjoint is a sum over runs, in a fixed order, without
// atomics, the same bits every time.  All arithmetic is in double and rounded once to the element type at the store: the
// passes are bound by memory (a few operations per element), the conversions are free next to the loads.
#include "common.h"
#include "tramp_math.h"

#include <algorithm>
#include <new>
#include <vector>

struct tramp_lookup {
    int device;
    int dtype;
    size_t V, D, T;
    size_t seen;                 // positions that read a row
    double s;                    // scale
    void* mem;                   // one allocation behind all the arrays below
    const int* tok;              // [T]    token, -1 where padded
    const int* perm;             // [seen] positions sorted by token, ascending within a token
    const int* off;              // [V + 1] the run of token v is perm[off[v] .. off[v + 1])
    const double* cnt;           // [2, K] distinct counts and how many rows have them
    int K;
};

// what the kernels need of one instance, written by lookup_scalars_kernel
struct LkScal {
    double az, ax, an, lik1;     // floored az, ax, a' before damping, ax scale^2
};

// ---------------------------------------------------------------- scalars
// v, a' and n_eff of every instance from the table of distinct counts (n of them sum to at least n(n-1)/2 positions: 1414
// at 10^6 positions), one workgroup per instance.
__global__ __launch_bounds__(kBlock) void lookup_scalars_kernel(int K, const double* __restrict__ cnt, double V, double T,
                                                                double padded, double s, int dir, const double* az_d,
                                                                const double* ax_d, double damping, const double* a_old,
                                                                LkScal* __restrict__ scal, double* v_out, double* a_new_out,
                                                                double* n_eff_out) {
    __shared__ double smem[kBlock / kWave];
    const size_t b = blockIdx.x;
    const double ax = ax_d[b], az = dir == TRAMP_BWD ? fmax(1e-11, az_d[b]) : az_d[b];     // linear_channel.py:92-94
    const double lik1 = ax * s * s;
    double sv = 0.0, sn = 0.0, se = 0.0;
    for (int k = threadIdx.x; k < K; k += kBlock) {
        const double c = cnt[k], m = cnt[K + k];
        if (dir == TRAMP_FWD && c == 0.0) continue;              // a row nobody reads does not reach x
        const double prec = az + lik1 * c;
        if (dir == TRAMP_BWD) {
            sv += m / prec;
            sn += m * (lik1 * c / prec);
        } else {
            sv += m * c / prec;
            sn += m * c * ((az + lik1 * (c - 1.0)) / prec);
        }
        if (ax != 0.0) se += m * (lik1 * c / prec);
    }
    sv = block_sum(sv, smem);
    sn = block_sum(sn, smem);
    se = block_sum(se, smem);
    if (threadIdx.x != 0) return;
    double v, an;
    if (dir == TRAMP_BWD) {
        v = sv / V;
        an = (sn / V) / v;
    } else {
        v = s * s * sv / T;
        an = ((padded + sn) / T) / v;
    }
    if (v > 1.7976931348623157e308) an = 0.0;                    // both precisions zero: 1 / v - a <= 0
    if (an < tmath::kAMin) an = tmath::kAMin;                    // (comparisons: a NaN passes through, tramp/base.py:252)
    if (an > tmath::kAMax) an = tmath::kAMax;
    if (scal) scal[b] = LkScal{az, ax, an, lik1};
    if (v_out) v_out[b] = v;
    if (n_eff_out) n_eff_out[b] = se / V;
    if (a_new_out) a_new_out[b] = damping != 0.0 ? damping * a_old[b] + (1.0 - damping) * an : an;
}

// ---------------------------------------------------------------- x = scale z[token]
template <typename T>
__global__ __launch_bounds__(kBlock) void lookup_apply_kernel(size_t V, size_t D, size_t n, double s, const int* __restrict__ tok,
                                                              const T* __restrict__ z, T* __restrict__ x) {
    const size_t b = blockIdx.y;
    for (size_t i = (size_t)blockIdx.x * kBlock + threadIdx.x; i < n; i += (size_t)gridDim.x * kBlock) {
        const size_t t = i / D, d = i - t * D;
        const int k = tok[t];
        x[b * n + i] = k < 0 ? T(0) : T(s * (double)z[(b * V + (size_t)k) * D + d]);
    }
}

// ---------------------------------------------------------------- sums over the runs
// MODE 0: g = scale sum.  1: the message to the table.  2: r of the table in double (workspace of the forward message).
template <typename T, int MODE>
__global__ __launch_bounds__(kBlock) void lookup_rows_kernel(size_t V, size_t D, size_t Tn, double s, const int* __restrict__ off,
                                                             const int* __restrict__ perm, const LkScal* __restrict__ scal,
                                                             const T* __restrict__ bz, const T* __restrict__ x, double damping,
                                                             const T* b_old, T* out, T* __restrict__ r_out,
                                                             double* __restrict__ r_ws) {
    const size_t b = blockIdx.y, n = V * D;
    LkScal c{};
    if (MODE) c = scal[b];
    for (size_t i = (size_t)blockIdx.x * kBlock + threadIdx.x; i < n; i += (size_t)gridDim.x * kBlock) {
        const size_t v = i / D, d = i - v * D;
        const int j0 = off[v], j1 = off[v + 1];
        double g = 0.0;
        for (int j = j0; j < j1; ++j) g += (double)x[(b * Tn + (size_t)perm[j]) * D + d];
        g *= s;
        if (MODE == 0) {
            out[b * n + i] = T(g);
        } else {
            const double lik = c.lik1 * (double)(j1 - j0), prec = c.az + lik, z = (double)bz[b * n + i];
            if (MODE == 2) {
                r_ws[b * n + i] = (z + g) / prec;
            } else {
                double o = (g * (c.az + c.an) + z * (c.an - lik)) / prec;
                if (damping != 0.0) o = damping * (double)b_old[b * n + i] + (1.0 - damping) * o;
                out[b * n + i] = T(o);
                if (r_out) r_out[b * n + i] = T((z + g) / prec);
            }
        }
    }
}

// ---------------------------------------------------------------- the message to the positions
template <typename T>
__global__ __launch_bounds__(kBlock) void lookup_positions_kernel(size_t V, size_t D, size_t n, double s, const int* __restrict__ tok,
                                                                  const LkScal* __restrict__ scal, const double* __restrict__ r_ws,
                                                                  const T* __restrict__ bx, double damping, const T* b_old,
                                                                  T* out, T* __restrict__ r_out) {
    const size_t b = blockIdx.y;
    const double asum = scal[b].ax + scal[b].an;
    for (size_t i = (size_t)blockIdx.x * kBlock + threadIdx.x; i < n; i += (size_t)gridDim.x * kBlock) {
        const size_t t = i / D, d = i - t * D;
        const int k = tok[t];
        const double r = k < 0 ? 0.0 : s * r_ws[(b * V + (size_t)k) * D + d];
        double o = r * asum - (double)bx[b * n + i];
        if (damping != 0.0) o = damping * (double)b_old[b * n + i] + (1.0 - damping) * o;
        out[b * n + i] = T(o);
        if (r_out) r_out[b * n + i] = T(r);
    }
}

// ---------------------------------------------------------------- log-partition
// A = 1/2 sum_v (bz + g)^2 / prec + D/2 sum_v log(2 pi / prec)   (linear_channel.py:127-132)
template <typename T>
__global__ __launch_bounds__(kBlock) void lookup_logz_kernel(size_t V, size_t D, size_t Tn, double s, const int* __restrict__ off,
                                                             const int* __restrict__ perm, const double* __restrict__ az_d,
                                                             const double* __restrict__ ax_d, const T* __restrict__ bz,
                                                             const T* __restrict__ x, double* __restrict__ partials) {
    __shared__ double smem[kBlock / kWave];
    const size_t b = blockIdx.y, n = V * D;
    const double az = az_d[b], lik1 = ax_d[b] * s * s;
    double acc = 0.0;
    for (size_t i = (size_t)blockIdx.x * kBlock + threadIdx.x; i < n; i += (size_t)gridDim.x * kBlock) {
        const size_t v = i / D, d = i - v * D;
        const int j0 = off[v], j1 = off[v + 1];
        double g = 0.0;
        for (int j = j0; j < j1; ++j) g += (double)x[(b * Tn + (size_t)perm[j]) * D + d];
        const double prec = az + lik1 * (double)(j1 - j0), h = (double)bz[b * n + i] + s * g;
        acc += 0.5 * (h * h / prec) + 0.5 * log(2.0 * tmath::kPi / prec);
    }
    acc = block_sum(acc, smem);
    if (threadIdx.x == 0) partials[b * gridDim.x + blockIdx.x] = acc;
}

__global__ __launch_bounds__(kBlock) void lookup_fold_kernel(int n, const double* __restrict__ partials, double* __restrict__ out) {
    __shared__ double smem[kBlock / kWave];
    double acc = 0.0;
    for (int i = threadIdx.x; i < n; i += kBlock) acc += partials[(size_t)blockIdx.x * n + i];
    acc = block_sum(acc, smem);
    if (threadIdx.x == 0) out[blockIdx.x] = acc;
}

// ---------------------------------------------------------------- handle
extern "C" int tramp_lookup_create(tramp_ctx* ctx, int dtype, size_t n_rows, size_t n_cols, size_t n_pos, const int* tokens_h,
                                   double scale, tramp_lookup** out) {
    if (!ctx || !out) return TRAMP_EINVAL;
    *out = nullptr;
    TRAMP_REQUIRE(ctx, dtype == TRAMP_F32 || dtype == TRAMP_F64);
    TRAMP_REQUIRE(ctx, n_rows > 0 && n_cols > 0 && n_pos > 0 && tokens_h);
    TRAMP_REQUIRE(ctx, n_rows < 0x7fffffffu && n_cols < 0x7fffffffu && n_pos < 0x7fffffffu);
    TRAMP_REQUIRE(ctx, scale - scale == 0.0);
    TRAMP_REQUIRE(ctx, !ctx->capturing);
    for (size_t t = 0; t < n_pos; ++t)
        if (tokens_h[t] < -1 || (tokens_h[t] >= 0 && (size_t)tokens_h[t] >= n_rows))
            return tramp_fail(ctx, TRAMP_EINVAL, "tramp_lookup_create", "a token is neither a row of the table nor -1");
    try {
        std::vector<int> off(n_rows + 1, 0), perm;
        for (size_t t = 0; t < n_pos; ++t)
            if (tokens_h[t] >= 0) ++off[(size_t)tokens_h[t] + 1];
        std::vector<int> counts(off.begin() + 1, off.end());
        for (size_t v = 0; v < n_rows; ++v) off[v + 1] += off[v];
        const size_t seen = (size_t)off[n_rows];
        perm.resize(seen);
        {
            std::vector<int> at(off.begin(), off.end() - 1);
            for (size_t t = 0; t < n_pos; ++t)
                if (tokens_h[t] >= 0) perm[(size_t)at[(size_t)tokens_h[t]]++] = (int)t;
        }
        std::sort(counts.begin(), counts.end());
        std::vector<double> cval, cmul;
        for (size_t v = 0; v < n_rows; ++v) {
            if (cval.empty() || cval.back() != (double)counts[v]) {
                cval.push_back((double)counts[v]);
                cmul.push_back(0.0);
            }
            cmul.back() += 1.0;
        }
        const size_t K = cval.size();
        cval.insert(cval.end(), cmul.begin(), cmul.end());
        auto up = [](size_t bytes) { return (bytes + 255) & ~(size_t)255; };
        const size_t o_perm = up(n_pos * 4), o_off = o_perm + up(seen * 4), o_cnt = o_off + up((n_rows + 1) * 4);
        const size_t total = o_cnt + up(2 * K * 8);
        tramp_lookup* lk = new tramp_lookup();
        *lk = tramp_lookup{};
        (void)hipSetDevice(ctx->device);
        if (hipMalloc(&lk->mem, total) != hipSuccess) {
            (void)hipGetLastError();
            delete lk;
            return tramp_fail(ctx, TRAMP_ENOMEM, "tramp_lookup_create", "hipMalloc failed");
        }
        char* m = static_cast<char*>(lk->mem);
        hipError_t e = hipMemcpyAsync(m, tokens_h, n_pos * 4, hipMemcpyHostToDevice, ctx->stream);
        if (e == hipSuccess && seen) e = hipMemcpyAsync(m + o_perm, perm.data(), seen * 4, hipMemcpyHostToDevice, ctx->stream);
        if (e == hipSuccess) e = hipMemcpyAsync(m + o_off, off.data(), (n_rows + 1) * 4, hipMemcpyHostToDevice, ctx->stream);
        if (e == hipSuccess) e = hipMemcpyAsync(m + o_cnt, cval.data(), 2 * K * 8, hipMemcpyHostToDevice, ctx->stream);
        if (e == hipSuccess) e = hipStreamSynchronize(ctx->stream);      // the host arrays end here
        if (e != hipSuccess) {
            (void)hipFree(lk->mem);
            delete lk;
            return tramp_fail(ctx, TRAMP_EHIP, "tramp_lookup_create", hipGetErrorString(e));
        }
        lk->device = ctx->device;
        lk->dtype = dtype;
        lk->V = n_rows;
        lk->D = n_cols;
        lk->T = n_pos;
        lk->seen = seen;
        lk->s = scale;
        lk->tok = reinterpret_cast<const int*>(m);
        lk->perm = reinterpret_cast<const int*>(m + o_perm);
        lk->off = reinterpret_cast<const int*>(m + o_off);
        lk->cnt = reinterpret_cast<const double*>(m + o_cnt);
        lk->K = (int)K;
        *out = lk;
        return TRAMP_OK;
    } catch (const std::bad_alloc&) {
        return tramp_fail(ctx, TRAMP_ENOMEM, "tramp_lookup_create", "host memory");
    }
}

extern "C" int tramp_lookup_destroy(tramp_ctx* ctx, tramp_lookup* lk) {
    if (!ctx || !lk) return TRAMP_EINVAL;
    (void)hipStreamSynchronize(ctx->stream);
    (void)hipFree(lk->mem);
    delete lk;
    return TRAMP_OK;
}

#define LK_REQUIRE_CALL(ctx, lk, batch)                      \
    if (!ctx) return TRAMP_EINVAL;                           \
    TRAMP_REQUIRE(ctx, lk && lk->device == ctx->device);     \
    TRAMP_REQUIRE(ctx, batch <= 65535)

extern "C" int tramp_lookup_apply(tramp_ctx* ctx, tramp_lookup* lk, size_t batch, const void* z_d, void* x_d) {
    LK_REQUIRE_CALL(ctx, lk, batch);
    TRAMP_REQUIRE(ctx, z_d && x_d && z_d != x_d);
    if (!batch) return TRAMP_OK;
    const size_t n = lk->T * lk->D;
    dim3 grid(blocks_for(n, 1), (unsigned)batch);
    if (lk->dtype == TRAMP_F64)
        hipLaunchKernelGGL((lookup_apply_kernel<double>), grid, dim3(kBlock), 0, ctx->stream, lk->V, lk->D, n, lk->s, lk->tok,
                           (const double*)z_d, (double*)x_d);
    else
        hipLaunchKernelGGL((lookup_apply_kernel<float>), grid, dim3(kBlock), 0, ctx->stream, lk->V, lk->D, n, lk->s, lk->tok,
                           (const float*)z_d, (float*)x_d);
    TRAMP_LAUNCH_CHECK(ctx);
    return TRAMP_OK;
}

template <typename T, int MODE>
static void launch_rows(tramp_ctx* ctx, const tramp_lookup* lk, size_t batch, const LkScal* scal, const void* bz, const void* x,
                        double damping, const void* b_old, void* out, void* r_out, double* r_ws) {
    dim3 grid(blocks_for(lk->V * lk->D, 1), (unsigned)batch);
    hipLaunchKernelGGL((lookup_rows_kernel<T, MODE>), grid, dim3(kBlock), 0, ctx->stream, lk->V, lk->D, lk->T, lk->s, lk->off,
                       lk->perm, scal, (const T*)bz, (const T*)x, damping, (const T*)b_old, (T*)out, (T*)r_out, r_ws);
}

extern "C" int tramp_lookup_gradient(tramp_ctx* ctx, tramp_lookup* lk, size_t batch, const void* x_d, void* g_d) {
    LK_REQUIRE_CALL(ctx, lk, batch);
    TRAMP_REQUIRE(ctx, x_d && g_d && x_d != g_d);
    if (!batch) return TRAMP_OK;
    if (lk->dtype == TRAMP_F64)
        launch_rows<double, 0>(ctx, lk, batch, nullptr, nullptr, x_d, 0.0, nullptr, g_d, nullptr, nullptr);
    else
        launch_rows<float, 0>(ctx, lk, batch, nullptr, nullptr, x_d, 0.0, nullptr, g_d, nullptr, nullptr);
    TRAMP_LAUNCH_CHECK(ctx);
    return TRAMP_OK;
}

static void launch_scalars(tramp_ctx* ctx, const tramp_lookup* lk, int dir, size_t batch, const double* az_d, const double* ax_d,
                           double damping, const double* a_old_d, LkScal* scal, double* v_d, double* a_new_d, double* n_eff_d) {
    hipLaunchKernelGGL(lookup_scalars_kernel, dim3((unsigned)batch), dim3(kBlock), 0, ctx->stream, lk->K, lk->cnt, (double)lk->V,
                       (double)lk->T, (double)(lk->T - lk->seen), lk->s, dir, az_d, ax_d, damping, a_old_d, scal, v_d, a_new_d,
                       n_eff_d);
}

extern "C" int tramp_lookup_variance(tramp_ctx* ctx, tramp_lookup* lk, int dir, size_t batch, const double* az_d,
                                     const double* ax_d, double* v_d, double* a_new_d, double* n_eff_d) {
    LK_REQUIRE_CALL(ctx, lk, batch);
    TRAMP_REQUIRE(ctx, (dir == TRAMP_FWD || dir == TRAMP_BWD) && az_d && ax_d);
    if (!batch) return TRAMP_OK;
    launch_scalars(ctx, lk, dir, batch, az_d, ax_d, 0.0, nullptr, nullptr, v_d, a_new_d, n_eff_d);
    TRAMP_LAUNCH_CHECK(ctx);
    return TRAMP_OK;
}

template <typename T>
static int lookup_message(tramp_ctx* ctx, tramp_lookup* lk, int dir, size_t batch, const double* az_d, const T* bz,
                          const double* ax_d, const T* bx, double damping, const double* a_old_d, const T* b_old, double* a_new_d,
                          T* b_new, T* r_d, double* v_d) {
    const size_t n_scal = (batch * sizeof(LkScal) + 255) & ~(size_t)255;
    int rc = tramp_ws_reserve(ctx, n_scal + (dir == TRAMP_FWD ? batch * lk->V * lk->D * sizeof(double) : 0));
    if (rc) return rc;
    LkScal* scal = reinterpret_cast<LkScal*>(ctx->ws);
    double* r_ws = reinterpret_cast<double*>(reinterpret_cast<char*>(ctx->ws) + n_scal);
    launch_scalars(ctx, lk, dir, batch, az_d, ax_d, damping, a_old_d, scal, v_d, a_new_d, nullptr);
    if (dir == TRAMP_BWD) {
        launch_rows<T, 1>(ctx, lk, batch, scal, bz, bx, damping, b_old, b_new, r_d, nullptr);
    } else {
        launch_rows<T, 2>(ctx, lk, batch, scal, bz, bx, 0.0, nullptr, nullptr, nullptr, r_ws);
        const size_t n = lk->T * lk->D;
        dim3 grid(blocks_for(n, 1), (unsigned)batch);
        hipLaunchKernelGGL((lookup_positions_kernel<T>), grid, dim3(kBlock), 0, ctx->stream, lk->V, lk->D, n, lk->s, lk->tok, scal,
                           r_ws, bx, damping, b_old, b_new, r_d);
    }
    TRAMP_LAUNCH_CHECK(ctx);
    return TRAMP_OK;
}

extern "C" int tramp_lookup_message(tramp_ctx* ctx, tramp_lookup* lk, int dir, size_t batch, const double* az_d, const void* bz_d,
                                    const double* ax_d, const void* bx_d, double damping, const double* a_old_d,
                                    const void* b_old_d, double* a_new_d, void* b_new_d, void* r_d, double* v_d) {
    LK_REQUIRE_CALL(ctx, lk, batch);
    TRAMP_REQUIRE(ctx, (dir == TRAMP_FWD || dir == TRAMP_BWD) && az_d && bz_d && ax_d && bx_d && a_new_d && b_new_d);
    TRAMP_REQUIRE(ctx, b_new_d != bz_d && b_new_d != bx_d);
    TRAMP_REQUIRE(ctx, damping == 0.0 || (a_old_d && b_old_d));
    if (!batch) return TRAMP_OK;
    if (lk->dtype == TRAMP_F64)
        return lookup_message<double>(ctx, lk, dir, batch, az_d, (const double*)bz_d, ax_d, (const double*)bx_d, damping, a_old_d,
                                      (const double*)b_old_d, a_new_d, (double*)b_new_d, (double*)r_d, v_d);
    return lookup_message<float>(ctx, lk, dir, batch, az_d, (const float*)bz_d, ax_d, (const float*)bx_d, damping, a_old_d,
                                 (const float*)b_old_d, a_new_d, (float*)b_new_d, (float*)r_d, v_d);
}

extern "C" int tramp_lookup_log_partition(tramp_ctx* ctx, tramp_lookup* lk, size_t batch, const double* az_d, const void* bz_d,
                                          const double* ax_d, const void* bx_d, double* out_d) {
    LK_REQUIRE_CALL(ctx, lk, batch);
    TRAMP_REQUIRE(ctx, az_d && bz_d && ax_d && bx_d && out_d);
    if (!batch) return TRAMP_OK;
    const int nblk = blocks_for(lk->V * lk->D, 1);
    int rc = tramp_ws_reserve(ctx, batch * (size_t)nblk * sizeof(double));
    if (rc) return rc;
    dim3 grid(nblk, (unsigned)batch);
    if (lk->dtype == TRAMP_F64)
        hipLaunchKernelGGL((lookup_logz_kernel<double>), grid, dim3(kBlock), 0, ctx->stream, lk->V, lk->D, lk->T, lk->s, lk->off,
                           lk->perm, az_d, ax_d, (const double*)bz_d, (const double*)bx_d, ctx->ws);
    else
        hipLaunchKernelGGL((lookup_logz_kernel<float>), grid, dim3(kBlock), 0, ctx->stream, lk->V, lk->D, lk->T, lk->s, lk->off,
                           lk->perm, az_d, ax_d, (const float*)bz_d, (const float*)bx_d, ctx->ws);
    hipLaunchKernelGGL(lookup_fold_kernel, dim3((unsigned)batch), dim3(kBlock), 0, ctx->stream, nblk, ctx->ws, out_d);
    TRAMP_LAUNCH_CHECK(ctx);
    return TRAMP_OK;
}
