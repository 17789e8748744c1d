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

struct LkItem;
struct tramp_lookup {
    int device;
    int dtype;
    size_t V, D, T;
    size_t seen;                 // positions that read a row
    double s;                    // scale
    void* mem;                   // one allocation behind all the arrays below
    const int* tok;              // [T]     token, -1 where padded
    const int* perm;             // [T]     positions sorted by token, ascending within a token, the padded ones last
    const int* off;              // [V + 1] the run of token v is perm[off[v] .. off[v + 1])
    const double* cnt;           // [2, K]  distinct counts and how many rows have them
    int K;
    const LkItem* items;         // runs for whole workgroups (lookup_rows_kernel)
    const LkItem* joins;         // heavy runs
    const LkItem* spreads;       // their positions and the padded ones, in chunks
    const int* waves;
    unsigned n_items, n_joins, n_spreads, n_waves, n_slots;
    int lw;                      // log2 of the lanes per row
    unsigned tiles;              // column tiles per row
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

// ---------------------------------------------------------------- rows in 16-byte pieces
// A row of D elements is walked by LPR = min(64, 2^ceil(log2(D / N))) lanes, one 16-byte piece (N elements) per lane, in
// column tiles of LPR pieces where the row is longer (1 KiB per wave and row).  The pieces start wherever the row does: a
// 16-byte access needs element alignment only, so odd D and views cost nothing but the last piece of a row (TAIL).
template <typename T> struct LkVec;
template <> struct LkVec<float> {
    typedef float U __attribute__((ext_vector_type(4), aligned(4)));
    static constexpr int N = 4;
};
template <> struct LkVec<double> {
    typedef double U __attribute__((ext_vector_type(2), aligned(8)));
    static constexpr int N = 2;
};

template <typename T, bool TAIL>
__device__ __forceinline__ void lk_load(const T* __restrict__ p, int valid, T (&v)[LkVec<T>::N]) {
    constexpr int N = LkVec<T>::N;
    if (!TAIL || valid == N) {
        const typename LkVec<T>::U u = *reinterpret_cast<const typename LkVec<T>::U*>(p);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = u[i];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = i < valid ? p[i] : T(0);
    }
}

template <typename T, bool TAIL>
__device__ __forceinline__ void lk_store(T* p, int valid, const T (&v)[LkVec<T>::N]) {
    constexpr int N = LkVec<T>::N;
    if (!TAIL || valid == N) {
        typename LkVec<T>::U u;
#pragma unroll
        for (int i = 0; i < N; ++i) u[i] = v[i];
        *reinterpret_cast<typename LkVec<T>::U*>(p) = u;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < valid) p[i] = v[i];
    }
}

// where a lane stands: its group (one row at a time per group), its piece of the row
struct LkLane {
    int lw;                      // log2 LPR
    int group, l;
    size_t col;                  // first element of the piece
    int valid;                   // elements of the piece that exist (<= 0: none)
};
template <typename T> __device__ __forceinline__ LkLane lk_lane(int lw, unsigned tile, size_t D) {
    LkLane k;
    k.lw = lw;
    k.group = threadIdx.x >> lw;
    k.l = threadIdx.x & ((1 << lw) - 1);
    k.col = (((size_t)tile << lw) + k.l) * LkVec<T>::N;
    const long left = (long)D - (long)k.col;
    k.valid = left >= LkVec<T>::N ? LkVec<T>::N : (int)left;
    return k;
}

// ---------------------------------------------------------------- x = scale z[token]
// Bound by the write of x (and the read of the distinct rows of z).  Four rows per group in flight.
template <typename T, bool TAIL>
__global__ __launch_bounds__(kBlock) void lookup_apply_kernel(size_t V, size_t D, size_t n_pos, double s, int lw, unsigned tiles,
                                                              const int* __restrict__ tok, const T* __restrict__ z, T* __restrict__ x) {
    constexpr int N = LkVec<T>::N, UR = 4;
    const size_t b = blockIdx.y;
    const unsigned blk = blockIdx.x / tiles, tile = blockIdx.x - blk * tiles;
    const LkLane k = lk_lane<T>(lw, tile, D);
    if (k.valid <= 0) return;
    const size_t G = kBlock >> lw;
    int row[UR];
    T v[UR][N];
    size_t t0 = (size_t)blk * UR * G + k.group;
#pragma unroll
    for (int i = 0; i < UR; ++i) row[i] = t0 + i * G < n_pos ? tok[t0 + i * G] : -1;
#pragma unroll
    for (int i = 0; i < UR; ++i) {
        if (row[i] >= 0) {
            lk_load<T, TAIL>(z + (b * V + (size_t)row[i]) * D + k.col, k.valid, v[i]);
#pragma unroll
            for (int e = 0; e < N; ++e) v[i][e] = T(s * (double)v[i][e]);
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) v[i][e] = T(0);
        }
    }
#pragma unroll
    for (int i = 0; i < UR; ++i)
        if (t0 + i * G < n_pos) lk_store<T, TAIL>(x + (b * n_pos + t0 + i * G) * D + k.col, k.valid, v[i]);
}

// one column: N positions per lane, written as one piece
template <typename T>
__global__ __launch_bounds__(kBlock) void lookup_apply1_kernel(size_t V, size_t n_pos, double s, const int* __restrict__ tok,
                                                               const T* __restrict__ z, T* __restrict__ x) {
    constexpr int N = LkVec<T>::N;
    const size_t b = blockIdx.y, t = ((size_t)blockIdx.x * kBlock + threadIdx.x) * N;
    if (t >= n_pos) return;
    const int valid = n_pos - t >= N ? N : (int)(n_pos - t);
    int row[N];
    T v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) row[i] = i < valid ? tok[t + i] : -1;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = row[i] >= 0 ? T(s * (double)z[b * V + (size_t)row[i]]) : T(0);
    lk_store<T, true>(x + b * n_pos + t, valid, v);
}

// ---------------------------------------------------------------- sums over the runs
// The run lengths of real tokens differ by orders of magnitude, so the work is cut by them, at creation:
//   light  run <= kKeep                       one group, all rows of the run in flight at once
//   wave   run <= kKeep * 64 / LPR            the groups of one wave, joined by a butterfly
//   block  run <= kKeep * 256 / LPR           the groups of one workgroup, the four waves joined through LDS
//   heavy  longer                             chunks of a multiple of that; partial sums in double, joined by a second launch
// In the first three every row stays in registers from the sum to the message that goes back to its position: the message to
// the positions reads bx once.  Only the runs of the last kind read it twice.
constexpr int kKeep = 16;

struct LkItem {
    int token, start, end, slot;      // slot: of the partial sum; < 0: the item is a whole run
};

struct LkArgs {
    const int* off;
    const int* perm;
    const LkItem* items;         // [n_items] heavy chunks, then the block runs
    const int* waves;            // [n_waves] tokens of the wave runs
    size_t V, D, T;
    unsigned n_items, n_waves, wave_blocks, blocks, tiles, n_slots;
    int lw;
    double s;
};

enum { LK_GRAD = 0, LK_BWD = 1, LK_FWD = 2 };

// rows perm[j0 + sub], perm[j0 + sub + S], ... of the run [j0, j0 + c), S = 1 << ls: added into acc, kept if KEEP (c <= kKeep S)
template <typename T, bool TAIL, bool KEEP>
__device__ __forceinline__ void lk_gather(const LkArgs& a, const T* __restrict__ xb, const LkLane& k, int j0, int c, int sub, int ls,
                                          double (&acc)[LkVec<T>::N], int (&pj)[kKeep], T (&rows)[kKeep][LkVec<T>::N]) {
    constexpr int N = LkVec<T>::N;
    const int cnt = c > sub ? ((c - sub - 1) >> ls) + 1 : 0;
    const int* pp = a.perm + j0 + sub;
    for (int base = 0; base < cnt; base += kKeep) {
#pragma unroll
        for (int q = 0; q < kKeep; q += 4)
            if (base + q < cnt) {
#pragma unroll
                for (int i = q; i < q + 4; ++i) pj[i] = base + i < cnt ? pp[(size_t)(base + i) << ls] : -1;
            }
#pragma unroll
        for (int q = 0; q < kKeep; q += 4)
            if (base + q < cnt) {
#pragma unroll
                for (int i = q; i < q + 4; ++i)
                    if (base + i < cnt) lk_load<T, TAIL>(xb + (size_t)pj[i] * a.D + k.col, k.valid, rows[i]);
            }
#pragma unroll
        for (int i = 0; i < kKeep; ++i)
            if (base + i < cnt) {
#pragma unroll
                for (int e = 0; e < N; ++e) acc[e] += (double)rows[i][e];
            }
        if (KEEP) break;
    }
}

// sum over the groups of a wave: a butterfly, so that every group ends with the same bits
template <int N> __device__ __forceinline__ void lk_wave_join(int lw, double (&acc)[N]) {
    for (int off = 32; off >= (1 << lw); off >>= 1) {
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] += __shfl_xor(acc[e], off, 64);
    }
}

// and over the four waves of the workgroup
template <int N> __device__ __forceinline__ void lk_block_join(const LkLane& k, double (&acc)[N], double (*sm)[kWave][N]) {
    lk_wave_join<N>(k.lw, acc);
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
    for (int e = 0; e < N; ++e) sm[w][lane][e] = acc[e];
    __syncthreads();
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = ((sm[0][lane][e] + sm[1][lane][e]) + sm[2][lane][e]) + sm[3][lane][e];
}

// what is done with the sum of row v: the gradient or the message to the table; `first`: one group of those that hold the sum
template <typename T, bool TAIL, int MODE>
__device__ __forceinline__ void lk_row_out(const LkArgs& a, const LkScal& c, const LkLane& k, size_t b, int v, int count,
                                           const double (&acc)[LkVec<T>::N], const T* __restrict__ bz, double damping, const T* b_old,
                                           T* out, T* __restrict__ r_out) {
    constexpr int N = LkVec<T>::N;
    const size_t at = (b * a.V + (size_t)v) * a.D + k.col;
    T o[N];
    if (MODE == LK_GRAD) {
#pragma unroll
        for (int e = 0; e < N; ++e) o[e] = T(a.s * acc[e]);
    } else {
        const double lik = c.lik1 * (double)count, prec = c.az + lik;
        T z[N], r[N], old[N];
        lk_load<T, TAIL>(bz + at, k.valid, z);
        if (damping != 0.0) lk_load<T, TAIL>(b_old + at, k.valid, old);
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const double g = a.s * acc[e];
            double m = (g * (c.az + c.an) + (double)z[e] * (c.an - lik)) / prec;
            if (damping != 0.0) m = damping * (double)old[e] + (1.0 - damping) * m;
            o[e] = T(m);
            r[e] = T(((double)z[e] + g) / prec);
        }
        if (r_out) lk_store<T, TAIL>(r_out + at, k.valid, r);
    }
    lk_store<T, TAIL>(out + at, k.valid, o);
}

// the message to one position of a row with posterior mean r: rx = s r, b' = rx (ax + a') - bx
template <typename T, bool TAIL>
__device__ __forceinline__ void lk_position_out(const LkArgs& a, double asum, const LkLane& k, size_t b, int t,
                                                const double (&sr)[LkVec<T>::N], const T (&bx)[LkVec<T>::N], double damping, const T* b_old,
                                                T* out, T* __restrict__ r_out) {
    constexpr int N = LkVec<T>::N;
    const size_t at = (b * a.T + (size_t)t) * a.D + k.col;
    T o[N], old[N];
    if (damping != 0.0) lk_load<T, TAIL>(b_old + at, k.valid, old);
#pragma unroll
    for (int e = 0; e < N; ++e) {
        double m = sr[e] * asum - (double)bx[e];
        if (damping != 0.0) m = damping * (double)old[e] + (1.0 - damping) * m;
        o[e] = T(m);
    }
    lk_store<T, TAIL>(out + at, k.valid, o);
    if (r_out) {
#pragma unroll
        for (int e = 0; e < N; ++e) o[e] = T(sr[e]);
        lk_store<T, TAIL>(r_out + at, k.valid, o);
    }
}

template <typename T, bool TAIL, int MODE>
__global__ __launch_bounds__(kBlock) void lookup_rows_kernel(LkArgs a, const LkScal* __restrict__ scal, const T* __restrict__ bz,
                                                             const T* __restrict__ x, double damping, const T* b_old, T* out,
                                                             T* __restrict__ r_out, double* __restrict__ partials) {
    constexpr int N = LkVec<T>::N;
    __shared__ double sm[kBlock / kWave][kWave][N];
    const size_t b = blockIdx.y;
    const unsigned blk = blockIdx.x / a.tiles, tile = blockIdx.x - blk * a.tiles;
    const LkLane k = lk_lane<T>(a.lw, tile, a.D);
    LkScal c{};
    if (MODE != LK_GRAD) c = scal[b];
    const T* xb = x + b * a.T * a.D;
    const bool act = k.valid > 0;
    double acc[N];
    int pj[kKeep];
    T rows[kKeep][N];
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = 0.0;
    int v, j0, run, count, sub, ls;
    bool first = true;
    if (blk < a.n_items) {
        // a block run, or a chunk of a heavy one
        const LkItem it = a.items[blk];
        v = it.token;
        j0 = it.start;
        run = it.end - it.start;
        sub = k.group;
        ls = 8 - a.lw;
        first = threadIdx.x < (1 << a.lw);
        if (it.slot >= 0) {
            if (act) lk_gather<T, TAIL, false>(a, xb, k, j0, run, sub, ls, acc, pj, rows);
            lk_block_join<N>(k, acc, sm);
            if (first && act) {
                double* p = partials + (b * a.n_slots + (size_t)it.slot) * a.D + k.col;
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (e < k.valid) p[e] = acc[e];
            }
            return;
        }
        if (act) lk_gather<T, TAIL, true>(a, xb, k, j0, run, sub, ls, acc, pj, rows);
        lk_block_join<N>(k, acc, sm);
        count = run;
    } else {
        if (blk < a.n_items + a.wave_blocks) {
            const unsigned w = (blk - a.n_items) * (kBlock / kWave) + (threadIdx.x >> 6);
            if (w >= a.n_waves) return;
            v = a.waves[w];
            sub = (threadIdx.x & 63) >> a.lw;
            ls = 6 - a.lw;
            first = (threadIdx.x & 63) < (1 << a.lw);
        } else {
            const size_t u = (size_t)(blk - a.n_items - a.wave_blocks) * (kBlock >> a.lw) + k.group;
            if (u >= a.V) return;
            v = (int)u;
            sub = 0;
            ls = 0;
        }
        j0 = a.off[v];
        run = count = a.off[v + 1] - j0;
        if (ls == 0 && run > kKeep) return;                        // listed above
        if (act) lk_gather<T, TAIL, true>(a, xb, k, j0, run, sub, ls, acc, pj, rows);
        if (ls) lk_wave_join<N>(a.lw, acc);
    }
    if (!act) return;
    if (MODE != LK_FWD) {
        if (first) lk_row_out<T, TAIL, MODE>(a, c, k, b, v, count, acc, bz, damping, b_old, out, r_out);
        return;
    }
    if (count == 0) return;
    T z[N];
    lk_load<T, TAIL>(bz + (b * a.V + (size_t)v) * a.D + k.col, k.valid, z);
    const double prec = c.az + c.lik1 * (double)count, asum = c.ax + c.an;
    double sr[N];
#pragma unroll
    for (int e = 0; e < N; ++e) sr[e] = a.s * (((double)z[e] + a.s * acc[e]) / prec);
    const int cnt = run > sub ? ((run - sub - 1) >> ls) + 1 : 0;
#pragma unroll
    for (int i = 0; i < kKeep; ++i)
        if (i < cnt) lk_position_out<T, TAIL>(a, asum, k, b, pj[i], sr, rows[i], damping, b_old, out, r_out);
}

// the partial sums of a heavy run: {token, first slot, one behind the last, index among the heavy runs}
template <typename T, bool TAIL, int MODE>
__global__ __launch_bounds__(kBlock) void lookup_join_kernel(LkArgs a, const LkItem* __restrict__ joins, unsigned n_joins,
                                                             const LkScal* __restrict__ scal, const T* __restrict__ bz,
                                                             const double* __restrict__ partials, double damping, const T* b_old, T* out,
                                                             T* __restrict__ r_out, double* __restrict__ r_ws) {
    constexpr int N = LkVec<T>::N;
    __shared__ double sm[kBlock / kWave][kWave][N];
    const size_t b = blockIdx.y;
    const unsigned blk = blockIdx.x / a.tiles, tile = blockIdx.x - blk * a.tiles;
    const LkLane k = lk_lane<T>(a.lw, tile, a.D);
    LkScal c{};
    if (MODE != LK_GRAD) c = scal[b];
    const LkItem it = joins[blk];
    const int v = it.token, G = kBlock >> a.lw, count = a.off[v + 1] - a.off[v];
    double acc[N];
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = 0.0;
    const double* p = partials + b * a.n_slots * a.D + k.col;
#pragma unroll 4
    for (int j = it.start + k.group; j < it.end; j += G) {
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] += e < k.valid ? p[(size_t)j * a.D + e] : 0.0;
    }
    lk_block_join<N>(k, acc, sm);
    if (threadIdx.x >= (1u << a.lw) || k.valid <= 0) return;
    if (MODE != LK_FWD) {
        lk_row_out<T, TAIL, MODE>(a, c, k, b, v, count, acc, bz, damping, b_old, out, r_out);
        return;
    }
    T z[N];
    lk_load<T, TAIL>(bz + (b * a.V + (size_t)v) * a.D + k.col, k.valid, z);
    const double prec = c.az + c.lik1 * (double)count;
    double* r = r_ws + (b * n_joins + (size_t)it.slot) * a.D + k.col;
#pragma unroll
    for (int e = 0; e < N; ++e)
        if (e < k.valid) r[e] = a.s * (((double)z[e] + a.s * acc[e]) / prec);
}

// the message to the positions of the heavy runs and to the padded ones: {-, start, end, index of the heavy run or -1}
template <typename T, bool TAIL>
__global__ __launch_bounds__(kBlock) void lookup_spread_kernel(LkArgs a, const LkItem* __restrict__ spreads, unsigned n_joins,
                                                               const LkScal* __restrict__ scal, const double* __restrict__ r_ws,
                                                               const T* __restrict__ bx, double damping, const T* b_old, T* out,
                                                               T* __restrict__ r_out) {
    constexpr int N = LkVec<T>::N, UR = 4;
    const size_t b = blockIdx.y;
    const unsigned blk = blockIdx.x / a.tiles, tile = blockIdx.x - blk * a.tiles;
    const LkLane k = lk_lane<T>(a.lw, tile, a.D);
    if (k.valid <= 0) return;
    const LkItem it = spreads[blk];
    const double asum = scal[b].ax + scal[b].an;
    double sr[N];
#pragma unroll
    for (int e = 0; e < N; ++e)
        sr[e] = it.slot >= 0 && e < k.valid ? r_ws[(b * n_joins + (size_t)it.slot) * a.D + k.col + e] : 0.0;
    const int G = kBlock >> a.lw;
    for (int j = it.start + k.group; j < it.end; j += UR * G) {
        int t[UR];
        T v[UR][N];
#pragma unroll
        for (int i = 0; i < UR; ++i) t[i] = j + i * G < it.end ? a.perm[j + i * G] : -1;
#pragma unroll
        for (int i = 0; i < UR; ++i)
            if (t[i] >= 0) lk_load<T, TAIL>(bx + (b * a.T + (size_t)t[i]) * a.D + k.col, k.valid, v[i]);
#pragma unroll
        for (int i = 0; i < UR; ++i)
            if (t[i] >= 0) lk_position_out<T, TAIL>(a, asum, k, b, t[i], sr, v[i], damping, b_old, out, r_out);
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
        std::vector<int> off(n_rows + 1, 0), perm(n_pos);
        for (size_t t = 0; t < n_pos; ++t)
            if (tokens_h[t] >= 0) ++off[(size_t)tokens_h[t] + 1];
        std::vector<int> counts(off.begin() + 1, off.end());
        for (size_t v = 0; v < n_rows; ++v) off[v + 1] += off[v];
        const size_t seen = (size_t)off[n_rows];
        {
            std::vector<int> at(off.begin(), off.end() - 1);
            size_t pad = seen;
            for (size_t t = 0; t < n_pos; ++t) perm[tokens_h[t] >= 0 ? (size_t)at[(size_t)tokens_h[t]]++ : pad++] = (int)t;
        }
        // lanes per row and the cut by run lengths (lookup_rows_kernel)
        const size_t piece = 16 / dtype_size(dtype), pieces = (n_cols + piece - 1) / piece;
        int lw = 0;
        while (lw < 6 && ((size_t)1 << lw) < pieces) ++lw;
        const size_t tiles = (pieces + ((size_t)1 << lw) - 1) >> lw;
        const int per_wave = kKeep << (6 - lw), per_block = kKeep << (8 - lw);
        std::vector<LkItem> chunks, runs, joins, spreads;
        std::vector<int> waves;
        for (size_t v = 0; v < n_rows; ++v) {
            const int c = counts[v], j0 = off[v];
            if (c <= kKeep) continue;
            if (c <= per_wave) {
                waves.push_back((int)v);
            } else if (c <= per_block) {
                runs.push_back(LkItem{(int)v, j0, j0 + c, -1});
            } else {
                // at most 256 partial sums per run: the second launch adds them in one workgroup
                const long step = (long)per_block * (((long)c + 256L * per_block - 1) / (256L * per_block));
                const int slot0 = (int)chunks.size();
                for (long j = 0; j < c; j += step) {
                    const int lo = j0 + (int)j, hi = j0 + (int)std::min((long)c, j + step);
                    chunks.push_back(LkItem{(int)v, lo, hi, (int)chunks.size()});
                    spreads.push_back(LkItem{(int)v, lo, hi, (int)joins.size()});
                }
                joins.push_back(LkItem{(int)v, slot0, (int)chunks.size(), (int)joins.size()});
            }
        }
        for (size_t j = seen; j < n_pos; j += (size_t)per_block)
            spreads.push_back(LkItem{-1, (int)j, (int)std::min(n_pos, j + (size_t)per_block), -1});
        const size_t n_slots = chunks.size();
        chunks.insert(chunks.end(), runs.begin(), runs.end());
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
        // one allocation: the arrays one behind the other
        std::vector<char> host;
        auto put = [&host](const void* p, size_t bytes) {
            const size_t at = host.size();
            host.resize(at + ((bytes + 255) & ~(size_t)255));
            if (bytes) memcpy(host.data() + at, p, bytes);
            return at;
        };
        const size_t o_tok = put(tokens_h, n_pos * 4), o_perm = put(perm.data(), n_pos * 4), o_off = put(off.data(), (n_rows + 1) * 4);
        const size_t o_cnt = put(cval.data(), 2 * K * 8), o_items = put(chunks.data(), chunks.size() * sizeof(LkItem));
        const size_t o_joins = put(joins.data(), joins.size() * sizeof(LkItem)), o_spreads = put(spreads.data(), spreads.size() * sizeof(LkItem));
        const size_t o_waves = put(waves.data(), waves.size() * 4);
        tramp_lookup* lk = new tramp_lookup();
        *lk = tramp_lookup{};
        (void)hipSetDevice(ctx->device);
        if (hipMalloc(&lk->mem, host.size()) != hipSuccess) {
            (void)hipGetLastError();
            delete lk;
            return tramp_fail(ctx, TRAMP_ENOMEM, "tramp_lookup_create", "hipMalloc failed");
        }
        char* m = static_cast<char*>(lk->mem);
        hipError_t e = hipMemcpyAsync(m, host.data(), host.size(), hipMemcpyHostToDevice, ctx->stream);
        if (e == hipSuccess) e = hipStreamSynchronize(ctx->stream);      // the host array ends here
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
        lk->tok = reinterpret_cast<const int*>(m + o_tok);
        lk->perm = reinterpret_cast<const int*>(m + o_perm);
        lk->off = reinterpret_cast<const int*>(m + o_off);
        lk->cnt = reinterpret_cast<const double*>(m + o_cnt);
        lk->K = (int)K;
        lk->items = reinterpret_cast<const LkItem*>(m + o_items);
        lk->joins = reinterpret_cast<const LkItem*>(m + o_joins);
        lk->spreads = reinterpret_cast<const LkItem*>(m + o_spreads);
        lk->waves = reinterpret_cast<const int*>(m + o_waves);
        lk->n_items = (unsigned)chunks.size();
        lk->n_joins = (unsigned)joins.size();
        lk->n_spreads = (unsigned)spreads.size();
        lk->n_waves = (unsigned)waves.size();
        lk->n_slots = (unsigned)n_slots;
        lk->lw = lw;
        lk->tiles = (unsigned)tiles;
        *out = lk;
        return TRAMP_OK;
    } catch (const std::exception&) {
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

// the rows fill whole pieces: no tails to look after
static bool lk_whole(const tramp_lookup* lk) { return lk->D % (16 / dtype_size(lk->dtype)) == 0; }

template <typename T>
static int lookup_apply(tramp_ctx* ctx, const tramp_lookup* lk, size_t batch, const T* z, T* x) {
    constexpr size_t N = LkVec<T>::N;
    if (lk->D == 1) {
        const size_t nb = (lk->T + kBlock * N - 1) / (kBlock * N);
        hipLaunchKernelGGL((lookup_apply1_kernel<T>), dim3((unsigned)nb, (unsigned)batch), dim3(kBlock), 0, ctx->stream, lk->V, lk->T,
                           lk->s, lk->tok, z, x);
    } else {
        const size_t per = (size_t)4 * (kBlock >> lk->lw), nb = (lk->T + per - 1) / per * lk->tiles;
        TRAMP_REQUIRE(ctx, nb < 0x7fffffffu);
        dim3 grid((unsigned)nb, (unsigned)batch);
        if (lk_whole(lk))
            hipLaunchKernelGGL((lookup_apply_kernel<T, false>), grid, dim3(kBlock), 0, ctx->stream, lk->V, lk->D, lk->T, lk->s, lk->lw,
                               lk->tiles, lk->tok, z, x);
        else
            hipLaunchKernelGGL((lookup_apply_kernel<T, true>), grid, dim3(kBlock), 0, ctx->stream, lk->V, lk->D, lk->T, lk->s, lk->lw,
                               lk->tiles, lk->tok, z, x);
    }
    TRAMP_LAUNCH_CHECK(ctx);
    return TRAMP_OK;
}

extern "C" int tramp_lookup_apply(tramp_ctx* ctx, tramp_lookup* lk, size_t batch, const void* z_d, void* x_d) {
    LK_REQUIRE_CALL(ctx, lk, batch);
    TRAMP_REQUIRE(ctx, z_d && x_d && z_d != x_d);
    if (!batch) return TRAMP_OK;
    return lk->dtype == TRAMP_F64 ? lookup_apply<double>(ctx, lk, batch, (const double*)z_d, (double*)x_d)
                                  : lookup_apply<float>(ctx, lk, batch, (const float*)z_d, (float*)x_d);
}

// sums over the runs and what MODE makes of them; ctx->ws holds [scalars | partial sums | r of the heavy runs]
template <typename T, bool TAIL, int MODE>
static int launch_rows(tramp_ctx* ctx, const tramp_lookup* lk, size_t batch, size_t ws_at, const LkScal* scal, const T* bz, const T* x,
                       double damping, const T* b_old, T* out, T* r_out) {
    double* partials = reinterpret_cast<double*>(reinterpret_cast<char*>(ctx->ws) + ws_at);
    double* r_ws = partials + batch * lk->n_slots * lk->D;
    LkArgs a{};
    a.off = lk->off;
    a.perm = lk->perm;
    a.items = lk->items;
    a.waves = lk->waves;
    a.V = lk->V;
    a.D = lk->D;
    a.T = lk->T;
    a.n_items = lk->n_items;
    a.n_waves = lk->n_waves;
    a.wave_blocks = (lk->n_waves + kBlock / kWave - 1) / (kBlock / kWave);
    a.tiles = lk->tiles;
    a.n_slots = lk->n_slots;
    a.lw = lk->lw;
    a.s = lk->s;
    const size_t G = kBlock >> lk->lw;
    const size_t blocks = lk->n_items + a.wave_blocks + (lk->V + G - 1) / G;
    TRAMP_REQUIRE(ctx, blocks * lk->tiles < 0x7fffffffu && (size_t)lk->n_spreads * lk->tiles < 0x7fffffffu);
    a.blocks = (unsigned)blocks;
    hipLaunchKernelGGL((lookup_rows_kernel<T, TAIL, MODE>), dim3((unsigned)(blocks * lk->tiles), (unsigned)batch), dim3(kBlock), 0,
                       ctx->stream, a, scal, bz, x, damping, b_old, out, r_out, partials);
    if (lk->n_joins)
        hipLaunchKernelGGL((lookup_join_kernel<T, TAIL, MODE>), dim3(lk->n_joins * lk->tiles, (unsigned)batch), dim3(kBlock), 0,
                           ctx->stream, a, lk->joins, lk->n_joins, scal, bz, partials, damping, b_old, out, r_out, r_ws);
    if (MODE == LK_FWD && lk->n_spreads)
        hipLaunchKernelGGL((lookup_spread_kernel<T, TAIL>), dim3(lk->n_spreads * lk->tiles, (unsigned)batch), dim3(kBlock), 0,
                           ctx->stream, a, lk->spreads, lk->n_joins, scal, r_ws, x, damping, b_old, out, r_out);
    TRAMP_LAUNCH_CHECK(ctx);
    return TRAMP_OK;
}

static size_t scal_bytes(size_t batch) { return (batch * sizeof(LkScal) + 255) & ~(size_t)255; }

static int lookup_ws(tramp_ctx* ctx, const tramp_lookup* lk, size_t batch) {
    return tramp_ws_reserve(ctx, scal_bytes(batch) + batch * ((size_t)lk->n_slots + lk->n_joins) * lk->D * sizeof(double));
}

template <typename T, int MODE>
static int run_rows(tramp_ctx* ctx, const tramp_lookup* lk, size_t batch, const LkScal* scal, const T* bz, const T* x, double damping,
                    const T* b_old, T* out, T* r_out) {
    return lk_whole(lk) ? launch_rows<T, false, MODE>(ctx, lk, batch, scal_bytes(batch), scal, bz, x, damping, b_old, out, r_out)
                        : launch_rows<T, true, MODE>(ctx, lk, batch, scal_bytes(batch), scal, bz, x, damping, b_old, out, r_out);
}

extern "C" int tramp_lookup_gradient(tramp_ctx* ctx, tramp_lookup* lk, size_t batch, const void* x_d, void* g_d) {
    LK_REQUIRE_CALL(ctx, lk, batch);
    TRAMP_REQUIRE(ctx, x_d && g_d && x_d != g_d);
    if (!batch) return TRAMP_OK;
    int rc = lookup_ws(ctx, lk, batch);
    if (rc) return rc;
    if (lk->dtype == TRAMP_F64)
        return run_rows<double, LK_GRAD>(ctx, lk, batch, nullptr, nullptr, (const double*)x_d, 0.0, nullptr, (double*)g_d, nullptr);
    return run_rows<float, LK_GRAD>(ctx, lk, batch, nullptr, nullptr, (const float*)x_d, 0.0, nullptr, (float*)g_d, nullptr);
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
    int rc = lookup_ws(ctx, lk, batch);
    if (rc) return rc;
    LkScal* scal = reinterpret_cast<LkScal*>(ctx->ws);
    launch_scalars(ctx, lk, dir, batch, az_d, ax_d, damping, a_old_d, scal, v_d, a_new_d, nullptr);
    return dir == TRAMP_BWD ? run_rows<T, LK_BWD>(ctx, lk, batch, scal, bz, bx, damping, b_old, b_new, r_d)
                            : run_rows<T, LK_FWD>(ctx, lk, batch, scal, bz, bx, damping, b_old, b_new, r_d);
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
