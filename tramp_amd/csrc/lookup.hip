// lookup.hip - lookup channel x_t = scale z[token_t] of a table z of V rows and D columns.
//
// The linear factor of categorical data: W [T D, V D] has one entry `scale` per row (none where the position is padded), so
// W^T W = scale^2 diag(count_v) (x) I_D and every quantity of LinearChannel (tramp/channels/linear/linear_channel.py:58-132)
// is closed form in the counts.  With  g_v = scale sum_{t: token_t = v} bx_t  (the adjoint),  lik_v = ax scale^2 count_v,
// prec_v = az + lik_v:
//     r_v  = (bz_v + g_v) / prec_v                                  posterior mean of the table
//     rx_t = scale r_{token_t}                                      posterior mean of the positions (0 where padded)
//     vz   = (1/V) sum_v 1 / prec_v            vx = (scale^2 / T) sum_v count_v / prec_v
// and the messages a' = clip(1/v - a), b' = r (a + a') - b (tramp/base.py:250-255).  Both ends of 1/v - a, the b' to the table and
// the b' to a position that reads its row alone are sums without cancellation, which is how they are formed here:
//     1/vz - az = [(1/V) sum_v lik_v / prec_v] / vz
//     1/vx - ax = [padded / T + (1/T) sum_v count_v (az + ax scale^2 (count_v - 1)) / prec_v] / vx
//     b'_v = [g_v (az + a') + bz_v (a' - lik_v)] / prec_v
//     b'_t = [s (ax + a') bz_v + (s^2 a' - az) bx_t] / prec_v       where t is the only position of v; otherwise rx_t (ax + a') - bx_t
// (a table of 10^5 rows of which ten are read has a' of order 10^-4 az: the difference would lose the digits of f64).
//
// The positions are sorted by token once, at creation (perm, off): the adjoint is a sum over runs, in a fixed order, without
// atomics, the same bits every time.  All arithmetic is in double and rounded once to the element type at the store: the
// passes are bound by memory (a few operations per element), the conversions are free next to the loads.
#include "common.h"
#include "lookup_buffers.h"
#include "lookup_grid.h"
#include "tramp_math.h"

#include <algorithm>
#include <new>
#include <type_traits>
#include <vector>

struct LkItem {
    int token, start, end, slot;      // positions perm[start .. end); slot: by list (tramp_lookup)
};

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
    const LkItem* chunks;        // heavy runs in chunks, one partial sum each
    const LkItem* joins;         // {token, first chunk, one behind the last, index}
    const LkItem* spreads;       // the chunks' positions
    const LkItem* runs;          // runs for one workgroup
    const LkItem* waves;         // runs for one wave
    const LkItem* light;         // the shorter runs, by falling length; slot: the first position, which the runs of one are read by
    const int* empty;            // rows without positions
    const int* idx;              // [V] place among the runs of two and more positions (short rows only)
    const int* code;             // [T] that place, -1 where padded, -2 - token where the run is this position (short rows only)
    int K;
    unsigned n_chunks, n_joins, n_spreads, n_runs, n_waves, n_light, n_light2, n_empty, n_multi;
    int lw;                      // log2 of the lanes per row
    unsigned tiles;              // column tiles per row
    int row;                     // LK_TAIL / LK_WHOLE / LK_LINES
    bool short_rows;             // under half a line: the message to x may go in the order of the positions
    bool long_runs;              // runs of one workgroup that its registers do not hold
};

// what the kernels need of one instance, written by lk_scalars
struct LkScal {
    double az, ax, an, lik1;     // floored az, ax, a' before damping, ax scale^2
};

// ---------------------------------------------------------------- scalars
// v, a' and n_eff of every instance from the table of distinct counts (n of them sum to at least n(n-1)/2 positions: 1414
// at 10^6 positions), one workgroup per instance: a few us, bound by its latency, so it rides in a launch that is there anyway.
struct LkScalArgs {
    const double* cnt;
    const double* az;
    const double* ax;
    const double* a_old;
    LkScal* scal;
    double* v_out;
    double* a_new_out;
    double* n_eff_out;
    double V, T, padded, s, damping;
    int K, dir;
};

// every workgroup that calls it ends with the same bits; `write`: this one stores them
__device__ __forceinline__ LkScal lk_scalars(const LkScalArgs& q, size_t b, bool write) {
    __shared__ double smem[kBlock / kWave];
    const int K = q.K, dir = q.dir;
    const double* cnt = q.cnt;
    const double s = q.s;
    const double ax = q.ax[b], az_in = q.az[b];
    const double az = dir == TRAMP_BWD && az_in < 1e-11 ? 1e-11 : az_in;       // linear_channel.py:92-94 (a NaN stays one)
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
    double v, an;
    if (dir == TRAMP_BWD) {
        v = sv / q.V;
        an = (sn / q.V) / v;
    } else {
        v = s * s * sv / q.T;
        an = ((q.padded + sn) / q.T) / v;
    }
    if (v > 1.7976931348623157e308) an = 0.0;                    // both precisions zero: 1 / v - a <= 0
    if (an < tmath::kAMin) an = tmath::kAMin;                    // (comparisons: a NaN passes through, tramp/base.py:252)
    if (an > tmath::kAMax) an = tmath::kAMax;
    const LkScal c{az, ax, an, lik1};
    if (write && threadIdx.x == 0) {
        if (q.scal) q.scal[b] = c;
        // a' before v: v may replace a_old, whose scalar load is only waited for where its value is used
        if (q.a_new_out) q.a_new_out[b] = q.damping != 0.0 ? q.damping * q.a_old[b] + (1.0 - q.damping) * an : an;
        if (q.v_out) q.v_out[b] = v;
        if (q.n_eff_out) q.n_eff_out[b] = se / q.V;
    }
    return c;
}

__global__ __launch_bounds__(kBlock) void lookup_scalars_kernel(LkScalArgs q) { (void)lk_scalars(q, blockIdx.x, true); }

// ---------------------------------------------------------------- rows in 16-byte pieces
// A row of D elements is walked by LPR lanes, one 16-byte piece (N elements) per lane: the power of two that holds the row, up to
// 64, and column tiles of LPR pieces where the row is longer (tramp_lookup_create).  The pieces start wherever the row does: a
// 16-byte access needs element alignment only, so odd D and views cost nothing but the last piece of a row (LK_TAIL).
template <typename T> struct LkVec;
template <> struct LkVec<float> {
    typedef float U __attribute__((ext_vector_type(4), aligned(4)));
    static constexpr int N = 4;
};
template <> struct LkVec<double> {
    typedef double U __attribute__((ext_vector_type(2), aligned(8)));
    static constexpr int N = 2;
};

// kinds of rows: LK_TAIL the last piece of a row is short; LK_WHOLE whole pieces; LK_LINES whole 128-byte lines, which nobody
// else touches: read and written past the caches where they are used once
enum { LK_TAIL = 0, LK_WHOLE = 1, LK_LINES = 2 };

template <typename T, int ROW, bool ONCE = false>
__device__ __forceinline__ void lk_load(const T* __restrict__ p, int valid, T (&v)[LkVec<T>::N]) {
    constexpr int N = LkVec<T>::N;
    using U = typename LkVec<T>::U;
    if (ROW != LK_TAIL || valid == N) {
        const U u = ROW == LK_LINES && ONCE ? __builtin_nontemporal_load(reinterpret_cast<const U*>(p)) : *reinterpret_cast<const U*>(p);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = u[i];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = i < valid ? p[i] : T(0);
    }
}

template <typename T, int ROW>
__device__ __forceinline__ void lk_store(T* p, int valid, const T (&v)[LkVec<T>::N]) {
    constexpr int N = LkVec<T>::N;
    using U = typename LkVec<T>::U;
    if (ROW != LK_TAIL || valid == N) {
        U u;
#pragma unroll
        for (int i = 0; i < N; ++i) u[i] = v[i];
        if (ROW == LK_LINES)
            __builtin_nontemporal_store(u, reinterpret_cast<U*>(p));
        else
            *reinterpret_cast<U*>(p) = u;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < valid) p[i] = v[i];
    }
}

// one column in its own order: pieces side by side past the caches, which are left to what is gathered (lookup of 64 x 100000 f64
// 53.7 -> 49.9 us, of 10^6 7.2 -> 6.1; message to x by position of 64 x 100000 f64 99.1 -> 95.4 us, read so too; one instance, whose x
// the sums have just read, 37.5 -> 38.5 if read so)
template <typename T> __device__ __forceinline__ void lk_stream_load(const T* __restrict__ p, int valid, T (&v)[LkVec<T>::N]) {
    if (valid == LkVec<T>::N)
        lk_load<T, LK_LINES, true>(p, valid, v);
    else
        lk_load<T, LK_TAIL>(p, valid, v);
}
template <typename T> __device__ __forceinline__ void lk_stream_store(T* p, int valid, const T (&v)[LkVec<T>::N]) {
    if (valid == LkVec<T>::N)
        lk_store<T, LK_LINES>(p, valid, v);
    else
        lk_store<T, LK_TAIL>(p, valid, v);
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

// Which instance, which workgroup of it, which column tile.  Workgroups go to the eight XCDs in turn; with `spread` the grid is
// one-dimensional and all workgroups of an instance get numbers of one residue modulo 8: its table and positions, read and
// written in the order of the tokens, then meet in one L2 (4 MiB) instead of in eight.
struct LkPlace {
    size_t b;
    unsigned blk, tile;
    bool in;
};
__device__ __forceinline__ LkPlace lk_place(unsigned blocks, unsigned tiles, unsigned batch, int spread) {
    LkPlace p;
    unsigned id = blockIdx.x;
    if (spread) {
        const unsigned per = blocks * tiles, j = id >> 3, r = j / per;
        p.b = (size_t)r * 8 + (id & 7);
        id = j - r * per;
    } else {
        p.b = blockIdx.y;
    }
    p.in = p.b < batch;
    p.blk = id / tiles;
    p.tile = id - p.blk * tiles;
    return p;
}

// ---------------------------------------------------------------- x = scale z[token]
// Bound by the write of x (and the read of the distinct rows of z).  Four rows per group in flight.  65536 positions of 1024 f32
// from 32000 rows, 316 MB: 46 us, 6.8 TB/s (a copy of that size from memory runs at 5.2; most of z comes from the cache, which
// the non-temporal stores of x leave alone: 80 us with ordinary ones).
template <typename T, int ROW>
__global__ __launch_bounds__(kBlock) void lookup_apply_kernel(size_t V, size_t D, size_t n_pos, double s, int lw, unsigned blocks,
                                                              unsigned tiles, unsigned batch, int spread, const int* __restrict__ tok,
                                                              const T* __restrict__ z, T* __restrict__ x) {
    constexpr int N = LkVec<T>::N, UR = 4;
    const LkPlace w = lk_place(blocks, tiles, batch, spread);
    const size_t b = w.b;
    const LkLane k = lk_lane<T>(lw, w.tile, D);
    if (!w.in || k.valid <= 0) return;
    const size_t G = kBlock >> lw;
    int row[UR];
    T v[UR][N];
    const size_t t0 = (size_t)w.blk * UR * G + k.group;
#pragma unroll
    for (int i = 0; i < UR; ++i) row[i] = t0 + i * G < n_pos ? tok[t0 + i * G] : -1;
#pragma unroll
    for (int i = 0; i < UR; ++i) {
        if (row[i] >= 0) {
            lk_load<T, ROW>(z + (b * V + (size_t)row[i]) * D + k.col, k.valid, v[i]);
#pragma unroll
            for (int e = 0; e < N; ++e) v[i][e] = T(s * (double)v[i][e]);
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) v[i][e] = T(0);
        }
    }
#pragma unroll
    for (int i = 0; i < UR; ++i)
        if (t0 + i * G < n_pos) lk_store<T, ROW>(x + (b * n_pos + t0 + i * G) * D + k.col, k.valid, v[i]);
}

// one column: N positions per lane, written as one piece; bound by the gathers (64 x 100000 f64 of 200000: 50 us)
template <typename T>
__global__ __launch_bounds__(kBlock) void lookup_apply1_kernel(size_t V, size_t n_pos, double s, unsigned blocks, unsigned batch, int spread,
                                                               const int* __restrict__ tok, const T* __restrict__ z, T* __restrict__ x) {
    constexpr int N = LkVec<T>::N;
    const LkPlace w = lk_place(blocks, 1, batch, spread);
    const size_t b = w.b, t = ((size_t)w.blk * kBlock + threadIdx.x) * N;
    if (!w.in || t >= n_pos) return;
    const int valid = n_pos - t >= N ? N : (int)(n_pos - t);
    int row[N];
    T v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) row[i] = i < valid ? tok[t + i] : -1;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = row[i] >= 0 ? T(s * (double)z[b * V + (size_t)row[i]]) : T(0);
    lk_stream_store<T>(x + b * n_pos + t, valid, v);
}

// ---------------------------------------------------------------- sums over the runs
// The run lengths of real tokens differ by orders of magnitude, so the work is cut by them, at creation:
//   light  run <= kKeep                       one group, all rows of the run in flight at once (of none or one position: below)
//   wave   run <= kKeep * 64 / LPR            the groups of one wave, joined by a butterfly
//   block  run <= kKeep * 256 / LPR           the groups of one workgroup, the four waves joined through LDS (LONG: twice that)
//   heavy  longer                             chunks of a multiple of that, summed in a first launch (lookup_chunks_kernel),
//                                             the partial sums in double joined by one workgroup in the second
// In the first three every row stays in registers from the sum to the message that goes back to its position: the message to
// the positions reads bx once.  Only the heavy runs are read twice, the second time in a third launch.
// kKeep: 8 rows in flight per group leave 5 to 8 waves per SIMD; 16 leave 3 to 5 and cost a third (gradient 121 against 84 us,
// message to 10^6 positions of 64 columns 136 against 104 us), 4 make longer runs of every kind (89 and 103 us).
constexpr int kKeep = 8;
// Rows that no position reads (most rows of a table of many, in a batch of few) have a kind of their own, four per group, and the
// others come from the list, unless rows are short and want to be written side by side.  Gradient of 65536 x 1024 f32 to 32000 rows
// (20600 without positions) 78.6 -> 69.3 us, 133588 x 76 f64 to 172932 rows 105 -> 77, 8 x 201 x 71 f32 to 68544 rows 75 -> 40.
constexpr int kEmpty = 4;
// Rows that one position reads, two per group: gradient of 133588 x 76 f64 to 172932 rows 76.9 -> 70.8 us, the message to that table
// 96.4 -> 84.9, to those positions 99.8 -> 77.6.  Four cost registers: 68.5, 92.9 and 77.0, but message to 8 x 10007 x 21 f64 46 -> 50.
// Padded positions go with them (a launch of their own before: 31 x 152 f64 11.0 -> 8.1 us, 284412 x 9 f32, 30 % padded, 29.9 -> 23.5).
constexpr int kOne = 2;

struct LkArgs {
    const int* off;
    const int* perm;
    const LkItem* chunks;
    const LkItem* joins;
    const LkItem* runs;
    const LkItem* waves;
    const LkItem* light;         // null: all rows of the table (those of the kinds above left out)
    const int* empty;
    const int* idx;
    size_t V, D, T;
    unsigned n_chunks, n_joins, n_runs, n_waves, wave_blocks, n_light, light_blocks, n_single, n_pad, single_blocks, n_empty, n_multi, blocks, tiles, batch;
    size_t pad0;                 // the padded positions: perm[pad0 .. pad0 + n_pad), for the message to x
    unsigned n_lead;             // chunks summed in the launch of the runs (gradient)
    int lw, spread;
    double s;
};

// what is made of the sum of a run: the gradient, the message to the table, the message to its positions, scale times the mean,
// the row's share of the log-partition
enum { LK_GRAD = 0, LK_BWD = 1, LK_FWD = 2, LK_MEAN = 3, LK_LOGZ = 4 };

// rows perm[j0 + sub], perm[j0 + sub + S], ... of the run [j0, j0 + c), S = 1 << ls: added into acc, C in flight; KEEP: there are
// at most C and they stay in `rows`.
template <typename T, int ROW, int C, bool KEEP, bool ONCE>
__device__ __forceinline__ void lk_gather(const LkArgs& a, const T* __restrict__ xb, const LkLane& k, int j0, int c, int sub, int ls,
                                          double (&acc)[LkVec<T>::N], int (&pj)[C], T (&rows)[C][LkVec<T>::N]) {
    constexpr int N = LkVec<T>::N, Q = C < 4 ? C : 4;
    const int cnt = c > sub ? ((c - sub - 1) >> ls) + 1 : 0;
    const int* pp = a.perm + j0 + sub;
    for (int base = 0; base < cnt; base += C) {
#pragma unroll
        for (int q = 0; q < C; q += Q)
            if (base + q < cnt) {
#pragma unroll
                for (int i = q; i < q + Q; ++i) pj[i] = base + i < cnt ? pp[(size_t)(base + i) << ls] : -1;
            }
#pragma unroll
        for (int q = 0; q < C; q += Q)
            if (base + q < cnt) {
#pragma unroll
                for (int i = q; i < q + Q; ++i)
                    if (base + i < cnt) lk_load<T, ROW, ONCE>(xb + (size_t)pj[i] * a.D + k.col, k.valid, rows[i]);
            }
#pragma unroll
        for (int i = 0; i < C; ++i)
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

// the gradient or the message to the table
template <typename T, int ROW, int MODE>
__device__ __forceinline__ void lk_row_out(const LkArgs& a, const LkScal& c, const LkLane& k, size_t b, int v, int count,
                                           const double (&acc)[LkVec<T>::N], const T (&z)[LkVec<T>::N], double damping, const T* b_old,
                                           T* out, T* __restrict__ r_out) {
    constexpr int N = LkVec<T>::N;
    const size_t at = (b * a.V + (size_t)v) * a.D + k.col;
    T o[N];
    if (MODE == LK_GRAD) {
#pragma unroll
        for (int e = 0; e < N; ++e) o[e] = T(a.s * acc[e]);
    } else {
        const double lik = c.lik1 * (double)count, inv = 1.0 / (c.az + lik);
        const double mg = a.s * ((c.az + c.an) * inv), mz = (c.an - lik) * inv;
        T old[N];
        if (damping != 0.0) lk_load<T, ROW>(b_old + at, k.valid, old);
#pragma unroll
        for (int e = 0; e < N; ++e) {
            double m = mg * acc[e] + mz * (double)z[e];
            if (damping != 0.0) m = damping * (double)old[e] + (1.0 - damping) * m;
            o[e] = T(m);
        }
        if (r_out) {
            T r[N];
#pragma unroll
            for (int e = 0; e < N; ++e) r[e] = T(((double)z[e] + a.s * acc[e]) * inv);
            lk_store<T, ROW>(r_out + at, k.valid, r);
        }
    }
    lk_store<T, ROW>(out + at, k.valid, o);
}

// the message m to one position, and rx = scale r
template <typename T, int ROW>
__device__ __forceinline__ void lk_position_store(const LkArgs& a, const LkLane& k, size_t b, size_t t, const double (&m)[LkVec<T>::N],
                                                  const double (&sr)[LkVec<T>::N], double damping, const T* b_old, T* out,
                                                  T* __restrict__ r_out) {
    constexpr int N = LkVec<T>::N;
    const size_t at = (b * a.T + t) * a.D + k.col;
    T o[N], old[N];
    if (damping != 0.0) lk_load<T, ROW>(b_old + at, k.valid, old);
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] = T(damping != 0.0 ? damping * (double)old[e] + (1.0 - damping) * m[e] : m[e]);
    lk_store<T, ROW>(out + at, k.valid, o);
    if (r_out) {
#pragma unroll
        for (int e = 0; e < N; ++e) o[e] = T(sr[e]);
        lk_store<T, ROW>(r_out + at, k.valid, o);
    }
}

// b' = rx (ax + a') - bx
template <typename T, int ROW>
__device__ __forceinline__ void lk_position_out(const LkArgs& a, double asum, const LkLane& k, size_t b, size_t t,
                                                const double (&sr)[LkVec<T>::N], const T (&bx)[LkVec<T>::N], double damping, const T* b_old,
                                                T* out, T* __restrict__ r_out) {
    constexpr int N = LkVec<T>::N;
    double m[N];
#pragma unroll
    for (int e = 0; e < N; ++e) m[e] = sr[e] * asum - (double)bx[e];
    lk_position_store<T, ROW>(a, k, b, t, m, sr, damping, b_old, out, r_out);
}

// A position alone in its run: b' = kz bz + kx bx.  Where ax s^2 is far above az, rx (ax + a') and bx agree in most of their digits
// (a' is about az / s^2) and the difference would be left with none of bz's; kz bz and kx bx do not cancel.  A longer run says
// itself what bx does not: its difference is off by roundings of bx, as that of the definition.
struct LkOne {
    double mean, kz, kx;             // rx = mean (bz + s bx)
};
__device__ __forceinline__ LkOne lk_one(const LkScal& c, double s) {
    const double inv = 1.0 / (c.az + c.lik1), mean = s * inv;
    return LkOne{mean, mean * (c.ax + c.an), fma(s * s, c.an, -c.az) * inv};
}

// the partial sum of a chunk of a heavy run
template <typename T, int ROW, bool ONCE>
__device__ __forceinline__ void lk_chunk(const LkArgs& a, const LkLane& k, size_t b, unsigned blk, const T* __restrict__ xb,
                                         double* __restrict__ partials, double (*sm)[kWave][LkVec<T>::N]) {
    constexpr int N = LkVec<T>::N;
    const LkItem it = a.chunks[blk];
    double acc[N];
    int pj[kKeep];
    T rows[kKeep][N];
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = 0.0;
    if (k.valid > 0) lk_gather<T, ROW, kKeep, false, ONCE>(a, xb, k, it.start, it.end - it.start, k.group, 8 - a.lw, acc, pj, rows);
    lk_block_join<N>(k, acc, sm);
    if (threadIdx.x >= (1u << a.lw) || k.valid <= 0) return;
    double* p = partials + (b * a.n_chunks + (size_t)it.slot) * a.D + k.col;
#pragma unroll
    for (int e = 0; e < N; ++e)
        if (e < k.valid) p[e] = acc[e];
}

// First launch: the partial sums of the heavy runs; one more workgroup per instance makes its scalars.  Bound by the read of their
// positions: 622000 of 64 f32 (of 10^6 over 50000 rows, Zipf), 159 MB, 35 us, 4.6 TB/s.
template <typename T, int ROW, bool ONCE>
__global__ __launch_bounds__(kBlock) void lookup_chunks_kernel(LkArgs a, LkScalArgs q, const T* __restrict__ x, double* __restrict__ partials) {
    __shared__ double sm[kBlock / kWave][kWave][LkVec<T>::N];
    const size_t b = blockIdx.y;
    if (blockIdx.x == a.n_chunks * a.tiles) {
        (void)lk_scalars(q, b, true);
        return;
    }
    const unsigned blk = blockIdx.x / a.tiles;
    const LkLane k = lk_lane<T>(a.lw, blockIdx.x - blk * a.tiles, a.D);
    lk_chunk<T, ROW, ONCE>(a, k, b, blk, x + b * a.T * a.D, partials, sm);
}

// Second launch: every run.  Workgroups, in this order: joins of the partial sums, block runs, wave runs, light ones, rows of one
// position, rows of none.  The gradient needs no scalars: with short rows its chunks lead this launch and only their joins are
// left for another.
// Bound by the bytes where a row fills its lines: the other 378000 positions of that message, 207 MB read and written, 47 us,
// 4.4 TB/s; gradient of 65536 x 1024 f32 to 32000 rows 246 MB 46 us, 5.3 TB/s, after 23 us for 110 MB of heavy runs.  Rows that
// share lines are bound by the lines: 168 bytes touch 2.3 of 128 on average, message of 8 x 80021 x 21 f64 to 10007 rows 34 us;
// one column by lines fetched again: every XCD gathers from all of x, more than its L2 of 4 MiB holds, and the 8 MB of 1000001 f64
// come past the L2s eleven times, 88 MB in 17 us.
template <typename T, int ROW, int MODE, bool SELF, bool LONG>
__global__ __launch_bounds__(kBlock) void lookup_rows_kernel(LkArgs a, LkScalArgs q, const LkScal* __restrict__ scal, const T* __restrict__ bz,
                                                             const T* __restrict__ x, double damping, const T* b_old, T* out,
                                                             T* __restrict__ r_out, double* __restrict__ partials,
                                                             double* __restrict__ sr_ws) {
    constexpr int N = LkVec<T>::N;
    __shared__ double sm[kBlock / kWave][kWave][N];
    const LkPlace place = lk_place(a.blocks, a.tiles, a.batch, a.spread);
    if (!place.in) return;
    const size_t b = place.b;
    unsigned blk = place.blk;
    const LkLane k = lk_lane<T>(a.lw, place.tile, a.D);
    LkScal c{};
    if (MODE != LK_GRAD) c = SELF ? lk_scalars(q, b, place.blk == 0 && place.tile == 0) : scal[b];
    const T* xb = x + b * a.T * a.D;
    if (MODE == LK_GRAD && ROW != LK_LINES) {                      // lines are no short rows
        if (blk < a.n_lead) {
            lk_chunk<T, ROW, true>(a, k, b, blk, xb, partials, sm);
            return;
        }
        blk -= a.n_lead;
    }
    const bool act = k.valid > 0;
    double acc[N];
    int pj[kKeep];
    T rows[kKeep][N], z[N];
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = 0.0;
    int v, j0, count, sub, ls, place_ws = -1;
    bool first = true;
    // the row of the table is asked for as soon as it is known, the sum comes later
    const auto row_of = [&](int v) {
        if (MODE != LK_GRAD && act) lk_load<T, ROW, MODE == LK_BWD>(bz + (b * a.V + (size_t)v) * a.D + k.col, k.valid, z);
    };
    if (blk < a.n_joins) {
        const LkItem it = a.joins[blk];
        v = it.token;
        row_of(v);
        count = a.off[v + 1] - a.off[v];
        const int G = kBlock >> a.lw;
        const double* p = partials + b * a.n_chunks * a.D + k.col;
#pragma unroll 4
        for (int j = it.start + k.group; j < it.end; j += G) {
#pragma unroll
            for (int e = 0; e < N; ++e) acc[e] += e < k.valid ? p[(size_t)j * a.D + e] : 0.0;
        }
        lk_block_join<N>(k, acc, sm);
        first = threadIdx.x < (1u << a.lw);
        place_ws = it.slot;
        sub = ls = j0 = 0;
    } else if ((blk -= a.n_joins) < a.n_runs) {
        const LkItem it = a.runs[blk];
        v = it.token;
        row_of(v);
        j0 = it.start;
        count = it.end - it.start;
        sub = k.group;
        ls = 8 - a.lw;
        first = threadIdx.x < (1u << a.lw);
        if (act) lk_gather<T, ROW, kKeep, MODE == LK_FWD && !LONG, true>(a, xb, k, j0, count, sub, ls, acc, pj, rows);
        lk_block_join<N>(k, acc, sm);
    } else {
        blk -= a.n_runs;
        if (blk < a.wave_blocks) {
            const unsigned w = blk * (kBlock / kWave) + (threadIdx.x >> 6);
            if (w >= a.n_waves) return;
            const LkItem it = a.waves[w];
            v = it.token;
            row_of(v);
            j0 = it.start;
            count = it.end - it.start;
            sub = (threadIdx.x & 63) >> a.lw;
            ls = 6 - a.lw;
            first = (threadIdx.x & 63) < (1u << a.lw);
        } else if ((MODE == LK_GRAD || MODE == LK_BWD || MODE == LK_FWD) && blk >= a.wave_blocks + a.light_blocks &&
                   blk < a.wave_blocks + a.light_blocks + a.single_blocks) {
            // rows that one position reads, two per group; behind them the padded positions (token -2), whose rx is 0
            const size_t G = kBlock >> a.lw, u0 = (size_t)(blk - a.wave_blocks - a.light_blocks) * kOne * G + k.group;
            LkItem it[kOne];
            T xs[kOne][N], zs[kOne][N];
            if (!act) return;
#pragma unroll
            for (int i = 0; i < kOne; ++i) {
                const size_t u = u0 + i * G;
                it[i] = u < a.n_single ? a.light[a.n_light + u] : LkItem{-1, 0, 0, 0};
                if (MODE == LK_FWD && u >= a.n_single && u - a.n_single < a.n_pad) it[i] = LkItem{-2, 0, 0, a.perm[a.pad0 + (u - a.n_single)]};
            }
#pragma unroll
            for (int i = 0; i < kOne; ++i)
                if (it[i].token != -1) {
                    lk_load<T, ROW, true>(xb + (size_t)it[i].slot * a.D + k.col, k.valid, xs[i]);
                    if (MODE != LK_GRAD && it[i].token >= 0) lk_load<T, ROW, MODE == LK_BWD>(bz + (b * a.V + (size_t)it[i].token) * a.D + k.col, k.valid, zs[i]);
                }
            const LkOne one = lk_one(c, a.s);
#pragma unroll
            for (int i = 0; i < kOne; ++i) {
                if (it[i].token == -1) continue;
                if (MODE == LK_FWD) {
                    double sr[N], m[N];
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        const double bz_e = (double)zs[i][e], bx_e = (double)xs[i][e];
                        sr[e] = it[i].token >= 0 ? one.mean * (bz_e + a.s * bx_e) : 0.0;
                        m[e] = it[i].token >= 0 ? one.kz * bz_e + one.kx * bx_e : 0.0 * (c.ax + c.an) - bx_e;
                    }
                    lk_position_store<T, ROW>(a, k, b, (size_t)it[i].slot, m, sr, damping, b_old, out, r_out);
                } else {
#pragma unroll
                    for (int e = 0; e < N; ++e) acc[e] = 0.0 + (double)xs[i][e];
                    lk_row_out<T, ROW, MODE>(a, c, k, b, it[i].token, 1, acc, zs[i], damping, b_old, out, r_out);
                }
            }
            return;
        } else if ((MODE == LK_GRAD || MODE == LK_BWD) && blk >= a.wave_blocks + a.light_blocks) {
            // rows that no position reads, four per group: the table alone makes their result
            const size_t G = kBlock >> a.lw, u0 = (size_t)(blk - a.wave_blocks - a.light_blocks - a.single_blocks) * kEmpty * G + k.group;
            int row[kEmpty];
            T zs[kEmpty][N];
            if (!act) return;
#pragma unroll
            for (int i = 0; i < kEmpty; ++i) row[i] = u0 + i * G < a.n_empty ? a.empty[u0 + i * G] : -1;
#pragma unroll
            for (int i = 0; i < kEmpty; ++i)
                if (MODE == LK_BWD && row[i] >= 0) lk_load<T, ROW, true>(bz + (b * a.V + (size_t)row[i]) * a.D + k.col, k.valid, zs[i]);
#pragma unroll
            for (int i = 0; i < kEmpty; ++i)
                if (row[i] >= 0) lk_row_out<T, ROW, MODE>(a, c, k, b, row[i], 0, acc, zs[i], damping, b_old, out, r_out);
            return;
        } else {
            const size_t u = (size_t)(blk - a.wave_blocks) * (kBlock >> a.lw) + k.group;
            if (u >= a.n_light) return;
            sub = 0;
            ls = 0;
            if (a.light) {
                const LkItem it = a.light[u];
                v = it.token;
                row_of(v);
                j0 = it.start;
                count = it.end - it.start;
            } else {
                v = (int)u;
                row_of(v);
                j0 = a.off[v];
                count = a.off[v + 1] - j0;
            }
        }
        if (ls == 0 && count > kKeep) return;                      // of another kind
        // Most runs are of one or two positions.  Where a row costs instructions rather than bytes a wave goes no deeper than its
        // longest run (8 x 55612 positions of 78 f32 161 -> 155 us, 64 x 96196 of 6 f64 357 -> 320 us, gradient of 64 x 100000
        // f64 92 -> 78 us); whole lines and long f64 rows are better off with one body (100000 x 21 f64 119 us against 125).
        constexpr bool may = ROW == LK_TAIL || (ROW == LK_WHOLE && (MODE == LK_FWD || MODE == LK_MEAN));
        const bool shallow = may && (sizeof(T) == 4 || a.lw <= 2);
        if (shallow && MODE != LK_LOGZ && ls == 0 && !__any(count > 4)) {
            const auto run = [&](auto depth) {
                constexpr int C = decltype(depth)::value;
                int qj[C];
                T part[C][N];
                lk_gather<T, ROW, C, true, true>(a, xb, k, j0, count, 0, 0, acc, qj, part);
                if (MODE == LK_GRAD || MODE == LK_BWD) {
                    lk_row_out<T, ROW, MODE>(a, c, k, b, v, count, acc, z, damping, b_old, out, r_out);
                    return;
                }
                double sr[N];
                const double f = a.s / (c.az + c.lik1 * (double)count);
#pragma unroll
                for (int e = 0; e < N; ++e) sr[e] = f * ((double)z[e] + a.s * acc[e]);
                if (MODE == LK_MEAN) {
                    double* r = sr_ws + (b * a.n_multi + (size_t)a.idx[v]) * a.D + k.col;
#pragma unroll
                    for (int e = 0; e < N; ++e)
                        if (e < k.valid) r[e] = sr[e];
                    return;
                }
#pragma unroll
                for (int i = 0; i < C; ++i)
                    if (i < count) lk_position_out<T, ROW>(a, c.ax + c.an, k, b, (size_t)qj[i], sr, part[i], damping, b_old, out, r_out);
            };
            const bool two = __any(count > 1), four = __any(count > 2);
            if (!act) return;
            if (four)
                run(std::integral_constant<int, 4>{});
            else if (MODE == LK_FWD || MODE == LK_MEAN || two)     // these come from the list of runs of two and more
                run(std::integral_constant<int, 2>{});
            else
                run(std::integral_constant<int, 1>{});
            return;
        }
        if (act) lk_gather<T, ROW, kKeep, true, true>(a, xb, k, j0, count, sub, ls, acc, pj, rows);
        if (ls) lk_wave_join<N>(a.lw, acc);
    }
    if (MODE == LK_LOGZ) {
        // 1/2 sum (bz + g)^2 / prec + D/2 log(2 pi / prec) over this column tile of the row
        double h = 0.0;
        if (act) {
            const double prec = c.az + c.lik1 * (double)count, lg = 0.5 * log(2.0 * tmath::kPi / prec), half = 0.5 / prec;
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const double t = (double)z[e] + a.s * acc[e];
                if (e < k.valid) h += half * (t * t) + lg;
            }
        }
        for (int off = (1 << a.lw) >> 1; off; off >>= 1) h += __shfl_xor(h, off, 64);
        if (first && k.l == 0) sr_ws[(b * a.V + (size_t)v) * a.tiles + place.tile] = h;
        return;
    }
    if (!act) return;
    if (MODE == LK_GRAD || MODE == LK_BWD) {
        if (first) lk_row_out<T, ROW, MODE>(a, c, k, b, v, count, acc, z, damping, b_old, out, r_out);
        return;
    }
    double sr[N];
    const double f = a.s / (c.az + c.lik1 * (double)count);
#pragma unroll
    for (int e = 0; e < N; ++e) sr[e] = f * ((double)z[e] + a.s * acc[e]);
    if (MODE == LK_MEAN || place_ws >= 0) {
        if (!first) return;
        double* r = sr_ws + (MODE == LK_MEAN ? b * a.n_multi + (size_t)a.idx[v] : b * a.n_joins + (size_t)place_ws) * a.D + k.col;
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (e < k.valid) r[e] = sr[e];
        return;
    }
    const int cnt = count > sub ? ((count - sub - 1) >> ls) + 1 : 0;
    if (LONG && ls == 8 - a.lw && count > kKeep << ls) {           // more than stayed in the registers
        for (int j = 0; j < cnt; j += 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) pj[i] = j + i < cnt ? a.perm[j0 + sub + ((j + i) << ls)] : -1;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (pj[i] >= 0) lk_load<T, ROW>(xb + (size_t)pj[i] * a.D + k.col, k.valid, rows[i]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (pj[i] >= 0) lk_position_out<T, ROW>(a, c.ax + c.an, k, b, (size_t)pj[i], sr, rows[i], damping, b_old, out, r_out);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < kKeep; ++i)
        if (i < cnt) lk_position_out<T, ROW>(a, c.ax + c.an, k, b, (size_t)pj[i], sr, rows[i], damping, b_old, out, r_out);
}

// Third launch of the message to the positions: those of the heavy runs, the chunks that were summed last first - they are the
// likeliest to be cached still (10^6 x 64 f32: 150 us forwards, 138 us backwards).  Bound by the write and what is read twice:
// 318 MB, 53 us, 6.0 TB/s.
template <typename T, int ROW>
__global__ __launch_bounds__(kBlock) void lookup_spread_kernel(LkArgs a, const LkItem* __restrict__ spreads, const LkScal* __restrict__ scal,
                                                               const double* __restrict__ sr_ws, const T* __restrict__ bx, double damping,
                                                               const T* b_old, T* out, T* __restrict__ r_out) {
    constexpr int N = LkVec<T>::N, UR = 4;
    const size_t b = blockIdx.y;
    const unsigned blk = blockIdx.x / a.tiles;
    const LkLane k = lk_lane<T>(a.lw, blockIdx.x - blk * a.tiles, a.D);
    if (k.valid <= 0) return;
    const LkItem it = spreads[gridDim.x / a.tiles - 1 - blk];
    const double asum = scal[b].ax + scal[b].an;
    double sr[N];
#pragma unroll
    for (int e = 0; e < N; ++e)
        sr[e] = e < k.valid ? sr_ws[(b * a.n_joins + (size_t)it.slot) * a.D + k.col + e] : 0.0;
    const int G = kBlock >> a.lw;
    for (int j = it.start + k.group; j < it.end; j += UR * G) {
        int t[UR];
        T v[UR][N];
#pragma unroll
        for (int i = 0; i < UR; ++i) t[i] = j + i * G < it.end ? a.perm[j + i * G] : -1;
#pragma unroll
        for (int i = 0; i < UR; ++i)
            if (t[i] >= 0) lk_load<T, ROW, true>(bx + (b * a.T + (size_t)t[i]) * a.D + k.col, k.valid, v[i]);
#pragma unroll
        for (int i = 0; i < UR; ++i)
            if (t[i] >= 0) lk_position_out<T, ROW>(a, asum, k, b, (size_t)t[i], sr, v[i], damping, b_old, out, r_out);
    }
}

// ---------------------------------------------------------------- the message to x in the order of the positions
// Rows shorter than half a line cost a line each when they are read or written in the order of the tokens.  Here the sums of the
// runs of two and more positions leave scale r in double (LK_MEAN), and x is walked in its own order: a position that is
// alone in its run has its sum at hand, the others fetch theirs.  One column: a lane takes one 16-byte piece of positions.  Bound
// by memory: 64 instances of 100000 positions of 200000 f64 take 44 us, after 37 us for the sums, and the two launches miss the L2
// on 3.1 10^6 lines, 400 MB where z, x and the result are 205 MB: all instances pass the first launch before one passes the second,
// which finds nothing of its own in an L2.  Dropped: runs of two and three summed at each of their positions (102 us in all against
// 99), two pieces per lane (100).
template <typename T, int ROW>
__global__ __launch_bounds__(kBlock) void lookup_positions_kernel(LkArgs a, const int* __restrict__ code, const LkScal* __restrict__ scal,
                                                                  const T* __restrict__ bz, const double* __restrict__ sr_ws,
                                                                  const T* __restrict__ bx, double damping, const T* b_old, T* out,
                                                                  T* __restrict__ r_out) {
    constexpr int N = LkVec<T>::N, UR = 4;
    const LkPlace place = lk_place(a.blocks, a.tiles, a.batch, a.spread);
    const size_t b = place.b;
    const LkLane k = lk_lane<T>(a.lw, place.tile, a.D);
    if (!place.in || k.valid <= 0) return;
    const LkScal c = scal[b];
    const double asum = c.ax + c.an;
    const LkOne one = lk_one(c, a.s);
    const size_t G = kBlock >> a.lw, t0 = (size_t)place.blk * UR * G + k.group;
    int w[UR];
    T v[UR][N], z[UR][N];
    double sr[UR][N];
#pragma unroll
    for (int i = 0; i < UR; ++i) w[i] = t0 + i * G < a.T ? code[t0 + i * G] : -1;
#pragma unroll
    for (int i = 0; i < UR; ++i) {
        if (t0 + i * G < a.T) lk_load<T, ROW>(bx + (b * a.T + t0 + i * G) * a.D + k.col, k.valid, v[i]);
        if (w[i] <= -2) lk_load<T, ROW>(bz + (b * a.V + (size_t)(-2 - w[i])) * a.D + k.col, k.valid, z[i]);
#pragma unroll
        for (int e = 0; e < N; ++e)
            sr[i][e] = w[i] >= 0 && e < k.valid ? sr_ws[(b * a.n_multi + (size_t)w[i]) * a.D + k.col + e] : 0.0;
    }
#pragma unroll
    for (int i = 0; i < UR; ++i) {
        double m[N];
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const double bx_e = (double)v[i][e], bz_e = (double)z[i][e];
            if (w[i] <= -2) sr[i][e] = one.mean * (bz_e + a.s * bx_e);
            m[e] = w[i] <= -2 ? one.kz * bz_e + one.kx * bx_e : sr[i][e] * asum - bx_e;
        }
        if (t0 + i * G < a.T) lk_position_store<T, ROW>(a, k, b, t0 + i * G, m, sr[i], damping, b_old, out, r_out);
    }
}

template <typename T>
__global__ __launch_bounds__(kBlock) void lookup_positions1_kernel(LkArgs a, const int* __restrict__ code, const LkScal* __restrict__ scal,
                                                                   const T* __restrict__ bz, const double* __restrict__ sr_ws,
                                                                   const T* __restrict__ bx, double damping, const T* b_old, T* out,
                                                                   T* __restrict__ r_out) {
    constexpr int N = LkVec<T>::N;
    const LkPlace place = lk_place(a.blocks, 1, a.batch, a.spread);
    const size_t b = place.b, t = ((size_t)place.blk * kBlock + threadIdx.x) * N;
    if (!place.in || t >= a.T) return;
    const LkScal c = scal[b];
    const double asum = c.ax + c.an;
    const LkOne one = lk_one(c, a.s);
    const int valid = a.T - t >= N ? N : (int)(a.T - t);
    int w[N];
    T v[N], o[N], old[N];
    double z[N];
    if (valid == N) {
        typedef int I __attribute__((ext_vector_type(N), aligned(4)));
        const I u = *reinterpret_cast<const I*>(code + t);
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = u[i];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = i < valid ? code[t + i] : -1;
    }
    if (a.spread)                                                  // the L2 is for the table of the instance
        lk_stream_load<T>(bx + b * a.T + t, valid, v);
    else
        lk_load<T, LK_TAIL>(bx + b * a.T + t, valid, v);
    if (damping != 0.0) lk_load<T, LK_TAIL>(b_old + b * a.T + t, valid, old);
#pragma unroll
    for (int i = 0; i < N; ++i)
        z[i] = w[i] >= 0 ? sr_ws[b * a.n_multi + (size_t)w[i]] : w[i] == -1 ? 0.0 : (double)bz[b * a.V + (size_t)(-2 - w[i])];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        double m = w[i] <= -2 ? one.kz * z[i] + one.kx * (double)v[i] : z[i] * asum - (double)v[i];
        if (w[i] <= -2) z[i] = one.mean * (z[i] + a.s * (double)v[i]);
        if (damping != 0.0) m = damping * (double)old[i] + (1.0 - damping) * m;
        o[i] = T(m);
    }
    lk_stream_store<T>(out + b * a.T + t, valid, o);
    if (r_out) {
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] = T(z[i]);
        lk_store<T, LK_TAIL>(r_out + b * a.T + t, valid, o);
    }
}

// ---------------------------------------------------------------- log-partition
// A = 1/2 sum_v (bz + g)^2 / prec + D/2 sum_v log(2 pi / prec)   (linear_channel.py:127-132): the rows' shares, one double per row
// and column tile, added in two steps.  At the end of a run, but for every candidate of every edge under adaptive damping.
// Rows that nobody reads, or one position, have no kind of their own here: 8 x 10007 x 21 f64 of 80021 positions 48 us (the message to
// the table 39), 64 x 200000 f64 of 100000 146 us (98), 50000 x 64 f32 of 10^6 63 us (56).
__global__ __launch_bounds__(kBlock) void lookup_fold_kernel(size_t n, const double* __restrict__ in, double* __restrict__ out) {
    __shared__ double smem[kBlock / kWave];
    const size_t b = blockIdx.y;
    double acc = 0.0;
    for (size_t i = (size_t)blockIdx.x * kBlock + threadIdx.x; i < n; i += (size_t)gridDim.x * kBlock) acc += in[b * n + i];
    acc = block_sum(acc, smem);
    if (threadIdx.x == 0) out[b * gridDim.x + blockIdx.x] = acc;
}

// ---------------------------------------------------------------- handle
extern "C" int tramp_lookup_create(tramp_ctx* ctx, int dtype, size_t n_rows, size_t n_cols, size_t n_pos, const int* tokens_h,
                                   double scale, tramp_lookup** out) {
    if (!ctx || !out) return TRAMP_EINVAL;
    *out = nullptr;
    TRAMP_REQUIRE(ctx, dtype == TRAMP_F32 || dtype == TRAMP_F64);
    TRAMP_REQUIRE(ctx, n_rows > 0 && n_cols > 0 && n_pos > 0 && tokens_h);
    constexpr size_t most = 0x7fff0000u;                           // the strided loops step beyond the last position in 32 bits
    TRAMP_REQUIRE(ctx, n_rows <= most && n_cols <= most && n_pos <= most);
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
        const size_t e = dtype_size(dtype), piece = 16 / e, pieces = (n_cols + piece - 1) / piece;
        int lw = 0;
        while (lw < 6 && ((size_t)1 << lw) < pieces) ++lw;
        // longer rows in tiles of 32 or 16 pieces where tiles of 64 would leave a fifth of the lanes idle and more: 75 pieces in
        // five tiles of 16 (10^5 positions of 300 f32, gradient 47.8 -> 42.8 us, lookup of 200000 114 -> 96 us).  Not below 64
        // pieces: 20 pieces as three tiles of 8 gain in one direction and lose in the other (lookup 17 -> 25 us).
        for (int w = 5; pieces > 64 && w >= 4; --w)
            if (((((pieces - 1) >> w) + 1) << w) * 5 <= ((((pieces - 1) >> lw) + 1) << lw) * 4) lw = w;
        const size_t tiles = (pieces + ((size_t)1 << lw) - 1) >> lw;
        const int per_wave = kKeep << (6 - lw), per_block = kKeep << (8 - lw);
        const bool short_rows = n_cols * e < 64;
        // Runs of one workgroup: what its registers hold, or twice that where it spares the two launches of heavy runs: 2 x 177 x 107
        // f64, V = 20: message to x 14.0 -> 9.2 us, gradient 8.1 -> 5.2; 8 x 20000 x 256 f32, V = 500: 105 -> 98, 45 -> 29.  Four times
        // would leave too few workgroups: 7000 x 256 f32, V = 80, message to x 15.6 -> 17.9, 25000, V = 300: 23 -> 33.
        const int most_read = *std::max_element(counts.begin(), counts.end());
        const bool long_runs = most_read > per_block && most_read <= 2 * per_block;
        const int longest = long_runs ? most_read : per_block;
        std::vector<LkItem> chunks, runs, joins, spreads, waves, light, single;
        std::vector<int> idx, code, empty;
        for (size_t v = 0; v < n_rows; ++v) {
            const int c = counts[v], j0 = off[v];
            if (c == 0) {
                empty.push_back((int)v);
            } else if (c == 1) {
                single.push_back(LkItem{(int)v, j0, j0 + c, perm[(size_t)j0]});
            } else if (c <= kKeep) {
                light.push_back(LkItem{(int)v, j0, j0 + c, perm[(size_t)j0]});
            } else if (c <= per_wave) {
                waves.push_back(LkItem{(int)v, j0, j0 + c, -1});
            } else if (c <= longest) {
                runs.push_back(LkItem{(int)v, j0, j0 + c, -1});
            } else {
                // at most 256 partial sums per run: one workgroup adds them
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
        // equal lengths side by side: a wave goes no deeper than its longest run
        std::stable_sort(light.begin(), light.end(), [](const LkItem& x, const LkItem& y) { return x.end - x.start > y.end - y.start; });
        const size_t n_light2 = light.size();
        light.insert(light.end(), single.begin(), single.end());
        size_t n_multi = 0;
        if (short_rows) {
            idx.assign(n_rows, -1);
            for (size_t v = 0; v < n_rows; ++v)
                if (counts[v] > 1) idx[v] = (int)n_multi++;
            code.resize(n_pos);
            for (size_t t = 0; t < n_pos; ++t) {
                const int v = tokens_h[t];
                code[t] = v < 0 ? -1 : counts[(size_t)v] == 1 ? -2 - v : idx[(size_t)v];
            }
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
        // one allocation: the arrays one behind the other
        std::vector<char> host;
        host.reserve(n_pos * (short_rows ? 12 : 8) + n_rows * (short_rows ? 8 : 4) + empty.size() * 4 + 2 * K * 8 + 16 * 256 +
                     sizeof(LkItem) * (chunks.size() + joins.size() + spreads.size() + runs.size() + waves.size() + light.size()));
        auto put = [&host](const void* p, size_t bytes) {
            const size_t at = host.size();
            host.resize(at + ((bytes + 255) & ~(size_t)255));
            if (bytes) memcpy(host.data() + at, p, bytes);
            return at;
        };
        const size_t o_tok = put(tokens_h, n_pos * 4), o_perm = put(perm.data(), n_pos * 4), o_off = put(off.data(), (n_rows + 1) * 4);
        const size_t o_cnt = put(cval.data(), 2 * K * 8), o_chunks = put(chunks.data(), chunks.size() * sizeof(LkItem));
        const size_t o_joins = put(joins.data(), joins.size() * sizeof(LkItem)), o_spreads = put(spreads.data(), spreads.size() * sizeof(LkItem));
        const size_t o_runs = put(runs.data(), runs.size() * sizeof(LkItem)), o_waves = put(waves.data(), waves.size() * sizeof(LkItem));
        const size_t o_light = put(light.data(), light.size() * sizeof(LkItem)), o_idx = put(idx.data(), idx.size() * 4), o_code = put(code.data(), code.size() * 4);
        const size_t o_empty = put(empty.data(), empty.size() * 4);
        tramp_lookup* lk = new tramp_lookup();
        *lk = tramp_lookup{};
        (void)hipSetDevice(ctx->device);
        if (hipMalloc(&lk->mem, host.size()) != hipSuccess) {
            (void)hipGetLastError();
            delete lk;
            return tramp_fail(ctx, TRAMP_ENOMEM, "tramp_lookup_create", "hipMalloc failed");
        }
        char* m = static_cast<char*>(lk->mem);
        hipError_t err = hipMemcpyAsync(m, host.data(), host.size(), hipMemcpyHostToDevice, ctx->stream);
        if (err == hipSuccess) err = hipStreamSynchronize(ctx->stream);  // the host array ends here
        if (err != hipSuccess) {
            (void)hipFree(lk->mem);
            delete lk;
            return tramp_fail(ctx, TRAMP_EHIP, "tramp_lookup_create", hipGetErrorString(err));
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
        lk->chunks = reinterpret_cast<const LkItem*>(m + o_chunks);
        lk->joins = reinterpret_cast<const LkItem*>(m + o_joins);
        lk->spreads = reinterpret_cast<const LkItem*>(m + o_spreads);
        lk->runs = reinterpret_cast<const LkItem*>(m + o_runs);
        lk->waves = reinterpret_cast<const LkItem*>(m + o_waves);
        lk->light = reinterpret_cast<const LkItem*>(m + o_light);
        lk->idx = reinterpret_cast<const int*>(m + o_idx);
        lk->code = reinterpret_cast<const int*>(m + o_code);
        lk->empty = reinterpret_cast<const int*>(m + o_empty);
        lk->n_empty = (unsigned)empty.size();
        lk->K = (int)K;
        lk->n_chunks = (unsigned)chunks.size();
        lk->n_joins = (unsigned)joins.size();
        lk->n_spreads = (unsigned)spreads.size();
        lk->n_runs = (unsigned)runs.size();
        lk->n_waves = (unsigned)waves.size();
        lk->n_light = (unsigned)light.size();
        lk->n_light2 = (unsigned)n_light2;
        lk->n_multi = (unsigned)n_multi;
        lk->lw = lw;
        lk->tiles = (unsigned)tiles;
        lk->row = n_cols % piece ? LK_TAIL : n_cols * e % 128 ? LK_WHOLE : LK_LINES;
        lk->short_rows = short_rows;
        lk->long_runs = long_runs;
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

// CALL(ROW) for the handle's kind of rows
#define LK_BY_ROW(lk, CALL)               \
    switch ((lk)->row) {                  \
        case LK_TAIL: CALL(LK_TAIL);      \
        case LK_WHOLE: CALL(LK_WHOLE);    \
        default: CALL(LK_LINES);          \
    }

static dim3 lk_grid(size_t batch, size_t blocks, int spread) {
    return spread ? dim3((unsigned)((batch + 7) / 8 * 8 * blocks)) : dim3((unsigned)blocks, (unsigned)batch);
}

template <typename T>
static int lookup_apply(tramp_ctx* ctx, const tramp_lookup* lk, size_t batch, const T* z, T* x) {
    constexpr size_t N = LkVec<T>::N;
    if (lk->D == 1) {
        const size_t nb = (lk->T + kBlock * N - 1) / (kBlock * N);
        const int spread = lk_spread(batch, nb, lk->V * sizeof(T), 8u << 20);
        hipLaunchKernelGGL((lookup_apply1_kernel<T>), lk_grid(batch, nb, spread), dim3(kBlock), 0, ctx->stream, lk->V, lk->T, lk->s,
                           (unsigned)nb, (unsigned)batch, spread, lk->tok, z, x);
    } else {
        const size_t per = (size_t)4 * (kBlock >> lk->lw), nb = (lk->T + per - 1) / per;
        TRAMP_REQUIRE(ctx, nb * lk->tiles <= kLkMaxGrid);
        const int spread = lk_spread(batch, nb * lk->tiles, lk->V * lk->D * sizeof(T), 8u << 20);
        const dim3 grid = lk_grid(batch, nb * lk->tiles, spread);
#define LK_CALL(ROW)                                                                                                                   \
    hipLaunchKernelGGL((lookup_apply_kernel<T, ROW>), grid, dim3(kBlock), 0, ctx->stream, lk->V, lk->D, lk->T, lk->s, lk->lw, (unsigned)nb, \
                       lk->tiles, (unsigned)batch, spread, lk->tok, z, x);                                                             \
    break
        LK_BY_ROW(lk, LK_CALL)
#undef LK_CALL
    }
    TRAMP_LAUNCH_CHECK(ctx);
    return TRAMP_OK;
}

extern "C" int tramp_lookup_apply(tramp_ctx* ctx, tramp_lookup* lk, size_t batch, const void* z_d, void* x_d) {
    LK_REQUIRE_CALL(ctx, lk, batch);
    TRAMP_REQUIRE(ctx, z_d && x_d);
    const size_t row = batch * lk->D * dtype_size(lk->dtype);
    TRAMP_REQUIRE(ctx, !lk_overlap(z_d, lk->V * row, x_d, lk->T * row));
    if (!batch) return TRAMP_OK;
    return lk->dtype == TRAMP_F64 ? lookup_apply<double>(ctx, lk, batch, (const double*)z_d, (double*)x_d)
                                  : lookup_apply<float>(ctx, lk, batch, (const float*)z_d, (float*)x_d);
}

static LkScalArgs lk_scal_args(const tramp_lookup* lk, int dir, const double* az, const double* ax, double damping, const double* a_old) {
    LkScalArgs q{};
    q.cnt = lk->cnt;
    q.az = az;
    q.ax = ax;
    q.a_old = a_old;
    q.V = (double)lk->V;
    q.T = (double)lk->T;
    q.padded = (double)(lk->T - lk->seen);
    q.s = lk->s;
    q.damping = damping;
    q.K = lk->K;
    q.dir = dir;
    return q;
}

// ctx->ws of a call: [scalars | partial sums | scale r of the heavy runs, or of all runs of two and more positions, or the
// shares of the log-partition]
struct LkWs {
    LkScal* scal;
    double* partials;
    double* sr;
};
// Short rows in the order of the positions: one column from 4 MB of positions on (10^6 f64 44 -> 33 us, 16 x 60000 29 -> 22 us;
// 64 x 2000 would be 10.0 against 8.3 us, the price of the second launch), more columns where heavy runs take launches of
// their own anyway (10^6 x 7 f64 83 -> 63 us; 8 x 60000 x 4 f64 without any 19.5 against 23.7 us).
static bool lk_by_position(const tramp_lookup* lk, size_t batch) {
    return lk->short_rows && batch * lk->T * lk->D * dtype_size(lk->dtype) >= ((size_t)4 << 20) && (lk->D == 1 || lk->n_chunks);
}
static int lk_workspace(tramp_ctx* ctx, const tramp_lookup* lk, size_t batch, size_t n_extra, LkWs* w) {
    const size_t n_scal = (batch * sizeof(LkScal) + 255) & ~(size_t)255, n_part = batch * lk->n_chunks * lk->D * sizeof(double);
    const size_t n_sr = n_extra * sizeof(double);
    int rc = tramp_ws_reserve(ctx, n_scal + n_part + n_sr);
    if (rc) return rc;
    char* m = reinterpret_cast<char*>(ctx->ws);
    *w = LkWs{reinterpret_cast<LkScal*>(m), reinterpret_cast<double*>(m + n_scal), reinterpret_cast<double*>(m + n_scal + n_part)};
    return TRAMP_OK;
}

template <typename T, int ROW, int MODE>
static int launch_rows(tramp_ctx* ctx, const tramp_lookup* lk, size_t batch, const LkWs& w, const LkScalArgs* q, const T* bz, const T* x,
                       double damping, const T* b_old, T* out, T* r_out) {
    LkArgs a{};
    a.off = lk->off;
    a.perm = lk->perm;
    a.chunks = lk->chunks;
    a.joins = lk->joins;
    a.runs = lk->runs;
    a.waves = lk->waves;
    const bool listed = MODE == LK_FWD || MODE == LK_MEAN || ((MODE == LK_GRAD || MODE == LK_BWD) && !lk->short_rows);
    a.light = listed ? lk->light : nullptr;
    a.empty = lk->empty;
    a.idx = lk->idx;
    a.V = lk->V;
    a.D = lk->D;
    a.T = lk->T;
    a.n_chunks = lk->n_chunks;
    a.n_joins = lk->n_joins;
    a.n_runs = lk->n_runs;
    a.n_waves = lk->n_waves;
    a.wave_blocks = (lk->n_waves + kBlock / kWave - 1) / (kBlock / kWave);
    a.n_light = listed ? lk->n_light2 : (unsigned)lk->V;
    a.n_single = listed && MODE != LK_MEAN ? lk->n_light - lk->n_light2 : 0;
    a.n_empty = listed && (MODE == LK_GRAD || MODE == LK_BWD) ? lk->n_empty : 0;
    a.n_multi = lk->n_multi;
    a.tiles = lk->tiles;
    a.batch = (unsigned)batch;
    a.lw = lk->lw;
    a.s = lk->s;
    const size_t G = kBlock >> lk->lw;
    // short rows: 64 x 60000 f32 of one column 27.2 -> 21.5 us, 1000001 f64 21.9 -> 20.1, 8 x 200000 x 7 f64 43.4 -> 41.2; longer ones
    // would lose: 65536 x 1024 f32 78.7 against 83.1 us, 20000 x 300 f64 15.2 against 16.1
    a.n_lead = MODE == LK_GRAD && lk->short_rows ? lk->n_chunks : 0;
    if (a.n_lead) a.n_joins = 0;
    a.light_blocks = (unsigned)(((size_t)a.n_light + G - 1) / G);
    a.n_pad = MODE == LK_FWD ? (unsigned)(lk->T - lk->seen) : 0;
    a.pad0 = lk->seen;
    a.single_blocks = (unsigned)(((size_t)a.n_single + a.n_pad + kOne * G - 1) / (kOne * G));
    const size_t blocks = (size_t)a.n_lead + a.n_joins + a.n_runs + a.wave_blocks + a.light_blocks + a.single_blocks + (a.n_empty + kEmpty * G - 1) / (kEmpty * G);
    TRAMP_REQUIRE(ctx, blocks * lk->tiles <= kLkMaxGrid && (size_t)lk->n_chunks * lk->tiles < kLkMaxGrid);   // (as many spreads as chunks)
    a.blocks = (unsigned)blocks;
    a.spread = lk_spread(batch, blocks * lk->tiles, lk->T * lk->D * sizeof(T), 2u << 20);
    // few workgroups and few counts: each makes the scalars for itself, one launch less (V = 1000, 2000 positions 10.2 -> 7.6 us;
    // with up to 4096 workgroups 8 x 60000 x 8 f64 would be 31.5 against 27.1 us)
    const bool self = q && !lk->n_chunks && blocks && blocks * lk->tiles * batch <= 1024 && lk->K <= 4 * kBlock &&
                      !lk_scalars_in_place(q->az, q->ax, q->a_new_out, q->v_out, q->n_eff_out);
    if ((lk->n_chunks && !a.n_lead) || (q && !self))
        hipLaunchKernelGGL((lookup_chunks_kernel<T, ROW, MODE != LK_FWD && MODE != LK_MEAN>), dim3(lk->n_chunks * lk->tiles + (q ? 1 : 0), (unsigned)batch),
                           dim3(kBlock), 0, ctx->stream, a, q ? *q : LkScalArgs{}, x, w.partials);
    const dim3 grid = lk_grid(batch, blocks * lk->tiles, a.spread);
    constexpr bool fwd = MODE == LK_FWD;
    if (MODE != LK_GRAD && self)
        hipLaunchKernelGGL((lookup_rows_kernel<T, ROW, MODE, MODE != LK_GRAD, fwd>), grid, dim3(kBlock), 0, ctx->stream, a, *q, w.scal, bz, x, damping,
                           b_old, out, r_out, w.partials, w.sr);
    else if (blocks && fwd && lk->long_runs)
        hipLaunchKernelGGL((lookup_rows_kernel<T, ROW, MODE, false, fwd>), grid, dim3(kBlock), 0, ctx->stream, a, LkScalArgs{}, w.scal, bz, x, damping,
                           b_old, out, r_out, w.partials, w.sr);
    else if (blocks)
        hipLaunchKernelGGL((lookup_rows_kernel<T, ROW, MODE, false, false>), grid, dim3(kBlock), 0, ctx->stream, a, LkScalArgs{}, w.scal, bz, x, damping,
                           b_old, out, r_out, w.partials, w.sr);
    if (a.n_lead) {
        LkArgs j = a;
        j.n_joins = j.blocks = lk->n_joins;
        j.n_lead = j.n_runs = j.n_waves = j.wave_blocks = j.n_light = j.light_blocks = j.n_single = j.n_pad = j.single_blocks = j.n_empty = 0;
        j.spread = 0;
        hipLaunchKernelGGL((lookup_rows_kernel<T, ROW, MODE, false, false>), lk_grid(batch, (size_t)j.blocks * lk->tiles, 0), dim3(kBlock), 0, ctx->stream,
                           j, LkScalArgs{}, w.scal, bz, x, damping, b_old, out, r_out, w.partials, w.sr);
    }
    if (MODE == LK_FWD && lk->n_spreads)
        hipLaunchKernelGGL((lookup_spread_kernel<T, ROW>), dim3(lk->n_spreads * lk->tiles, (unsigned)batch), dim3(kBlock), 0, ctx->stream, a,
                           lk->spreads, w.scal, w.sr, x, damping, b_old, out, r_out);
    if (MODE == LK_MEAN) {
        const size_t per = lk->D == 1 ? (size_t)kBlock * LkVec<T>::N : 4 * G, nb = (lk->T + per - 1) / per;
        a.blocks = (unsigned)nb;
        a.spread = lk_spread(batch, nb * lk->tiles, lk->V * lk->D * sizeof(T), 8u << 20);
        if (lk->D == 1)
            hipLaunchKernelGGL((lookup_positions1_kernel<T>), lk_grid(batch, nb, a.spread), dim3(kBlock), 0, ctx->stream, a, lk->code, w.scal,
                               bz, w.sr, x, damping, b_old, out, r_out);
        else
            hipLaunchKernelGGL((lookup_positions_kernel<T, ROW>), lk_grid(batch, nb * lk->tiles, a.spread), dim3(kBlock), 0, ctx->stream, a,
                               lk->code, w.scal, bz, w.sr, x, damping, b_old, out, r_out);
    }
    TRAMP_LAUNCH_CHECK(ctx);
    return TRAMP_OK;
}

template <typename T, int MODE>
static int run_rows(tramp_ctx* ctx, const tramp_lookup* lk, size_t batch, const LkWs& w, const LkScalArgs* q, const T* bz, const T* x,
                    double damping, const T* b_old, T* out, T* r_out) {
#define LK_CALL(ROW) return launch_rows<T, ROW, MODE>(ctx, lk, batch, w, q, bz, x, damping, b_old, out, r_out)
    LK_BY_ROW(lk, LK_CALL)
#undef LK_CALL
}

extern "C" int tramp_lookup_gradient(tramp_ctx* ctx, tramp_lookup* lk, size_t batch, const void* x_d, void* g_d) {
    LK_REQUIRE_CALL(ctx, lk, batch);
    TRAMP_REQUIRE(ctx, x_d && g_d);
    const size_t row = batch * lk->D * dtype_size(lk->dtype);
    TRAMP_REQUIRE(ctx, !lk_overlap(g_d, lk->V * row, x_d, lk->T * row));
    if (!batch) return TRAMP_OK;
    LkWs w;
    int rc = lk_workspace(ctx, lk, batch, 0, &w);
    if (rc) return rc;
    if (lk->dtype == TRAMP_F64)
        return run_rows<double, LK_GRAD>(ctx, lk, batch, w, nullptr, nullptr, (const double*)x_d, 0.0, nullptr, (double*)g_d, nullptr);
    return run_rows<float, LK_GRAD>(ctx, lk, batch, w, nullptr, nullptr, (const float*)x_d, 0.0, nullptr, (float*)g_d, nullptr);
}

extern "C" int tramp_lookup_variance(tramp_ctx* ctx, tramp_lookup* lk, int dir, size_t batch, const double* az_d,
                                     const double* ax_d, double* v_d, double* a_new_d, double* n_eff_d) {
    LK_REQUIRE_CALL(ctx, lk, batch);
    TRAMP_REQUIRE(ctx, (dir == TRAMP_FWD || dir == TRAMP_BWD) && az_d && ax_d);
    const char* conflict = lk_conflict({az_d, ax_d, nullptr, nullptr, nullptr, nullptr, a_new_d, v_d, n_eff_d, nullptr, nullptr, batch * sizeof(double),
                                        0, 0, 0});
    if (conflict) return tramp_fail(ctx, TRAMP_EINVAL, "tramp_lookup_variance", conflict);
    if (!batch) return TRAMP_OK;
    LkScalArgs q = lk_scal_args(lk, dir, az_d, ax_d, 0.0, nullptr);
    q.v_out = v_d;
    q.a_new_out = a_new_d;
    q.n_eff_out = n_eff_d;
    hipLaunchKernelGGL(lookup_scalars_kernel, dim3((unsigned)batch), dim3(kBlock), 0, ctx->stream, q);
    TRAMP_LAUNCH_CHECK(ctx);
    return TRAMP_OK;
}

template <typename T>
static int lookup_message(tramp_ctx* ctx, tramp_lookup* lk, int dir, size_t batch, const double* az_d, const T* bz,
                          const double* ax_d, const T* bx, double damping, const double* a_old_d, const T* b_old, double* a_new_d,
                          T* b_new, T* r_d, double* v_d) {
    LkWs w;
    const bool by_position = dir == TRAMP_FWD && lk_by_position(lk, batch);
    int rc = lk_workspace(ctx, lk, batch, dir == TRAMP_BWD ? 0 : batch * (by_position ? lk->n_multi : lk->n_joins) * lk->D, &w);
    if (rc) return rc;
    LkScalArgs q = lk_scal_args(lk, dir, az_d, ax_d, damping, a_old_d);
    q.scal = w.scal;
    q.v_out = v_d;
    q.a_new_out = a_new_d;
    if (dir == TRAMP_BWD) return run_rows<T, LK_BWD>(ctx, lk, batch, w, &q, bz, bx, damping, b_old, b_new, r_d);
    if (by_position) return run_rows<T, LK_MEAN>(ctx, lk, batch, w, &q, bz, bx, damping, b_old, b_new, r_d);
    return run_rows<T, LK_FWD>(ctx, lk, batch, w, &q, bz, bx, damping, b_old, b_new, r_d);
}

extern "C" int tramp_lookup_message(tramp_ctx* ctx, tramp_lookup* lk, int dir, size_t batch, const double* az_d, const void* bz_d,
                                    const double* ax_d, const void* bx_d, double damping, const double* a_old_d,
                                    const void* b_old_d, double* a_new_d, void* b_new_d, void* r_d, double* v_d) {
    LK_REQUIRE_CALL(ctx, lk, batch);
    TRAMP_REQUIRE(ctx, (dir == TRAMP_FWD || dir == TRAMP_BWD) && az_d && bz_d && ax_d && bx_d && a_new_d && b_new_d);
    const size_t row = batch * lk->D * dtype_size(lk->dtype), nz = lk->V * row, nx = lk->T * row, no = dir == TRAMP_FWD ? nx : nz;
    TRAMP_REQUIRE(ctx, damping == 0.0 || (a_old_d && b_old_d));
    const bool damped = damping != 0.0;
    const char* conflict = lk_conflict({az_d, ax_d, damped ? a_old_d : nullptr, bz_d, bx_d, damped ? b_old_d : nullptr, a_new_d, v_d, nullptr, b_new_d, r_d,
                                        batch * sizeof(double), nz, nx, no});
    if (conflict) return tramp_fail(ctx, TRAMP_EINVAL, "tramp_lookup_message", conflict);
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
    const size_t n = lk->V * lk->tiles;
    const int nblk = blocks_for(n, 1);
    LkWs w;
    int rc = lk_workspace(ctx, lk, batch, batch * (n + (size_t)nblk), &w);
    if (rc) return rc;
    LkScalArgs q = lk_scal_args(lk, TRAMP_FWD, az_d, ax_d, 0.0, nullptr);
    q.scal = w.scal;
    rc = lk->dtype == TRAMP_F64
             ? run_rows<double, LK_LOGZ>(ctx, lk, batch, w, &q, (const double*)bz_d, (const double*)bx_d, 0.0, nullptr, nullptr, nullptr)
             : run_rows<float, LK_LOGZ>(ctx, lk, batch, w, &q, (const float*)bz_d, (const float*)bx_d, 0.0, nullptr, nullptr, nullptr);
    if (rc) return rc;
    hipLaunchKernelGGL(lookup_fold_kernel, dim3(nblk, (unsigned)batch), dim3(kBlock), 0, ctx->stream, n, w.sr, w.sr + batch * n);
    hipLaunchKernelGGL(lookup_fold_kernel, dim3(1, (unsigned)batch), dim3(kBlock), 0, ctx->stream, (size_t)nblk, w.sr + batch * n, out_d);
    TRAMP_LAUNCH_CHECK(ctx);
    return TRAMP_OK;
}
