// Layer norm over the last dim, forward and backward (no counterpart in the reference).
//
//   mu = mean(x), v = mean((x - mu)^2), r = 1 / sqrt(v + eps), xh = (x - mu) * r, y = xh * gain + shift
//   g = e * gain:  dx = r * (g - mean(g) - xh * mean(g * xh)),  dgain = sum over rows of e * xh,  dshift = sum over rows of e
//
// Every sum is taken in the tensor's type over a fixed partition of the row (or column), so the result does not depend on scheduling; v
// comes from the differences to a mean that is known before (no difference of large sums). Where a row lies far from zero, what these
// differences come to corrects the mean (norm_far, norm_settle).
#include <cooperative_groups.h>

#include <atomic>

#include "nk_internal.h"
#include "nk_ptx.cuh"

namespace cg = cooperative_groups;

namespace {

template <class T, int W> struct NormVec { using type = T; };
template <> struct NormVec<float, 4> { using type = float4; };
template <> struct NormVec<double, 2> { using type = double2; };
template <class T> constexpr int norm_w() { return 16 / int(sizeof(T)); }

// The rows of a call: what the outer dims come to after merging, with a stride per operand and dim.
struct NormPlan {
    int nd;                                  // outer dims, at least 1
    int64_t rows, n;
    int64_t ext[NK_MAX_RANK];
    int64_t s[3][NK_MAX_RANK], inner[3];     // 0: drain, 1: source, 2: error; strides of the outer dims and of the normalised one
    int64_t gain_s, shift_s;                 // strides of gain and shift
    int gain_v, shift_v;                     // 16-byte loads of them are possible
    const char *lo[2], *hi[2];               // the buffers of source and error
};

template <int OP>
__device__ __forceinline__ int64_t norm_row(const NormPlan& p, int64_t r) {
    int64_t off = 0;
    for (int k = p.nd - 1; k > 0; k--) {
        const int64_t q = r / p.ext[k];
        off += (r - q * p.ext[k]) * p.s[OP][k];
        r = q;
    }
    return off + r * p.s[OP][0];
}
// W elements from column c on; past n: zeros (W divides n where W > 1)
template <class T, int W>
__device__ __forceinline__ void norm_load(const T* row, int64_t c, int64_t inner, int64_t n, T (&v)[W]) {
    if (W > 1) {
        if (c < n) *reinterpret_cast<typename NormVec<T, W>::type*>(v) = *reinterpret_cast<const typename NormVec<T, W>::type*>(row + c);
        else {
#pragma unroll
            for (int k = 0; k < W; k++) v[k] = T(0);
        }
    } else v[0] = c < n ? row[c * inner] : T(0);
}
template <class T, int W>
__device__ __forceinline__ void norm_store(T* row, int64_t c, int64_t inner, int64_t n, const T (&v)[W]) {
    if (c >= n) return;
    if (W > 1) *reinterpret_cast<typename NormVec<T, W>::type*>(row + c) = *reinterpret_cast<const typename NormVec<T, W>::type*>(v);
    else row[c * inner] = v[0];
}

// W elements of gain or shift (all of them exist)
template <class T, int W>
__device__ __forceinline__ void norm_vector_load(const T* a, int64_t c, int64_t stride, int vec, T (&v)[W]) {
    if (W > 1 && vec) *reinterpret_cast<typename NormVec<T, W>::type*>(v) = __ldg(reinterpret_cast<const typename NormVec<T, W>::type*>(a + c));
    else {
#pragma unroll
        for (int j = 0; j < W; j++) v[j] = __ldg(a + (c + j) * stride);
    }
}

constexpr int NORM_THREADS = 256;
// sum over the CTA, the same value in every thread
template <class T>
__device__ __forceinline__ T norm_cta_sum(T v, T* smem) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    const int warp = threadIdx.x >> 5;
    __syncthreads();   // smem may still be read from the sum before
    if ((threadIdx.x & 31) == 0) smem[warp] = v;
    __syncthreads();
    v = smem[0];
#pragma unroll
    for (int w = 1; w < NORM_THREADS / 32; w++) v += smem[w];
    return v;
}

// sum over a CTA of THREADS threads, the same value in every thread; smem is not in use when the call begins and may be used again after the next
// barrier that follows the call
template <class T, int THREADS>
__device__ __forceinline__ T norm_sum(T v, T* smem) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = v;
    __syncthreads();
    v = smem[0];
#pragma unroll
    for (int w = 1; w < THREADS / 32; w++) v += smem[w];
    return v;
}
template <class T, int THREADS>
__device__ __forceinline__ void norm_sum2(T& a, T& b, T (*smem)[THREADS / 32]) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) { a += __shfl_xor_sync(0xffffffffu, a, o); b += __shfl_xor_sync(0xffffffffu, b, o); }
    if ((threadIdx.x & 31) == 0) { smem[0][threadIdx.x >> 5] = a; smem[1][threadIdx.x >> 5] = b; }
    __syncthreads();
    a = smem[0][0];
    b = smem[1][0];
#pragma unroll
    for (int w = 1; w < THREADS / 32; w++) { a += smem[0][w]; b += smem[1][w]; }
}
// A mean is off by some units in its last place (a sum was rounded on the way), and a row's result by that over its deviation: nothing where they are
// alike, everything where the row is far from zero and narrow (a row of 1000.0 came out as -0.019 instead of 0). There the differences d to the
// mean tell by how much: their sum is 0 for the true one. A row of equal values gets that value as its mean, whatever its length, since its
// differences are exact and all the same. Every row would pay for one more sum (8192 x 8192: 92 us -> 102, 16384 x 4096 F64: 192 -> 212), so only rows
// further from zero than four deviations do. The same answer in all threads that share mean and m2.
template <class T>
__device__ __forceinline__ bool norm_far(T mean, T v) {   // (asked after 1 / sqrt(v + eps) has been begun, which takes longer)
    return mean * mean > T(16) * v;                       // (false for a NaN)
}
// the same value, of which the compiler does not know that: the differences taken above need not stay in registers for the rows that need them again (24 more
// registers otherwise, which cost 200000 x 200 a third of its speed)
__device__ __forceinline__ float norm_again(float v) { asm volatile("" : "+f"(v)); return v; }
__device__ __forceinline__ double norm_again(double v) { asm volatile("" : "+d"(v)); return v; }
// d: the sum of the differences to the mean
template <class T>
__device__ __forceinline__ void norm_settle(T& mean, T& rstd, T m2, T d, T n, T eps) {
    const T by = d / n;
    mean += by;
    m2 -= d * by;
    rstd = T(1) / sqrt((m2 > T(0) ? m2 / n : T(0)) + eps);
}
// (x - mean) * rstd * gain + shift for the vectors at c0 + (k * lanes + lane) * W, stored
template <class T, int W, int NV>
__device__ __forceinline__ void norm_results(T* y, const T* gain, const T* shift, const NormPlan& p, int64_t c0, int lane, int lanes, T mean, T rstd, T (&v)[NV][W]) {
#pragma unroll
    for (int k = 0; k < NV; k++) {
        const int64_t c = c0 + (k * lanes + lane) * W;
        if (c >= p.n) continue;
        T g[W], s[W];
        if (gain) norm_vector_load<T, W>(gain, c, p.gain_s, p.gain_v, g);
        if (shift) norm_vector_load<T, W>(shift, c, p.shift_s, p.shift_v, s);
#pragma unroll
        for (int j = 0; j < W; j++) {
            v[k][j] = (v[k][j] - mean) * rstd;
            if (gain) v[k][j] *= g[j];
            if (shift) v[k][j] += s[j];
        }
        norm_store<T, W>(y, c, p.inner[0], p.n, v[k]);
    }
}

// ---- rows that a group of lanes, a CTA or a cluster holds in registers ---------------------------------------------------------------
// One pass over the data: x stays in registers between the mean, the variance and the result. Short rows, and calls with too few rows to keep teams
// with rings busy (below), which the latency of a row bounds: 1 x 4096 5.4 us, 1000 x 777 forward 8.2 us; 400000 x 64 69 us (3.0 TB/s: a row per group in flight, its two sums one after the other).

// CTAs per SM that the registers have to leave room for: fewer cost more than a few spilled words (200000 x 200 by two of them 140 us, by three 109)
template <class T, int W, int E>
constexpr int norm_lanes_ctas() {
    const bool wide = sizeof(T) == 8 && W > 1;
    return E == 4 ? (wide ? 3 : 4) : E == 8 ? (wide ? 2 : 3) : (W == 1 && sizeof(T) == 4 ? 3 : 2);
}
// A row per group of G lanes, E elements per lane.
template <class T, int W, int G, int E>
__global__ void __launch_bounds__(256, norm_lanes_ctas<T, W, E>()) nk_norm_lanes_kernel(T* out, const T* src, const T* __restrict__ gain, const T* __restrict__ shift, T* __restrict__ stats,
                                                            const NormPlan p, T eps) {
    constexpr int NV = E / W;
    const int lane = threadIdx.x % G;
    const int64_t rows_per = 256 / G;
    const T n = T(p.n);
    for (int64_t first = int64_t(blockIdx.x) * rows_per; first < p.rows; first += int64_t(gridDim.x) * rows_per) {
        const int64_t row = first + threadIdx.x / G;
        const bool mine = row < p.rows;
        const int64_t r = mine ? row : p.rows - 1;
        const T* x = src + norm_row<1>(p, r);
        T v[NV][W], sum = T(0);
#pragma unroll
        for (int k = 0; k < NV; k++) norm_load<T, W>(x, (k * G + lane) * W, p.inner[1], p.n, v[k]);
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
            for (int j = 0; j < W; j++) sum += v[k][j];
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        T mean = sum / n, m2 = T(0);
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
            for (int j = 0; j < W; j++)
                if ((k * G + lane) * W + j < p.n) m2 += (v[k][j] - mean) * (v[k][j] - mean);
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) m2 += __shfl_xor_sync(0xffffffffu, m2, o);
        const T v2 = m2 / n;
        T rstd = T(1) / sqrt(v2 + eps);
        if (__any_sync(0xffffffffu, norm_far(mean, v2))) {
            const T from = norm_again(mean);
            T off = T(0);
#pragma unroll
            for (int k = 0; k < NV; k++)
#pragma unroll
                for (int j = 0; j < W; j++)
                    if ((k * G + lane) * W + j < p.n) off += v[k][j] - from;
#pragma unroll
            for (int o = G / 2; o > 0; o >>= 1) off += __shfl_xor_sync(0xffffffffu, off, o);
            if (norm_far(mean, v2)) norm_settle(mean, rstd, m2, off, n, eps);   // (a row's result does not depend on its neighbours)
        }
        if (!mine) continue;
        if (stats && lane == 0) { stats[row] = mean; stats[p.rows + row] = rstd; }
        norm_results<T, W, NV>(out + norm_row<0>(p, row), gain, shift, p, int64_t(0), lane, G, mean, rstd, v);
    }
}
// A row per CTA, or per cluster of CTAs (each a slice of the row; their sums meet through distributed shared memory).
template <class T, int W, int THREADS, int E>
__global__ void __launch_bounds__(THREADS) nk_norm_cta_kernel(T* out, const T* src, const T* __restrict__ gain, const T* __restrict__ shift, T* __restrict__ stats,
                                                              const NormPlan p, T eps) {
    constexpr int NV = E / W;
    __shared__ T warps[3][THREADS / 32], parts[2][3];
    cg::cluster_group cluster = cg::this_cluster();
    const int size = int(cluster.num_blocks()), rank = int(cluster.block_rank());
    const int64_t c0 = int64_t(rank) * THREADS * E, step = gridDim.x / unsigned(size);
    const T n = T(p.n);
    int turn = 0;
    auto total = [&](T v, int which) {
        v = norm_sum<T, THREADS>(v, warps[which]);
        if (size == 1) return v;
        if (threadIdx.x == 0) parts[turn & 1][which] = v;   // two rows' worth: a slow neighbour may still read the last row's
        cluster.sync();
        v = T(0);
        for (int r = 0; r < size; r++) v += *cluster.map_shared_rank(&parts[turn & 1][which], r);
        return v;
    };
    for (int64_t row = blockIdx.x / unsigned(size); row < p.rows; row += step, turn++) {
        const T* x = src + norm_row<1>(p, row);
        T v[NV][W], sum = T(0);
#pragma unroll
        for (int k = 0; k < NV; k++) norm_load<T, W>(x, c0 + (k * THREADS + int(threadIdx.x)) * W, p.inner[1], p.n, v[k]);
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
            for (int j = 0; j < W; j++) sum += v[k][j];
        T mean = total(sum, 0) / n, m2 = T(0);
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
            for (int j = 0; j < W; j++)
                if (c0 + (k * THREADS + int(threadIdx.x)) * W + j < p.n) m2 += (v[k][j] - mean) * (v[k][j] - mean);
        m2 = total(m2, 1);
        const T v2 = m2 / n;
        T rstd = T(1) / sqrt(v2 + eps);
        if (norm_far(mean, v2)) {
            const T from = norm_again(mean);
            T off = T(0);
#pragma unroll
            for (int k = 0; k < NV; k++)
#pragma unroll
                for (int j = 0; j < W; j++)
                    if (c0 + (k * THREADS + int(threadIdx.x)) * W + j < p.n) off += v[k][j] - from;
            norm_settle(mean, rstd, m2, total(off, 2), n, eps);
        }
        if (stats && rank == 0 && threadIdx.x == 0) { stats[row] = mean; stats[p.rows + row] = rstd; }
        norm_results<T, W, NV>(out + norm_row<0>(p, row), gain, shift, p, c0, threadIdx.x, THREADS, mean, rstd, v);
    }
    if (size > 1) cluster.sync();   // nobody leaves while its sums may still be read
}

// Backward, a row per step of a CTA (or cluster): a thread owns E columns and walks the rows blockIdx.x, blockIdx.x + grid, ...; its columns' sums
// over these rows stay in registers and go to cols[(CTA * 2 + which) * n + column] at the end.
template <class T, int W, int THREADS, int E>
__global__ void __launch_bounds__(THREADS) nk_norm_grad_kernel(T* out, const T* err, const T* src, const T* __restrict__ gain, const T* __restrict__ stats, T* __restrict__ cols,
                                                               const NormPlan p) {
    constexpr int NV = E / W;
    __shared__ T warps[2][2][THREADS / 32], parts[2][2];
    cg::cluster_group cluster = cg::this_cluster();
    const int size = int(cluster.num_blocks()), rank = int(cluster.block_rank());
    const int64_t c0 = int64_t(rank) * THREADS * E, step = gridDim.x / unsigned(size), first = blockIdx.x / unsigned(size);
    const T n = T(p.n);
    T gv[NV][W], sg[NV][W], ss[NV][W];
#pragma unroll
    for (int k = 0; k < NV; k++)
#pragma unroll
        for (int j = 0; j < W; j++) {
            const int64_t c = c0 + (k * THREADS + int(threadIdx.x)) * W + j;
            gv[k][j] = gain && c < p.n ? gain[c * p.gain_s] : T(1);
            sg[k][j] = ss[k][j] = T(0);
        }
    int turn = 0;
    for (int64_t row = first; row < p.rows; row += step, turn++) {
        const T *x = src + norm_row<1>(p, row), *e = err + norm_row<2>(p, row);
        const T mean = stats[row], rstd = stats[p.rows + row];
        T xh[NV][W], ev[NV][W], s1 = T(0), s2 = T(0);
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int64_t c = c0 + (k * THREADS + int(threadIdx.x)) * W;
            norm_load<T, W>(x, c, p.inner[1], p.n, xh[k]);
            norm_load<T, W>(e, c, p.inner[2], p.n, ev[k]);   // zero past the end: nothing is added there
        }
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
            for (int j = 0; j < W; j++) {
                xh[k][j] = (xh[k][j] - mean) * rstd;
                sg[k][j] += ev[k][j] * xh[k][j];
                ss[k][j] += ev[k][j];
                const T g = ev[k][j] * gv[k][j];
                s1 += g;
                s2 += g * xh[k][j];
            }
        if (!out) continue;
        norm_sum2<T, THREADS>(s1, s2, warps[turn & 1]);
        if (size > 1) {
            if (threadIdx.x == 0) { parts[turn & 1][0] = s1; parts[turn & 1][1] = s2; }
            cluster.sync();
            s1 = s2 = T(0);
            for (int r = 0; r < size; r++) {
                const T* theirs = cluster.map_shared_rank(&parts[turn & 1][0], r);
                s1 += theirs[0];
                s2 += theirs[1];
            }
        }
        const T m1 = s1 / n, m2 = s2 / n;
        T* o = out + norm_row<0>(p, row);
#pragma unroll
        for (int k = 0; k < NV; k++) {
#pragma unroll
            for (int j = 0; j < W; j++) ev[k][j] = rstd * (ev[k][j] * gv[k][j] - m1 - xh[k][j] * m2);
            norm_store<T, W>(o, c0 + (k * THREADS + int(threadIdx.x)) * W, p.inner[0], p.n, ev[k]);
        }
    }
    if (size > 1) cluster.sync();   // nobody leaves while its sums may still be read
    if (!cols) return;
    T* part = cols + first * 2 * p.n;
#pragma unroll
    for (int k = 0; k < NV; k++) {
        const int64_t c = c0 + (k * THREADS + int(threadIdx.x)) * W;
        norm_store<T, W>(part, c, 1, p.n, sg[k]);
        norm_store<T, W>(part + p.n, c, 1, p.n, ss[k]);
    }
}
// The same with a row per group of G lanes; the groups of a CTA add their column sums through shared memory at the end, in order.
template <class T, int W, int G, int E>
__global__ void __launch_bounds__(256) nk_norm_grad_lanes_kernel(T* out, const T* err, const T* src, const T* __restrict__ gain, const T* __restrict__ stats, T* __restrict__ cols,
                                                                 const NormPlan p) {
    constexpr int NV = E / W, ROWS = 256 / G;
    __shared__ T sums[2][G * E];
    const int lane = threadIdx.x % G, group = threadIdx.x / G;
    const T n = T(p.n);
    T gv[NV][W], sg[NV][W], ss[NV][W];
#pragma unroll
    for (int k = 0; k < NV; k++)
#pragma unroll
        for (int j = 0; j < W; j++) {
            const int c = (k * G + lane) * W + j;
            gv[k][j] = gain && c < p.n ? gain[c * p.gain_s] : T(1);
            sg[k][j] = ss[k][j] = T(0);
        }
    for (int64_t base = int64_t(blockIdx.x) * ROWS; base < p.rows; base += int64_t(gridDim.x) * ROWS) {
        const bool mine = base + group < p.rows;
        const int64_t row = mine ? base + group : p.rows - 1;
        const T *x = src + norm_row<1>(p, row), *e = err + norm_row<2>(p, row);
        const T mean = stats[row], rstd = stats[p.rows + row];
        T xh[NV][W], ev[NV][W], s1 = T(0), s2 = T(0);
#pragma unroll
        for (int k = 0; k < NV; k++) {
            norm_load<T, W>(x, (k * G + lane) * W, p.inner[1], p.n, xh[k]);
            norm_load<T, W>(e, (k * G + lane) * W, p.inner[2], mine ? p.n : 0, ev[k]);
        }
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
            for (int j = 0; j < W; j++) {
                xh[k][j] = (xh[k][j] - mean) * rstd;
                if (mine) sg[k][j] += ev[k][j] * xh[k][j];   // (the last row's values may not be finite)
                ss[k][j] += ev[k][j];
                const T g = ev[k][j] * gv[k][j];
                s1 += g;
                s2 += g * xh[k][j];
            }
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) { s1 += __shfl_xor_sync(0xffffffffu, s1, o); s2 += __shfl_xor_sync(0xffffffffu, s2, o); }
        if (!out || !mine) continue;
        const T m1 = s1 / n, m2 = s2 / n;
        T* o = out + norm_row<0>(p, row);
#pragma unroll
        for (int k = 0; k < NV; k++) {
#pragma unroll
            for (int j = 0; j < W; j++) ev[k][j] = rstd * (ev[k][j] * gv[k][j] - m1 - xh[k][j] * m2);
            norm_store<T, W>(o, (k * G + lane) * W, p.inner[0], p.n, ev[k]);
        }
    }
    if (!cols) return;
    for (int r = 0; r < ROWS; r++) {
        if (group == r) {
#pragma unroll
            for (int k = 0; k < NV; k++)
#pragma unroll
                for (int j = 0; j < W; j++) {
                    const int c = (k * G + lane) * W + j;
                    sums[0][c] = r ? sums[0][c] + sg[k][j] : sg[k][j];
                    sums[1][c] = r ? sums[1][c] + ss[k][j] : ss[k][j];
                }
        }
        __syncthreads();
    }
    T* part = cols + int64_t(blockIdx.x) * 2 * p.n;
    for (int64_t c = threadIdx.x; c < p.n; c += 256) { part[c] = sums[0][c]; part[p.n + c] = sums[1][c]; }
}

// ---- many rows: one CTA per SM, rows fetched ahead by bulk copies --------------------------------------------------------------------
// A team of TW warps takes a row at a time. Its rows arrive in shared memory by cp.async.bulk, several ahead, so that the memory is kept busy
// through the reductions; the copies need nothing but 16-byte boundaries around a row, so rows that start anywhere cost no more than aligned ones
// (element-wise loads of rows into registers reached a third of the memory's rate). Forward and backward: 16384 x 4096 98 and 153 us (5.5 and 5.3
// TB/s, bound by the memory), 8192 x 8192 92 / 161, 30000 x 1001 47 / 81; rows that a cluster shares wait for its slowest CTA: 2000 x 20000 162 / 227
// (2 TB/s). A row's 16-byte boundaries may lie outside its buffer at
// the buffer's ends: such a row is read by plain loads.
constexpr int STREAM_WARPS = 16, STREAM_THREADS = 512, STREAM_SMEM = 200 * 1024, STREAM_STAGES = 8;

__device__ __forceinline__ void norm_bulk_load(void* smem, const void* gmem, unsigned bytes, uint64_t* bar) {
    const unsigned d = (unsigned)__cvta_generic_to_shared(smem), b = (unsigned)__cvta_generic_to_shared(bar);
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(d), "l"(gmem), "r"(bytes), "r"(b) : "memory");
}
struct StreamCall {
    const char *lo[2], *hi[2];   // the buffers of source and error
    int stages, stage_bytes;     // of the ring; a slot's for one tensor
    int cols;                    // columns of a CTA's slice (n for a CTA alone)
    int* status;
};

// sums over a team, the same in every thread; `turn` alternates between the calls' shared memory
template <class T, int TW, int K>
__device__ __forceinline__ void team_sum(T (&v)[K], T (*smem)[K], int team) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < K; i++) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    if (TW == 1) { __syncwarp(); return; }
    if ((threadIdx.x & 31) == 0)
#pragma unroll
        for (int i = 0; i < K; i++) smem[(threadIdx.x >> 5) % TW][i] = v[i];
    asm volatile("bar.sync %0, %1;\n" ::"r"(1 + team), "n"(TW * 32) : "memory");
#pragma unroll
    for (int i = 0; i < K; i++) {
        v[i] = smem[0][i];
#pragma unroll
        for (int w = 1; w < TW; w++) v[i] += smem[w][i];
    }
}

// What both kernels share: the team's ring of rows. The leader notes where in its slot a row begins (-1: it was not copied).
template <class T, int TW, int TENSORS>
struct StreamRing {
    const NormPlan& p;
    const StreamCall& c;
    unsigned char* base;
    uint64_t* bars;
    int (*places)[TENSORS];
    const T* src[2];
    int64_t step, next;   // rows between this team's rows; the next one to be fetched
    int64_t c0;           // first column of the slice
    int cols;
    int slot, fetch_slot;
    unsigned phase;
    bool leader, dead;

    __device__ __forceinline__ const T* row_of(int t, int64_t row) const { return src[t] + (t ? norm_row<2>(p, row) : norm_row<1>(p, row)) + c0; }
    __device__ __forceinline__ unsigned char* stage(int s, int t) const { return base + (s * TENSORS + t) * c.stage_bytes; }
    // requests the next row into the slot that was consumed last
    __device__ __forceinline__ void fetch() {
        if (leader && !dead && next < p.rows) {
            unsigned bytes[TENSORS], all = 0;
            const char* from[TENSORS];
#pragma unroll
            for (int t = 0; t < TENSORS; t++) {   // the 16-byte blocks around the row, where they lie in its buffer
                const uintptr_t a = reinterpret_cast<uintptr_t>(row_of(t, next)), lo = a & ~uintptr_t(15), hi = (a + unsigned(cols) * sizeof(T) + 15) & ~uintptr_t(15);
                const bool inside = reinterpret_cast<const char*>(lo) >= c.lo[t] && reinterpret_cast<const char*>(hi) <= c.hi[t];
                from[t] = reinterpret_cast<const char*>(lo);
                bytes[t] = inside ? unsigned(hi - lo) : 0u;
                all += bytes[t];
                places[fetch_slot][t] = inside ? int(a - lo) : -1;
            }
            if (all) nk_mbar_expect_tx(&bars[fetch_slot], all);
            else nk_mbar_arrive(&bars[fetch_slot]);
#pragma unroll
            for (int t = 0; t < TENSORS; t++)
                if (bytes[t]) norm_bulk_load(stage(fetch_slot, t), from[t], bytes[t], &bars[fetch_slot]);
        }
        next += step;
        if (++fetch_slot == c.stages) fetch_slot = 0;
    }
    __device__ __forceinline__ void wait() {
        if (dead) return;
        if (nk_mbar_wait_bounded(&bars[slot], phase, NK_WAIT_LIMIT_NS, nullptr) < 0) {
            dead = true;   // nothing more is fetched; what is on its way still lands
            if (c.status) atomicExch(c.status, 1);
            for (int i = 1; leader && i < c.stages; i++)
                if (next - (c.stages - i) * step < p.rows) nk_mbar_wait_bounded(&bars[(slot + i) % c.stages], phase ^ unsigned(slot + i >= c.stages), NK_WAIT_LIMIT_NS, nullptr);
        }
    }
    __device__ __forceinline__ void advance() {
        if (++slot == c.stages) { slot = 0; phase ^= 1u; }
    }
    // where the row of tensor t that is due can be read: shared memory, or (not copied) the row itself
    __device__ __forceinline__ const T* due(int t, int64_t row) const {
        const int at = places[slot][t];
        return at >= 0 ? reinterpret_cast<const T*>(stage(slot, t) + at) : row_of(t, row);
    }
};
template <class T, int W>
__device__ __forceinline__ void stream_read(const T* row, int c, T (&v)[W]) {
    if (W > 1) *reinterpret_cast<typename NormVec<T, W>::type*>(v) = *reinterpret_cast<const typename NormVec<T, W>::type*>(row + c);
    else v[0] = row[c];
}
template <class T, int W>
__device__ __forceinline__ void stream_write(T* row, int c, const T (&v)[W]) {
    if (W > 1) *reinterpret_cast<typename NormVec<T, W>::type*>(row + c) = *reinterpret_cast<const typename NormVec<T, W>::type*>(v);
    else row[c] = v[0];
}
template <class T, int TW, int TENSORS>
__device__ __forceinline__ StreamRing<T, TW, TENSORS> stream_ring(const NormPlan& p, const StreamCall& c, const T* src, const T* err, unsigned char* smem, uint64_t* bars,
                                                               int (*places)[TENSORS]) {
    constexpr int TEAMS = STREAM_WARPS / TW;
    cg::cluster_group cluster = cg::this_cluster();
    const int size = int(cluster.num_blocks()), rank = int(cluster.block_rank()), team = (threadIdx.x >> 5) / TW;
    if (threadIdx.x < unsigned(TEAMS * STREAM_STAGES)) {
        nk_mbar_init(&bars[threadIdx.x], 1);
        nk_fence_barrier_init();
        nk_fence_proxy_async();
    }
    __syncthreads();
    StreamRing<T, TW, TENSORS> r{p, c};
    r.base = smem + size_t(team) * c.stages * TENSORS * c.stage_bytes;
    r.bars = bars + team * STREAM_STAGES;
    r.places = places + team * STREAM_STAGES;
    r.src[0] = src;
    r.src[1] = err;
    r.step = int64_t(gridDim.x / unsigned(size)) * TEAMS;
    r.next = int64_t(blockIdx.x / unsigned(size)) * TEAMS + team;
    r.c0 = int64_t(rank) * c.cols;
    r.cols = p.n - r.c0 < c.cols ? int(p.n - r.c0) : c.cols;
    r.slot = r.fetch_slot = 0;
    r.phase = 0;
    r.leader = threadIdx.x % (TW * 32) == 0;
    r.dead = false;
    return r;
}

// A lane's vectors k < mine of a slice, SPAN columns apart. No thread of the team has more than `most`, which is looked at every fourth time (a branch
// per vector keeps their loads from being in flight together; none costs the instructions of vectors that nobody has).
#define NK_EACH(k) _Pragma("unroll") for (int k = 0; k < NV; k++) if (k % 4 == 0 && k >= most) break; else if (k < mine)

template <class T, int W, int TW, int E>
__global__ void __launch_bounds__(STREAM_THREADS, 1) nk_norm_stream_kernel(T* out, const T* src, const T* __restrict__ gain, const T* __restrict__ shift, T* __restrict__ stats,
                                                                          const NormPlan p, T eps, const StreamCall call) {
    constexpr int NV = E / W, TEAMS = STREAM_WARPS / TW, SPAN = TW * 32 * W;
    extern __shared__ __align__(16) unsigned char stream_smem[];
    __shared__ uint64_t bars[TEAMS * STREAM_STAGES];
    __shared__ int places[TEAMS * STREAM_STAGES][1];
    __shared__ T sums[3][TEAMS][TW][1], parts[2][3];
    cg::cluster_group cluster = cg::this_cluster();
    const int size = int(cluster.num_blocks());
    auto ring = stream_ring<T, TW, 1>(p, call, src, static_cast<const T*>(nullptr), stream_smem, bars, places);
    const int team = (threadIdx.x >> 5) / TW, c_lane = int(threadIdx.x % (TW * 32)) * W, cols = ring.cols;
    const int most = (cols + SPAN - 1) / SPAN, mine = c_lane < cols ? (cols - c_lane + SPAN - 1) / SPAN : 0;
    const T inv_n = T(1) / T(p.n), inv_cols = T(1) / T(cols);
    T gv[NV][W], sv[NV][W];
    NK_EACH(k) {
#pragma unroll
        for (int j = 0; j < W; j++) {
            const int64_t c = ring.c0 + c_lane + k * SPAN + j;
            gv[k][j] = gain ? gain[c * p.gain_s] : T(1);
            sv[k][j] = shift ? shift[c * p.shift_s] : T(0);
        }
    }
    int64_t row = ring.next;
    for (int s = 0; s < call.stages; s++) ring.fetch();
    for (int turn = 0; row < p.rows; row += ring.step, turn++) {
        ring.wait();
        const T* x = ring.due(0, row) + c_lane;
        T v[NV][W], sum[1] = {T(0)};
        NK_EACH(k) {
            stream_read<T, W>(x, k * SPAN, v[k]);
#pragma unroll
            for (int j = 0; j < W; j++) sum[0] += v[k][j];
        }
        team_sum<T, TW, 1>(sum, sums[0][team], team);   // (a barrier of the team: the row has been read)
        ring.fetch();
        ring.advance();
        T mean = sum[0] * inv_cols, m2[1] = {T(0)};
        NK_EACH(k) {
#pragma unroll
            for (int j = 0; j < W; j++) m2[0] += (v[k][j] - mean) * (v[k][j] - mean);
        }
        team_sum<T, TW, 1>(m2, sums[1][team], team);
        if (size > 1) {   // the slices' means and squares: mu = sum(n_i mu_i) / n, v = sum(m2_i + n_i (mu_i - mu)^2) / n
            if (threadIdx.x == 0) { parts[turn & 1][0] = mean; parts[turn & 1][1] = m2[0]; }
            cluster.sync();
            T all = T(0), all2 = T(0);
            for (int r = 0; r < size; r++) {
                const int64_t left = p.n - int64_t(r) * call.cols;
                all += T(left < call.cols ? left : call.cols) * cluster.map_shared_rank(&parts[turn & 1][0], r)[0];
            }
            all *= inv_n;
            for (int r = 0; r < size; r++) {
                const int64_t left = p.n - int64_t(r) * call.cols;
                const T* theirs = cluster.map_shared_rank(&parts[turn & 1][0], r);
                const T d = theirs[0] - all;
                all2 += theirs[1] + T(left < call.cols ? left : call.cols) * d * d;
            }
            mean = all;
            m2[0] = all2;
        }
        const T v2 = m2[0] * inv_n;
        T rstd = T(1) / sqrt(v2 + eps);
        if (norm_far(mean, v2)) {
            const T from = norm_again(mean);
            T off[1] = {T(0)};
            NK_EACH(k) {
#pragma unroll
                for (int j = 0; j < W; j++) off[0] += v[k][j] - from;
            }
            team_sum<T, TW, 1>(off, sums[2][team], team);
            if (size > 1) {
                if (threadIdx.x == 0) parts[turn & 1][2] = off[0];
                cluster.sync();
                off[0] = T(0);
                for (int r = 0; r < size; r++) off[0] += cluster.map_shared_rank(&parts[turn & 1][0], r)[2];
            }
            norm_settle(mean, rstd, m2[0], off[0], T(p.n), eps);
        }
        if (stats && ring.c0 == 0 && ring.leader) { stats[row] = mean; stats[p.rows + row] = rstd; }
        T* y = out + norm_row<0>(p, row) + ring.c0 + c_lane;
        NK_EACH(k) {
#pragma unroll
            for (int j = 0; j < W; j++) v[k][j] = (v[k][j] - mean) * rstd * gv[k][j] + sv[k][j];
            stream_write<T, W>(y, k * SPAN, v[k]);
        }
    }
    if (size > 1) cluster.sync();   // nobody leaves while its sums may still be read
}

template <class T, int W, int TW, int E>
__global__ void __launch_bounds__(STREAM_THREADS, 1) nk_norm_grad_stream_kernel(T* out, const T* err, const T* src, const T* __restrict__ gain, const T* __restrict__ stats,
                                                                               T* __restrict__ cols_out, const NormPlan p, const StreamCall call) {
    constexpr int NV = E / W, TEAMS = STREAM_WARPS / TW, SPAN = TW * 32 * W;
    extern __shared__ __align__(16) unsigned char stream_smem[];
    __shared__ uint64_t bars[TEAMS * STREAM_STAGES];
    __shared__ int places[TEAMS * STREAM_STAGES][2];
    __shared__ T sums[2][TEAMS][TW][2], parts[2][2];
    cg::cluster_group cluster = cg::this_cluster();
    const int size = int(cluster.num_blocks());
    auto ring = stream_ring<T, TW, 2>(p, call, src, err, stream_smem, bars, places);
    const int team = (threadIdx.x >> 5) / TW, c_lane = int(threadIdx.x % (TW * 32)) * W, cols = ring.cols;
    const int most = (cols + SPAN - 1) / SPAN, mine = c_lane < cols ? (cols - c_lane + SPAN - 1) / SPAN : 0;
    const T inv_n = T(1) / T(p.n);
    T gv[NV][W], sg[NV][W], ss[NV][W];
#pragma unroll
    for (int k = 0; k < NV; k++)
#pragma unroll
        for (int j = 0; j < W; j++) {
            gv[k][j] = gain && k < mine ? gain[(ring.c0 + c_lane + k * SPAN + j) * p.gain_s] : T(1);
            sg[k][j] = ss[k][j] = T(0);
        }
    int64_t row = ring.next;
    for (int s = 0; s < call.stages; s++) ring.fetch();
    T mean = T(0), rstd = T(0);
    if (row < p.rows) { mean = stats[row]; rstd = stats[p.rows + row]; }
    for (int turn = 0; row < p.rows; row += ring.step, turn++) {
        T next_mean = T(0), next_rstd = T(0);   // of the row after: on their way during this one
        if (row + ring.step < p.rows) { next_mean = stats[row + ring.step]; next_rstd = stats[p.rows + row + ring.step]; }
        ring.wait();
        const T *x = ring.due(0, row) + c_lane, *e = ring.due(1, row) + c_lane;
        T xh[NV][W], g[NV][W], s[2] = {T(0), T(0)};
        NK_EACH(k) {
            T ev[W];
            stream_read<T, W>(x, k * SPAN, xh[k]);
            stream_read<T, W>(e, k * SPAN, ev);
#pragma unroll
            for (int j = 0; j < W; j++) {
                xh[k][j] = (xh[k][j] - mean) * rstd;
                sg[k][j] += ev[j] * xh[k][j];
                ss[k][j] += ev[j];
                g[k][j] = ev[j] * gv[k][j];
                s[0] += g[k][j];
                s[1] += g[k][j] * xh[k][j];
            }
        }
        team_sum<T, TW, 2>(s, sums[turn & 1][team], team);   // (a barrier of the team: the row has been read)
        ring.fetch();
        ring.advance();
        if (size > 1) {
            if (threadIdx.x == 0) { parts[turn & 1][0] = s[0]; parts[turn & 1][1] = s[1]; }
            cluster.sync();
            s[0] = s[1] = T(0);
            for (int r = 0; r < size; r++) {
                const T* theirs = cluster.map_shared_rank(&parts[turn & 1][0], r);
                s[0] += theirs[0];
                s[1] += theirs[1];
            }
        }
        if (out) {
            const T m1 = s[0] * inv_n, m2 = s[1] * inv_n;
            T* o = out + norm_row<0>(p, row) + ring.c0 + c_lane;
            NK_EACH(k) {
#pragma unroll
                for (int j = 0; j < W; j++) g[k][j] = rstd * (g[k][j] - m1 - xh[k][j] * m2);
                stream_write<T, W>(o, k * SPAN, g[k]);
            }
        }
        mean = next_mean;
        rstd = next_rstd;
    }
    if (size > 1) cluster.sync();   // nobody leaves while its sums may still be read
    if (!cols_out) return;
    T* part = cols_out + int64_t(blockIdx.x / unsigned(size)) * 2 * p.n + ring.c0;
    if (TEAMS == 1) {
        NK_EACH(k) {
            stream_write<T, W>(part + c_lane, k * SPAN, sg[k]);
            stream_write<T, W>(part + p.n + c_lane, k * SPAN, ss[k]);
        }
        return;
    }
    // the teams' column sums, one after the other (all rows have been read: the ring's memory is free)
    T* all = reinterpret_cast<T*>(stream_smem);
    for (int t = 0; t < TEAMS; t++) {
        __syncthreads();
        if (team != t) continue;
        NK_EACH(k) {
#pragma unroll
            for (int j = 0; j < W; j++) {
                const int c = c_lane + k * SPAN + j;
                all[c] = t ? all[c] + sg[k][j] : sg[k][j];
                all[cols + c] = t ? all[cols + c] + ss[k][j] : ss[k][j];
            }
        }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < cols; c += STREAM_THREADS) { part[c] = all[c]; part[p.n + c] = all[cols + c]; }
}
#undef NK_EACH

// ---- rows of any length: cut into chunks of NORM_THREADS * W * 8 elements, a CTA per chunk ---------------------------------------
// The row is read twice (the second time from L2 where the call fits it); the mean and the variance cross a launch boundary in between.
constexpr int NORM_NV = 8;

// mean and sum of squared differences to it, per chunk: part[(row * chunks + chunk) * 2]
template <class T, int W>
__global__ void __launch_bounds__(NORM_THREADS) nk_norm_chunk_stats_kernel(const T* __restrict__ src, T* __restrict__ part, const NormPlan p, int64_t chunks) {
    __shared__ T smem[NORM_THREADS / 32];
    constexpr int64_t L = int64_t(NORM_THREADS) * W * NORM_NV;
    for (int64_t u = blockIdx.x; u < p.rows * chunks; u += gridDim.x) {
        const int64_t row = u / chunks, c0 = (u - row * chunks) * L, left = p.n - c0 < L ? p.n - c0 : L;
        const T* x = src + norm_row<1>(p, row);
        T v[NORM_NV][W], sum = T(0);
#pragma unroll
        for (int k = 0; k < NORM_NV; k++) {
            norm_load<T, W>(x, c0 + (k * NORM_THREADS + threadIdx.x) * W, p.inner[1], p.n, v[k]);
#pragma unroll
            for (int j = 0; j < W; j++) sum += v[k][j];
        }
        T mean = norm_cta_sum(sum, smem) / T(left), m2 = T(0), off = T(0);
#pragma unroll
        for (int k = 0; k < NORM_NV; k++)
#pragma unroll
            for (int j = 0; j < W; j++)
                if (c0 + (k * NORM_THREADS + threadIdx.x) * W + j < p.n) {
                    const T d = v[k][j] - mean;
                    off += d;
                    m2 += d * d;
                }
        off = norm_cta_sum(off, smem);   // (corrects the mean, as norm_settle does)
        m2 = norm_cta_sum(m2, smem);
        const T by = off / T(left);
        mean += by;
        m2 = m2 - off * by > T(0) ? m2 - off * by : T(0);
        if (threadIdx.x == 0) { part[2 * u] = mean; part[2 * u + 1] = m2; }
    }
}
// The row's mean and variance from its chunks': mu = mean_0 + sum(n_i (mean_i - mean_0)) / n, v = sum(m2_i + n_i (mean_i - mu)^2) / n; then the chunk's results.
template <class T, int W>
__global__ void __launch_bounds__(NORM_THREADS) nk_norm_chunk_apply_kernel(T* out, const T* src, const T* __restrict__ part, const T* __restrict__ gain,
                                                                           const T* __restrict__ shift, T* __restrict__ stats, const NormPlan p, int64_t chunks, T eps) {
    __shared__ T smem[NORM_THREADS / 32];
    constexpr int64_t L = int64_t(NORM_THREADS) * W * NORM_NV;
    for (int64_t u = blockIdx.x; u < p.rows * chunks; u += gridDim.x) {
        const int64_t row = u / chunks, chunk = u - row * chunks, c0 = chunk * L;
        auto length = [&](int64_t i) { return T(i + 1 < chunks ? L : p.n - i * L); };
        const T base = part[2 * row * chunks];
        T sum = T(0);
        for (int64_t i = threadIdx.x; i < chunks; i += NORM_THREADS) sum += length(i) * (part[2 * (row * chunks + i)] - base);
        const T mean = base + norm_cta_sum(sum, smem) / T(p.n);
        T m2 = T(0);
        for (int64_t i = threadIdx.x; i < chunks; i += NORM_THREADS) {
            const T d = part[2 * (row * chunks + i)] - mean;
            m2 += part[2 * (row * chunks + i) + 1] + length(i) * d * d;
        }
        const T rstd = T(1) / sqrt(norm_cta_sum(m2, smem) / T(p.n) + eps);
        if (stats && chunk == 0 && threadIdx.x == 0) { stats[row] = mean; stats[p.rows + row] = rstd; }
        const T* x = src + norm_row<1>(p, row);
        T* y = out + norm_row<0>(p, row);
#pragma unroll
        for (int k = 0; k < NORM_NV; k++) {
            const int64_t c = c0 + (k * NORM_THREADS + threadIdx.x) * W;
            T v[W];
            norm_load<T, W>(x, c, p.inner[1], p.n, v);
#pragma unroll
            for (int j = 0; j < W; j++) {
                v[j] = (v[j] - mean) * rstd;
                if (c + j < p.n) {
                    if (gain) v[j] *= gain[(c + j) * p.gain_s];
                    if (shift) v[j] += shift[(c + j) * p.shift_s];
                }
            }
            norm_store<T, W>(y, c, p.inner[0], p.n, v);
        }
    }
}

// sum(g) and sum(g * xh), per chunk
template <class T, int W>
__global__ void __launch_bounds__(NORM_THREADS) nk_norm_chunk_sums_kernel(const T* __restrict__ err, const T* __restrict__ src, const T* __restrict__ gain,
                                                                          const T* __restrict__ stats, T* __restrict__ part, const NormPlan p, int64_t chunks) {
    __shared__ T smem[NORM_THREADS / 32];
    constexpr int64_t L = int64_t(NORM_THREADS) * W * NORM_NV;
    for (int64_t u = blockIdx.x; u < p.rows * chunks; u += gridDim.x) {
        const int64_t row = u / chunks, c0 = (u - row * chunks) * L;
        const T *x = src + norm_row<1>(p, row), *e = err + norm_row<2>(p, row);
        const T mean = stats[row], rstd = stats[p.rows + row];
        T s1 = T(0), s2 = T(0);
#pragma unroll
        for (int k = 0; k < NORM_NV; k++) {
            const int64_t c = c0 + (k * NORM_THREADS + threadIdx.x) * W;
            T xv[W], ev[W];
            norm_load<T, W>(x, c, p.inner[1], p.n, xv);
            norm_load<T, W>(e, c, p.inner[2], p.n, ev);
#pragma unroll
            for (int j = 0; j < W; j++)
                if (c + j < p.n) {
                    const T g = gain ? ev[j] * gain[(c + j) * p.gain_s] : ev[j];
                    s1 += g;
                    s2 += g * ((xv[j] - mean) * rstd);
                }
        }
        s1 = norm_cta_sum(s1, smem);
        s2 = norm_cta_sum(s2, smem);
        if (threadIdx.x == 0) { part[2 * u] = s1; part[2 * u + 1] = s2; }
    }
}
// the chunks' sums to the row's means, a warp per row: means[row], means[rows + row]
template <class T>
__global__ void __launch_bounds__(NORM_THREADS) nk_norm_row_means_kernel(const T* __restrict__ part, T* __restrict__ means, int64_t rows, int64_t chunks, T n) {
    const int lane = threadIdx.x & 31;
    for (int64_t row = int64_t(blockIdx.x) * (NORM_THREADS / 32) + (threadIdx.x >> 5); row < rows; row += int64_t(gridDim.x) * (NORM_THREADS / 32)) {
        T s1 = T(0), s2 = T(0);
        for (int64_t i = lane; i < chunks; i += 32) { s1 += part[2 * (row * chunks + i)]; s2 += part[2 * (row * chunks + i) + 1]; }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) { s1 += __shfl_xor_sync(0xffffffffu, s1, o); s2 += __shfl_xor_sync(0xffffffffu, s2, o); }
        if (lane == 0) { means[row] = s1 / n; means[rows + row] = s2 / n; }
    }
}
// A thread owns W columns and walks a group of rows: dx, and the group's part of the column sums, cols[(group * 2 + which) * n + column].
template <class T, int W>
__global__ void __launch_bounds__(NORM_THREADS) nk_norm_columns_kernel(T* out, const T* err, const T* src, const T* __restrict__ gain, const T* __restrict__ stats,
                                                                       const T* __restrict__ means, T* __restrict__ cols, const NormPlan p, int64_t groups, int64_t per) {
    const int64_t blocks_c = (p.n + NORM_THREADS * W - 1) / (NORM_THREADS * W);
    for (int64_t u = blockIdx.x; u < blocks_c * groups; u += gridDim.x) {
        const int64_t group = u / blocks_c, c = ((u - group * blocks_c) * NORM_THREADS + threadIdx.x) * W;
        if (c >= p.n) continue;
        const int64_t r1 = (group + 1) * per < p.rows ? (group + 1) * per : p.rows;
        T gv[W], sg[W], ss[W];
#pragma unroll
        for (int j = 0; j < W; j++) { gv[j] = gain ? gain[(c + j) * p.gain_s] : T(1); sg[j] = ss[j] = T(0); }
        for (int64_t row = group * per; row < r1; row++) {
            const T mean = stats[row], rstd = stats[p.rows + row];
            T xv[W], ev[W];
            norm_load<T, W>(src + norm_row<1>(p, row), c, p.inner[1], p.n, xv);
            norm_load<T, W>(err + norm_row<2>(p, row), c, p.inner[2], p.n, ev);
#pragma unroll
            for (int j = 0; j < W; j++) {
                const T xh = (xv[j] - mean) * rstd;
                sg[j] += ev[j] * xh;
                ss[j] += ev[j];
                if (out) xv[j] = rstd * (ev[j] * gv[j] - means[row] - xh * means[p.rows + row]);
            }
            if (out) norm_store<T, W>(out + norm_row<0>(p, row), c, p.inner[0], p.n, xv);
        }
        if (cols) {
            norm_store<T, W>(cols + (group * 2) * p.n, c, 1, p.n, sg);
            norm_store<T, W>(cols + (group * 2 + 1) * p.n, c, 1, p.n, ss);
        }
    }
}
// The groups' parts of the column sums: 32 columns per CTA, 32 threads per column take every 32nd group, in order, and are added in order.
template <class T>
__global__ void __launch_bounds__(1024) nk_norm_columns_finish_kernel(T* dgain, int64_t dgain_s, T* dshift, int64_t dshift_s, const T* __restrict__ cols, int64_t n, int64_t groups) {
    __shared__ T sums[2][32][33];
    const int lane = threadIdx.x & 31, slot = threadIdx.x >> 5;
    for (int64_t c0 = int64_t(blockIdx.x) * 32; c0 < n; c0 += int64_t(gridDim.x) * 32) {
        const int64_t c = c0 + lane;
        T sg = T(0), ss = T(0);
        if (c < n) {
#pragma unroll 4
            for (int64_t g = slot; g < groups; g += 32) { sg += cols[(g * 2) * n + c]; ss += cols[(g * 2 + 1) * n + c]; }
        }
        __syncthreads();   // the sums of the columns before have been read
        sums[0][slot][lane] = sg;
        sums[1][slot][lane] = ss;
        __syncthreads();
        if (slot < 2 && c < n) {
            T v = sums[slot][0][lane];
#pragma unroll
            for (int k = 1; k < 32; k++) v += sums[slot][k][lane];
            if (slot == 0 && dgain) dgain[c * dgain_s] = v;
            if (slot == 1 && dshift) dshift[c * dshift_s] = v;
        }
    }
}

// ---- host side -----------------------------------------------------------------------------------------------------------------
// The outer dims of up to three views of one shape, size-1 dims dropped, neighbours merged where every operand is linear across them.
void norm_plan(const NkView* const (&v)[3], NormPlan* p) {
    memset(p, 0, sizeof(*p));
    const NkView& shape = *v[1];
    p->rows = 1;
    for (int k = 0; k + 1 < shape.rank; k++) {
        const int64_t e = shape.shape[k];
        p->rows *= e;
        if (e == 1) continue;
        const int l = p->nd - 1;
        bool merge = l >= 0;
        for (int t = 0; t < 3 && merge; t++) merge = !v[t] || p->s[t][l] == e * v[t]->estride[k];
        const int at = merge ? l : p->nd++;
        p->ext[at] = merge ? p->ext[at] * e : e;
        for (int t = 0; t < 3; t++) p->s[t][at] = v[t] ? v[t]->estride[k] : 0;
    }
    if (p->nd == 0) { p->nd = 1; p->ext[0] = 1; }
    p->n = shape.shape[shape.rank - 1];
    for (int t = 0; t < 3; t++) p->inner[t] = v[t] ? v[t]->estride[shape.rank - 1] : 1;
}
// 16-byte accesses along the rows of operand t
template <class T>
bool norm_vec(const NormPlan& p, int t, const T* base) {
    if (p.inner[t] != 1 || p.n % norm_w<T>() || reinterpret_cast<uintptr_t>(base) % 16) return false;
    for (int k = 0; k < p.nd; k++)
        if (p.s[t][k] % norm_w<T>()) return false;
    return true;
}

// at most per_sm CTAs per SM (the backward calls' are resident at once, since each leaves its column sums; the forward calls' are several waves, so that the
// hardware evens out what rows take); a cluster's CTAs lie side by side
template <class... A>
int norm_launch(nk_ctx* ctx, const char* name, void (*kern)(A...), int64_t rows, int threads, int cluster, int per_sm, A... args) {
    int64_t units = int64_t(ctx->prop.multiProcessorCount) * per_sm / cluster;
    if (units > rows) units = rows;
    if (units < 1) units = 1;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(unsigned(units * cluster));
    cfg.blockDim = dim3(threads);
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = cluster;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = cluster > 1 ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
    if (e != cudaSuccess) return nk_cuda_fail(ctx, e, name);
    return nk_after_launch(ctx, name);
}
// elements that a thread of the CTA kernels holds at most, and the longest row that they take (a cluster of eight)
template <class T> constexpr int norm_e() { return 128 / int(sizeof(T)); }

// Rows by bulk copies: at least two of them for every team, running along memory, and long: up to 256 elements on 16-byte boundaries a group of lanes
// per row is as fast or faster (200000 x 200: forward 109 us against 106, backward 133 against 158; 200000 x 203, which has no such
// boundaries: 139 against 107 and 229 against 152).
template <class T> constexpr int stream_e() { return 64 / int(sizeof(T)); }
struct StreamShape {
    int team, cluster, stages, stage_bytes, cols, grid;
    size_t smem;
};
// Clusters of CTAs of the kernels above that are resident at once (a GPU's SMs come in groups of unlike size that a cluster has to fit into: one that
// waits for room would run by itself at the end). Looked up once per device and size.
int stream_clusters(const nk_ctx* ctx, int size) {
    static std::atomic<int> known[16][9];
    if (size == 1) return ctx->prop.multiProcessorCount;
    std::atomic<int>* slot = ctx->device < 16 ? &known[ctx->device][size] : nullptr;
    int n = slot ? slot->load() : 0;
    if (n > 0) return n;
    auto* kern = nk_norm_grad_stream_kernel<float, 1, 16, 16>;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(unsigned(size));
    cfg.blockDim = dim3(STREAM_THREADS);
    cfg.dynamicSmemBytes = STREAM_SMEM;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = unsigned(size);
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, STREAM_SMEM) != cudaSuccess || cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n < 1) {
        cudaGetLastError();
        n = ctx->prop.multiProcessorCount / size / 2;
    }
    if (slot) slot->store(n);
    return n;
}
template <class T>
bool stream_shape(const nk_ctx* ctx, const NormPlan& p, int tensors, bool vec, StreamShape* s) {
    constexpr int E = stream_e<T>();
    if (p.n <= (vec ? 256 : 128) || p.inner[1] != 1 || (tensors == 2 && p.inner[2] != 1) || p.inner[0] != 1 || !p.lo[0]) return false;
    s->team = 1;
    while (s->team < STREAM_WARPS && int64_t(s->team) * 32 * E < p.n) s->team *= 2;
    s->cluster = 1;
    while (s->cluster < 8 && int64_t(s->cluster) * s->team * 32 * E < p.n) s->cluster *= 2;
    if (int64_t(s->cluster) * s->team * 32 * E < p.n) return false;
    s->cols = s->cluster > 1 ? int(((p.n + s->cluster - 1) / s->cluster + 3) / 4 * 4) : int(p.n);   // even slices, on 16-byte boundaries of an aligned row
    const int teams = STREAM_WARPS / s->team;
    s->grid = stream_clusters(ctx, s->cluster) * s->cluster;
    if (p.rows < int64_t(s->grid / s->cluster) * teams * 2) return false;
    s->stage_bytes = int((size_t(s->cols) * sizeof(T) + 30) / 16 * 16);
    s->stages = int(STREAM_SMEM / (size_t(teams) * tensors * s->stage_bytes));
    if (s->stages > STREAM_STAGES) s->stages = STREAM_STAGES;
    s->smem = size_t(teams) * s->stages * tensors * s->stage_bytes;
    return s->stages >= 2;
}
template <class... A>
int stream_launch(nk_ctx* ctx, const char* name, void (*kern)(A...), const StreamShape& s, A... args) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, STREAM_SMEM);
    if (e != cudaSuccess) return nk_cuda_fail(ctx, e, name);
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(unsigned(s.grid));
    cfg.blockDim = dim3(STREAM_THREADS);
    cfg.dynamicSmemBytes = s.smem;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = unsigned(s.cluster);
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = s.cluster > 1 ? 1 : 0;
    e = cudaLaunchKernelEx(&cfg, kern, args...);
    if (e != cudaSuccess) return nk_cuda_fail(ctx, e, name);
    return nk_after_launch(ctx, name);
}
StreamCall stream_call(const nk_ctx* ctx, const NormPlan& p, const StreamShape& s) {
    StreamCall c;
    for (int t = 0; t < 2; t++) { c.lo[t] = p.lo[t]; c.hi[t] = p.hi[t]; }
    c.stages = s.stages;
    c.stage_bytes = s.stage_bytes;
    c.cols = s.cols;
    c.status = ctx->tma_status_dev;
    return c;
}
template <class T, int W>
int forward_stream(nk_ctx* ctx, const StreamShape& s, T* out, const T* src, const T* gain, const T* shift, T* stats, const NormPlan& p, T eps) {
    constexpr int E = stream_e<T>();
    const StreamCall c = stream_call(ctx, p, s);
#define NK_TEAM(TW) case TW: return stream_launch(ctx, "nk_norm_stream_kernel", nk_norm_stream_kernel<T, W, TW, E>, s, out, src, gain, shift, stats, p, eps, c)
    switch (s.team) { NK_TEAM(1); NK_TEAM(2); NK_TEAM(4); NK_TEAM(8); default: NK_TEAM(16); }
#undef NK_TEAM
}

template <class T, int W>
int forward_rows(nk_ctx* ctx, T* out, const T* src, const T* gain, const T* shift, T* stats, const NormPlan& p, T eps) {
    constexpr int E = norm_e<T>();
#define NK_LANES(G, EL) return norm_launch(ctx, "nk_norm_lanes_kernel", nk_norm_lanes_kernel<T, W, G, EL>, (p.rows + 256 / G - 1) / (256 / G), 256, 1, 32, out, src, gain, shift, stats, p, eps)
#define NK_CTA(TH, EL, C) return norm_launch(ctx, "nk_norm_cta_kernel", nk_norm_cta_kernel<T, W, TH, EL>, p.rows, TH, C, 16, out, src, gain, shift, stats, p, eps)
    if (p.n <= 32) NK_LANES(8, 4);
    if (p.n <= 64) NK_LANES(16, 4);
    if (p.n <= 128) NK_LANES(32, 4);
    if (p.n <= 256) NK_LANES(32, 8);
    if (p.n <= 512) NK_LANES(32, 16);
    if (p.n <= 1024) NK_CTA(128, 8, 1);
    if (p.n <= 2048) NK_CTA(256, 8, 1);
    if (p.n <= 4096) NK_CTA(256, 16, 1);
    if (p.n <= 256 * E) NK_CTA(256, E, 1);
    if (p.n <= 512 * E) NK_CTA(512, E, 1);
    const int cluster = p.n <= 1024 * E ? 2 : p.n <= 2048 * E ? 4 : 8;
    NK_CTA(512, E, cluster);
#undef NK_LANES
#undef NK_CTA
}

template <class T, int W>
int forward_w(nk_ctx* ctx, T* out, const T* src, const T* gain, const T* shift, T* stats, const NormPlan& p, T eps) {
    StreamShape shape;
    if (stream_shape<T>(ctx, p, 1, W > 1, &shape)) return forward_stream<T, W>(ctx, shape, out, src, gain, shift, stats, p, eps);
    if (p.n <= 4096 * norm_e<T>()) return forward_rows<T, W>(ctx, out, src, gain, shift, stats, p, eps);
    constexpr int64_t L = int64_t(NORM_THREADS) * W * NORM_NV;
    const int64_t chunks = (p.n + L - 1) / L;
    NkWorkspace ws(ctx);
    int st = ws.get(size_t(p.rows) * chunks * 2 * sizeof(T));
    if (st) return st;
    T* part = static_cast<T*>(ws.ptr);
    const int grid = nk_grid_for(ctx, p.rows * chunks, 1, 32);
    nk_norm_chunk_stats_kernel<T, W><<<grid, NORM_THREADS, 0, ctx->stream>>>(src, part, p, chunks);
    if ((st = nk_after_launch(ctx, "nk_norm_chunk_stats_kernel"))) return st;
    nk_norm_chunk_apply_kernel<T, W><<<grid, NORM_THREADS, 0, ctx->stream>>>(out, src, part, gain, shift, stats, p, chunks, eps);
    return nk_after_launch(ctx, "nk_norm_chunk_apply_kernel");
}
template <class T>
int forward(nk_ctx* ctx, T* out, const T* src, const T* gain, const T* shift, T* stats, const NormPlan& p, double eps) {
    if (norm_vec(p, 0, out) && norm_vec(p, 1, src)) return forward_w<T, norm_w<T>()>(ctx, out, src, gain, shift, stats, p, T(eps));
    return forward_w<T, 1>(ctx, out, src, gain, shift, stats, p, T(eps));
}

template <class T>
struct NormGrad {
    T *out, *dgain, *dshift;
    const T *err, *src, *gain, *stats;
    int64_t dgain_s, dshift_s;
};
template <class T>
int columns_finish(nk_ctx* ctx, const NormGrad<T>& a, const T* cols, int64_t n, int64_t groups) {
    nk_norm_columns_finish_kernel<T><<<nk_grid_for(ctx, n, 32, 32), 1024, 0, ctx->stream>>>(a.dgain, a.dgain_s, a.dshift, a.dshift_s, cols, n, groups);
    return nk_after_launch(ctx, "nk_norm_columns_finish_kernel");
}
template <class T, int W>
int backward_rows(nk_ctx* ctx, const NormGrad<T>& a, const NormPlan& p) {
    constexpr int E = norm_e<T>() / 2;
    const int64_t sms = ctx->prop.multiProcessorCount;
    // Few rows per CTA cost column sums that go to memory and back, few CTAs latency: one resident wave, at least four rows each where there are many
    const bool cols = a.dgain || a.dshift;
    auto units = [&](int64_t rows, int per_sm, int cluster) {
        int64_t u = sms * per_sm / cluster, most = (rows + 3) / 4 > sms / cluster ? (rows + 3) / 4 : sms / cluster;
        if (u > most) u = most;
        if (u > rows) u = rows;
        return u < 1 ? 1 : u;
    };
    int64_t groups;
    T* part = nullptr;
    NkWorkspace ws(ctx);
    int st;
    auto space = [&]() {
        if (!cols) return int(NK_OK);
        const int s = ws.get(size_t(groups) * 2 * p.n * sizeof(T));
        part = static_cast<T*>(ws.ptr);
        return s;
    };
#define NK_LANES(G, EL, PER)                                                                                                                                       \
    do {                                                                                                                                                           \
        groups = units((p.rows + 256 / G - 1) / (256 / G), PER, 1);                                                                                                \
        if ((st = space())) return st;                                                                                                                             \
        st = norm_launch(ctx, "nk_norm_grad_lanes_kernel", nk_norm_grad_lanes_kernel<T, W, G, EL>, groups, 256, 1, PER, a.out, a.err, a.src, a.gain, a.stats, part, p); \
    } while (0)
#define NK_CTA(TH, EL, C, PER)                                                                                                                                     \
    do {                                                                                                                                                           \
        groups = units(p.rows, PER, C);                                                                                                                            \
        if ((st = space())) return st;                                                                                                                             \
        st = norm_launch(ctx, "nk_norm_grad_kernel", nk_norm_grad_kernel<T, W, TH, EL>, groups, TH, C, PER, a.out, a.err, a.src, a.gain, a.stats, part, p);              \
    } while (0)
    if (p.n <= 32) NK_LANES(8, 4, 4);
    else if (p.n <= 64) NK_LANES(16, 4, 4);
    else if (p.n <= 128) NK_LANES(32, 4, 4);
    else if (p.n <= 256) NK_LANES(32, 8, 4);
    else if (p.n <= 1024) NK_CTA(128, 8, 1, 6);
    else if (p.n <= 2048) NK_CTA(256, 8, 1, 3);
    else if (p.n <= 256 * E) NK_CTA(256, E, 1, 2);
    else if (p.n <= 512 * E) NK_CTA(512, E, 1, 1);
    else if (p.n <= 1024 * E) NK_CTA(512, E, 2, 1);
    else if (p.n <= 2048 * E) NK_CTA(512, E, 4, 1);
    else NK_CTA(512, E, 8, 1);
#undef NK_LANES
#undef NK_CTA
    if (st || !cols) return st;
    return columns_finish(ctx, a, static_cast<const T*>(part), p.n, groups);
}

template <class T, int W>
int backward_stream(nk_ctx* ctx, const StreamShape& s, const NormGrad<T>& a, const NormPlan& p) {
    constexpr int E = stream_e<T>();
    const StreamCall c = stream_call(ctx, p, s);
    const bool cols = a.dgain || a.dshift;
    const int64_t groups = s.grid / s.cluster;
    NkWorkspace ws(ctx);
    int st;
    if (cols && (st = ws.get(size_t(groups) * 2 * p.n * sizeof(T)))) return st;
    T* part = static_cast<T*>(ws.ptr);
#define NK_TEAM(TW) case TW: st = stream_launch(ctx, "nk_norm_grad_stream_kernel", nk_norm_grad_stream_kernel<T, W, TW, E>, s, a.out, a.err, a.src, a.gain, a.stats, part, p, c); break
    switch (s.team) { NK_TEAM(1); NK_TEAM(2); NK_TEAM(4); NK_TEAM(8); default: NK_TEAM(16); }
#undef NK_TEAM
    if (st || !cols) return st;
    return columns_finish(ctx, a, static_cast<const T*>(part), p.n, groups);
}

template <class T, int W>
int backward_w(nk_ctx* ctx, const NormGrad<T>& a, const NormPlan& p) {
    StreamShape shape;
    if (stream_shape<T>(ctx, p, 2, W > 1, &shape)) return backward_stream<T, W>(ctx, shape, a, p);
    if (p.n <= 2048 * norm_e<T>()) return backward_rows<T, W>(ctx, a, p);
    constexpr int64_t L = int64_t(NORM_THREADS) * W * NORM_NV;
    const int64_t chunks = (p.n + L - 1) / L, blocks_c = (p.n + NORM_THREADS * W - 1) / (NORM_THREADS * W);
    const bool cols = a.dgain || a.dshift;
    // row groups: as many as fill the chip, at most one per row
    int64_t groups = (int64_t(ctx->prop.multiProcessorCount) * 8 + blocks_c - 1) / blocks_c;
    if (groups > p.rows) groups = p.rows;
    const int64_t per = (p.rows + groups - 1) / groups;
    groups = (p.rows + per - 1) / per;
    auto pad = [](size_t b) { return (b + 255) / 256 * 256; };
    const size_t part_bytes = pad(size_t(p.rows) * chunks * 2 * sizeof(T)), mean_bytes = pad(size_t(p.rows) * 2 * sizeof(T));
    const size_t col_bytes = cols ? size_t(groups) * 2 * p.n * sizeof(T) : 0;
    NkWorkspace ws(ctx);
    int st = ws.get(part_bytes + mean_bytes + col_bytes);
    if (st) return st;
    T *part = static_cast<T*>(ws.ptr), *means = reinterpret_cast<T*>(static_cast<char*>(ws.ptr) + part_bytes);
    T* col = cols ? reinterpret_cast<T*>(static_cast<char*>(ws.ptr) + part_bytes + mean_bytes) : nullptr;
    if (a.out) {
        nk_norm_chunk_sums_kernel<T, W><<<nk_grid_for(ctx, p.rows * chunks, 1, 32), NORM_THREADS, 0, ctx->stream>>>(a.err, a.src, a.gain, a.stats, part, p, chunks);
        if ((st = nk_after_launch(ctx, "nk_norm_chunk_sums_kernel"))) return st;
        nk_norm_row_means_kernel<T><<<nk_grid_for(ctx, p.rows, NORM_THREADS / 32, 8), NORM_THREADS, 0, ctx->stream>>>(part, means, p.rows, chunks, T(p.n));
        if ((st = nk_after_launch(ctx, "nk_norm_row_means_kernel"))) return st;
    }
    nk_norm_columns_kernel<T, W><<<nk_grid_for(ctx, blocks_c * groups, 1, 32), NORM_THREADS, 0, ctx->stream>>>(a.out, a.err, a.src, a.gain, a.stats, means, col, p, groups, per);
    if ((st = nk_after_launch(ctx, "nk_norm_columns_kernel")) || !cols) return st;
    return columns_finish(ctx, a, static_cast<const T*>(col), p.n, groups);
}
template <class T>
int backward(nk_ctx* ctx, const NormGrad<T>& a, const NormPlan& p) {
    if ((!a.out || norm_vec<T>(p, 0, a.out)) && norm_vec<T>(p, 1, a.src) && norm_vec<T>(p, 2, a.err)) return backward_w<T, norm_w<T>()>(ctx, a, p);
    return backward_w<T, 1>(ctx, a, p);
}

// a view of rank 1 with n elements, or NULL
int norm_vector(nk_ctx* ctx, const char* who, nk_buf* buf, const int32_t* cfg, int32_t dtype, int64_t n, bool drain, void** ptr, int64_t* stride) {
    *ptr = nullptr;
    *stride = 1;
    if (!buf) return NK_OK;
    NkView v;
    int st;
    if ((st = nk_view_parse(ctx, who, buf, cfg, 1, dtype, &v))) return st;
    if (drain && (st = nk_check_drain(ctx, who, v))) return st;
    if (v.size != n) return nk_fail(ctx, NK_ERR_BAD_ARG, "%s: %lld elements, rows have %lld", who, (long long)v.size, (long long)n);
    *ptr = static_cast<char*>(buf->ptr) + v.base * int64_t(nk_dtype_size(dtype));
    *stride = v.estride[0];
    return NK_OK;
}
int norm_stats(nk_ctx* ctx, const char* who, const nk_buf* stats, int32_t dtype, int64_t rows) {
    if (stats->magic != 0x4e4b4246) return nk_fail(ctx, NK_ERR_BAD_ARG, "%s: invalid handle of the statistics' buffer", who);
    if (stats->dtype != dtype || stats->device != ctx->device) return nk_fail(ctx, NK_ERR_BAD_ARG, "%s: the statistics' buffer is of another type or device", who);
    if (stats->n_elems / 2 < rows) return nk_fail(ctx, NK_ERR_BOUNDS, "%s: the statistics need 2 * %lld elements, the buffer holds %lld", who, (long long)rows, (long long)stats->n_elems);
    return NK_OK;
}
void norm_bounds(const nk_buf* buf, int t, int32_t dtype, NormPlan* p) {
    p->lo[t] = static_cast<const char*>(buf->ptr);
    p->hi[t] = p->lo[t] + buf->n_elems * int64_t(nk_dtype_size(dtype));
}
int norm_same_shape(nk_ctx* ctx, const char* who, const NkView& a, const NkView& b) {
    for (int k = 0; k < a.rank; k++)
        if (a.shape[k] != b.shape[k]) return nk_fail(ctx, NK_ERR_BAD_ARG, "%s: shapes differ at dim %d (%lld vs %lld)", who, k, (long long)a.shape[k], (long long)b.shape[k]);
    return NK_OK;
}

template <class T> T* at(nk_buf* b, const NkView& v) { return static_cast<T*>(b->ptr) + v.base; }

}  // namespace

extern "C" int nk_layer_norm(nk_ctx* ctx, int32_t dtype, int32_t rank, nk_buf* drn, const int32_t* cfg0, nk_buf* src, const int32_t* cfg1, nk_buf* gain,
                             const int32_t* cfg_gain, nk_buf* shift, const int32_t* cfg_shift, double eps, nk_buf* stats) {
    NK_CHECK_CTX(ctx);
    if (dtype != NK_F32 && dtype != NK_F64) return nk_fail(ctx, NK_ERR_UNSUPPORTED, "nk_layer_norm: dtype %d not supported (F32/F64 only)", dtype);
    if (!(eps >= 0.0)) return nk_fail(ctx, NK_ERR_BAD_ARG, "nk_layer_norm: eps %g is not >= 0", eps);
    NkView v0, v1;
    int st;
    if ((st = nk_view_parse(ctx, "nk_layer_norm(drain)", drn, cfg0, rank, dtype, &v0))) return st;
    if ((st = nk_check_drain(ctx, "nk_layer_norm", v0))) return st;
    if ((st = nk_view_parse(ctx, "nk_layer_norm(src)", src, cfg1, rank, dtype, &v1))) return st;
    if ((st = norm_same_shape(ctx, "nk_layer_norm", v0, v1))) return st;
    const NkView* views[3] = {&v0, &v1, nullptr};
    NormPlan p;
    norm_plan(views, &p);
    void *g, *s;
    if ((st = norm_vector(ctx, "nk_layer_norm(gain)", gain, cfg_gain, dtype, p.n, false, &g, &p.gain_s))) return st;
    if ((st = norm_vector(ctx, "nk_layer_norm(shift)", shift, cfg_shift, dtype, p.n, false, &s, &p.shift_s))) return st;
    if (stats && (st = norm_stats(ctx, "nk_layer_norm", stats, dtype, p.rows))) return st;
    norm_bounds(src, 0, dtype, &p);
    p.gain_v = p.gain_s == 1 && reinterpret_cast<uintptr_t>(g) % 16 == 0;
    p.shift_v = p.shift_s == 1 && reinterpret_cast<uintptr_t>(s) % 16 == 0;
    void* keep = stats ? stats->ptr : nullptr;
    if (dtype == NK_F32) return forward<float>(ctx, at<float>(drn, v0), at<float>(src, v1), (float*)g, (float*)s, (float*)keep, p, eps);
    return forward<double>(ctx, at<double>(drn, v0), at<double>(src, v1), (double*)g, (double*)s, (double*)keep, p, eps);
}

namespace {
template <class T>
int norm_grad(nk_ctx* ctx, nk_buf* dsrc, const NkView& v0, void* dgain, int64_t dgain_s, void* dshift, int64_t dshift_s, nk_buf* err, const NkView& v2, nk_buf* src,
              const NkView& v1, void* gain, nk_buf* stats, const NormPlan& p) {
    NormGrad<T> a;
    a.out = dsrc ? at<T>(dsrc, v0) : nullptr;
    a.dgain = static_cast<T*>(dgain); a.dgain_s = dgain_s;
    a.dshift = static_cast<T*>(dshift); a.dshift_s = dshift_s;
    a.err = at<T>(err, v2);
    a.src = at<T>(src, v1);
    a.gain = static_cast<const T*>(gain);
    a.stats = static_cast<const T*>(stats->ptr);
    return backward<T>(ctx, a, p);
}
}  // namespace

extern "C" int nk_layer_norm_grad(nk_ctx* ctx, int32_t dtype, int32_t rank, nk_buf* dsrc, const int32_t* cfg_dsrc, nk_buf* dgain, const int32_t* cfg_dgain,
                                  nk_buf* dshift, const int32_t* cfg_dshift, nk_buf* err, const int32_t* cfg_err, nk_buf* src, const int32_t* cfg1, nk_buf* gain,
                                  const int32_t* cfg_gain, nk_buf* stats) {
    NK_CHECK_CTX(ctx);
    if (dtype != NK_F32 && dtype != NK_F64) return nk_fail(ctx, NK_ERR_UNSUPPORTED, "nk_layer_norm_grad: dtype %d not supported (F32/F64 only)", dtype);
    if (!stats) return nk_fail(ctx, NK_ERR_BAD_ARG, "nk_layer_norm_grad: the forward call's statistics are needed");
    NkView v0, v1, v2;
    int st;
    if ((st = nk_view_parse(ctx, "nk_layer_norm_grad(err)", err, cfg_err, rank, dtype, &v2))) return st;
    if ((st = nk_view_parse(ctx, "nk_layer_norm_grad(src)", src, cfg1, rank, dtype, &v1))) return st;
    if ((st = norm_same_shape(ctx, "nk_layer_norm_grad", v2, v1))) return st;
    if (dsrc) {
        if ((st = nk_view_parse(ctx, "nk_layer_norm_grad(dsrc)", dsrc, cfg_dsrc, rank, dtype, &v0))) return st;
        if ((st = nk_check_drain(ctx, "nk_layer_norm_grad", v0))) return st;
        if ((st = norm_same_shape(ctx, "nk_layer_norm_grad", v0, v1))) return st;
    }
    const NkView* views[3] = {dsrc ? &v0 : nullptr, &v1, &v2};
    NormPlan p;
    norm_plan(views, &p);
    void *g, *dg, *ds;
    int64_t dgain_s, dshift_s;
    if ((st = norm_vector(ctx, "nk_layer_norm_grad(gain)", gain, cfg_gain, dtype, p.n, false, &g, &p.gain_s))) return st;
    if ((st = norm_vector(ctx, "nk_layer_norm_grad(dgain)", dgain, cfg_dgain, dtype, p.n, true, &dg, &dgain_s))) return st;
    if ((st = norm_vector(ctx, "nk_layer_norm_grad(dshift)", dshift, cfg_dshift, dtype, p.n, true, &ds, &dshift_s))) return st;
    if ((st = norm_stats(ctx, "nk_layer_norm_grad", stats, dtype, p.rows))) return st;
    if (!dsrc && !dg && !ds) return NK_OK;
    norm_bounds(src, 0, dtype, &p);
    norm_bounds(err, 1, dtype, &p);
    if (dtype == NK_F32) return norm_grad<float>(ctx, dsrc, v0, dg, dgain_s, ds, dshift_s, err, v2, src, v1, g, stats, p);
    return norm_grad<double>(ctx, dsrc, v0, dg, dgain_s, ds, dshift_s, err, v2, src, v1, g, stats, p);
}
