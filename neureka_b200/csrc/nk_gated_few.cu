// The gated block for few tokens (at most 8): the weights are read once from memory, which is what bounds these calls.
//
// nk_gated_few_kernel, forward and dx: a CTA takes 32 vectors of the result's columns and a slice of k; the CTAs of a cluster share the columns and
// split k, their sums meet through distributed shared memory and each finishes a part of the columns (f(g) * u there, in the one launch). The slice
// of x lies in shared memory. Two ways through the weights, by their contiguous direction:
//   columns: a lane owns a vector of columns, the warps split the slice's k; every weight in registers meets TOK broadcast values of x;
//   turned (k contiguous): a warp takes two columns at a time, its lanes run along k, and the lanes' sums are added by shuffles.
// nk_gated_outer_kernel, dW: a thread owns a vector of columns of dg and du for all tokens in registers and walks the rows of dW.
// Sums run over fixed partitions of k and are joined in order: the same bits every time.
#include <cooperative_groups.h>

#include "nk_gated.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int FEW_THREADS = 256, FEW_WARPS = FEW_THREADS / 32, FEW_MAX = 8, FEW_K = 512, FEW_SLICE = 128;   // k per chunk of a slice; a slice is a multiple of
template <class T, int W> struct FewVec { using type = T; };
template <> struct FewVec<float, 4> { using type = float4; };
template <> struct FewVec<double, 2> { using type = double2; };
template <class T> constexpr int few_v = 16 / int(sizeof(T));

struct FewCall {
    int fun;
    int tokens;
    int64_t N, K, slice;      // columns of the result, length of the sums, k per CTA (a multiple of FEW_SLICE)
    GatedMatrix x[2];         // [tokens, K]; SUM: dg and du
    GatedMatrix w[2];         // [K, N]
    GatedMatrix out;          // [tokens, N]
    void *gate, *up;          // forward: row-major [tokens, N] or null
};

// SUM: out = x_0 w_0 + x_1 w_1; otherwise out = f(x_0 w_0) * (x_0 w_1)
template <class T, int TOK, bool TURNED, bool VEC, bool SUM>
__global__ void __launch_bounds__(FEW_THREADS) nk_gated_few_kernel(const FewCall p) {
    constexpr int V = few_v<T>, COLS = 32 * V, NX = SUM ? 2 : 1, NB = SUM ? 1 : 2;
    using W = typename FewVec<T, V>::type;
    extern __shared__ __align__(16) unsigned char few_smem[];
    T* xs = reinterpret_cast<T*>(few_smem);                   // [NX][FEW_K][TOK], turned: [NX][TOK][FEW_K]
    T* sums = xs + NX * TOK * FEW_K;                          // [NB][TOK][COLS]
    cg::cluster_group cluster = cg::this_cluster();
    const int size = int(cluster.num_blocks()), rank = int(cluster.block_rank());
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t n0 = int64_t(blockIdx.x / unsigned(size)) * COLS;
    const int64_t k_begin = int64_t(rank) * p.slice, k_end = k_begin + p.slice < p.K ? k_begin + p.slice : p.K;
    const T *w0 = static_cast<const T*>(p.w[0].ptr), *w1 = static_cast<const T*>(p.w[1].ptr);
    T acc[NB][TOK][V];
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
        for (int t = 0; t < TOK; t++)
#pragma unroll
            for (int j = 0; j < V; j++) acc[b][t][j] = T(0);
    if (TURNED)
        for (int i = threadIdx.x; i < NB * TOK * COLS; i += FEW_THREADS) sums[i] = T(0);
    for (int64_t k0 = k_begin; k0 < k_end; k0 += FEW_K) {
        const int kc = int(k_end - k0 < FEW_K ? k_end - k0 : FEW_K);
        __syncthreads();
        for (int i = threadIdx.x; i < NX * TOK * FEW_K; i += FEW_THREADS) {   // zero past the slice and the tokens
            const int b = i / (TOK * FEW_K), r = i % (TOK * FEW_K), t = r / FEW_K, k = r % FEW_K;
            const GatedMatrix& x = p.x[b];
            xs[TURNED ? i : b * TOK * FEW_K + k * TOK + t] = k < kc && t < p.tokens ? static_cast<const T*>(x.ptr)[t * x.rs + (k0 + k) * x.cs] : T(0);
        }
        __syncthreads();
        if constexpr (!TURNED) {
            // F32 vectors of one token: 16 loads in flight (4096 x 8192: 47 us, with 8 60); without vectors they are 64 and cost registers (2048 x 5461: 34 us
            // against 25), F64 gains nothing
            constexpr int U = TOK == 1 && VEC && sizeof(T) == 4 ? 8 : 4;
            for (int k = warp * U; k < kc; k += FEW_WARPS * U) {
                T wv[U][2][V];
#pragma unroll
                for (int u = 0; u < U; u++)
#pragma unroll
                    for (int b = 0; b < 2; b++) {
                        const T* row = (b ? w1 : w0) + (k0 + k + u) * p.w[b].rs;
                        if (VEC) {
                            const int64_t n = n0 + lane * V;
                            if (k + u < kc && n < p.N) *reinterpret_cast<W*>(wv[u][b]) = __ldcs(reinterpret_cast<const W*>(row + n));
                            else {
#pragma unroll
                                for (int j = 0; j < V; j++) wv[u][b][j] = T(0);
                            }
                        } else {
#pragma unroll
                            for (int j = 0; j < V; j++) {
                                const int64_t n = n0 + lane + 32 * j;
                                wv[u][b][j] = k + u < kc && n < p.N ? row[n * p.w[b].cs] : T(0);
                            }
                        }
                    }
#pragma unroll
                for (int u = 0; u < U; u++)
#pragma unroll
                    for (int t = 0; t < TOK; t++)
#pragma unroll
                        for (int b = 0; b < 2; b++) {
                            // (k + u may pass the chunk, never the buffer: FEW_K is a multiple of the warps' share; it is zero there, like the weights)
                            const T x = xs[(SUM ? b : 0) * TOK * FEW_K + (k + u) * TOK + t];
#pragma unroll
                            for (int j = 0; j < V; j++) acc[SUM ? 0 : b][t][j] = fma(wv[u][b][j], x, acc[SUM ? 0 : b][t][j]);
                        }
            }
        } else {
            constexpr int R = 2, STEPS = FEW_K / (32 * V);
            for (int i = 0; i < COLS / FEW_WARPS; i += R) {
                const int c = warp * (COLS / FEW_WARPS) + i;
                if (n0 + c >= p.N) break;
                T wv[STEPS][R][2][V], s[R][NB][TOK];
#pragma unroll
                for (int q = 0; q < STEPS; q++)
#pragma unroll
                    for (int r = 0; r < R; r++)
#pragma unroll
                        for (int b = 0; b < 2; b++) {
                            const T* col = (b ? w1 : w0) + (n0 + c + r) * p.w[b].cs + k0;
                            const bool in = n0 + c + r < p.N;
                            const int k = (q * 32 + lane) * V;
                            if (VEC) {
                                if (in && k < kc) *reinterpret_cast<W*>(wv[q][r][b]) = __ldcs(reinterpret_cast<const W*>(col + k));
                                else {
#pragma unroll
                                    for (int j = 0; j < V; j++) wv[q][r][b][j] = T(0);
                                }
                            } else {
#pragma unroll
                                for (int j = 0; j < V; j++) {
                                    const int kj = (q * V + j) * 32 + lane;
                                    wv[q][r][b][j] = in && kj < kc ? col[kj] : T(0);
                                }
                            }
                        }
#pragma unroll
                for (int r = 0; r < R; r++)
#pragma unroll
                    for (int b = 0; b < NB; b++)
#pragma unroll
                        for (int t = 0; t < TOK; t++) s[r][b][t] = T(0);
#pragma unroll
                for (int q = 0; q < STEPS; q++)
#pragma unroll
                    for (int t = 0; t < TOK; t++)
#pragma unroll
                        for (int b = 0; b < 2; b++) {
                            T xv[V];
                            const T* x = xs + ((SUM ? b : 0) * TOK + t) * FEW_K;
                            if (VEC) *reinterpret_cast<W*>(xv) = *reinterpret_cast<const W*>(x + (q * 32 + lane) * V);
                            else {
#pragma unroll
                                for (int j = 0; j < V; j++) xv[j] = x[(q * V + j) * 32 + lane];
                            }
#pragma unroll
                            for (int r = 0; r < R; r++)
#pragma unroll
                                for (int j = 0; j < V; j++) s[r][SUM ? 0 : b][t] = fma(wv[q][r][b][j], xv[j], s[r][SUM ? 0 : b][t]);
                        }
#pragma unroll
                for (int r = 0; r < R; r++)
#pragma unroll
                    for (int b = 0; b < NB; b++)
#pragma unroll
                        for (int t = 0; t < TOK; t++) {
                            T v = s[r][b][t];
#pragma unroll
                            for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
                            if (lane == 0) sums[(b * TOK + t) * COLS + c + r] += v;
                        }
            }
        }
    }
    if (!TURNED) {   // the warps' sums, one warp after the other
        for (int q = 0; q < FEW_WARPS; q++) {
            __syncthreads();
            if (warp != q) continue;
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int t = 0; t < TOK; t++)
#pragma unroll
                    for (int j = 0; j < V; j++) {
                        T* at = sums + (b * TOK + t) * COLS + (VEC ? lane * V + j : lane + 32 * j);
                        *at = q ? *at + acc[b][t][j] : acc[b][t][j];
                    }
        }
    }
    cluster.sync();   // (a CTA alone: a barrier)
    for (int i = rank * FEW_THREADS + threadIdx.x; i < TOK * COLS; i += size * FEW_THREADS) {
        const int t = i / COLS;
        const int64_t n = n0 + i % COLS;
        if (t >= p.tokens || n >= p.N) continue;
        T v[NB];
#pragma unroll
        for (int b = 0; b < NB; b++) {
            v[b] = T(0);
            for (int r = 0; r < size; r++) v[b] += *cluster.map_shared_rank(sums + b * TOK * COLS + i, r);
        }
        T* o = static_cast<T*>(p.out.ptr) + t * p.out.rs + n * p.out.cs;
        if (SUM) *o = v[0];
        else {
            *o = gate_fun<T>(p.fun, false, v[0]) * v[NB - 1];
            if (p.gate) {
                static_cast<T*>(p.gate)[t * p.N + n] = v[0];
                static_cast<T*>(p.up)[t * p.N + n] = v[NB - 1];
            }
        }
    }
    if (size > 1) cluster.sync();   // nobody leaves while its sums may still be read
}

// dW_b[d, h] = sum over the tokens of x[t, d] e_b[t, h]; e_b row-major [tokens, H]
constexpr int OUTER_ROWS = 64;   // rows of dW per CTA
struct OuterCall {
    int tokens;
    int64_t D, H;
    GatedMatrix x, dw[2];
    const void* e[2];
};
template <class T, int TOK, bool VEC>
__global__ void __launch_bounds__(FEW_THREADS) nk_gated_outer_kernel(const OuterCall p, int64_t tiles_h) {
    constexpr int V = few_v<T>, COLS = 32 * V;
    using W = typename FewVec<T, V>::type;
    __shared__ T xs[OUTER_ROWS][TOK];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t h0 = (blockIdx.x % tiles_h) * COLS, d0 = (blockIdx.x / tiles_h) * OUTER_ROWS;
    for (int i = threadIdx.x; i < OUTER_ROWS * TOK; i += FEW_THREADS) {
        const int t = i / OUTER_ROWS, r = i % OUTER_ROWS;
        xs[r][t] = t < p.tokens && d0 + r < p.D ? static_cast<const T*>(p.x.ptr)[t * p.x.rs + (d0 + r) * p.x.cs] : T(0);
    }
    T e[2][TOK][V];
#pragma unroll
    for (int b = 0; b < 2; b++)
#pragma unroll
        for (int t = 0; t < TOK; t++)
#pragma unroll
            for (int j = 0; j < V; j++) {
                const int64_t h = h0 + (VEC ? lane * V + j : lane + 32 * j);
                e[b][t][j] = t < p.tokens && h < p.H ? static_cast<const T*>(p.e[b])[t * p.H + h] : T(0);
            }
    __syncthreads();
    for (int r = warp; r < OUTER_ROWS && d0 + r < p.D; r += FEW_WARPS) {
#pragma unroll
        for (int b = 0; b < 2; b++) {
            if (!p.dw[b].ptr) continue;
            T v[V];
#pragma unroll
            for (int j = 0; j < V; j++) v[j] = T(0);
#pragma unroll
            for (int t = 0; t < TOK; t++)
                if (t < p.tokens) {
#pragma unroll
                    for (int j = 0; j < V; j++) v[j] = fma(xs[r][t], e[b][t][j], v[j]);
                }
            T* row = static_cast<T*>(p.dw[b].ptr) + (d0 + r) * p.dw[b].rs;
            if (VEC) {
                if (h0 + lane * V < p.H) __stcs(reinterpret_cast<W*>(row + h0 + lane * V), *reinterpret_cast<W*>(v));
            } else {
#pragma unroll
                for (int j = 0; j < V; j++)
                    if (h0 + lane + 32 * j < p.H) row[(h0 + lane + 32 * j) * p.dw[b].cs] = v[j];
            }
        }
    }
}

template <class T>
bool few_aligned(const GatedMatrix& m, bool along_columns) {   // 16-byte accesses along the contiguous direction
    const int64_t fast = along_columns ? m.cs : m.rs, slow = along_columns ? m.rs : m.cs;
    return fast == 1 && slow % few_v<T> == 0 && reinterpret_cast<uintptr_t>(m.ptr) % 16 == 0;
}

template <class T, int TOK, bool TURNED, bool VEC, bool SUM>
int few_launch(nk_ctx* ctx, FewCall p) {
    constexpr int COLS = 32 * few_v<T>;
    constexpr size_t smem = sizeof(T) * TOK * ((SUM ? 2 : 1) * FEW_K + (SUM ? 1 : 2) * COLS);
    // k is split until there are at least three CTAs per SM (it doubles, so up to six), at most eight ways (a portable cluster)
    const int64_t tiles = (p.N + COLS - 1) / COLS, pieces = (p.K + FEW_SLICE - 1) / FEW_SLICE;
    int split = 1;
    while (split < 8 && split < pieces && tiles * split < int64_t(ctx->prop.multiProcessorCount) * 3) split *= 2;
    p.slice = (pieces + split - 1) / split * FEW_SLICE;
    if (tiles * split > 0x7fffffffLL) return nk_fail(ctx, NK_ERR_UNSUPPORTED, "nk_gated: a result of %lld columns is too large", (long long)p.N);
    auto* kern = nk_gated_few_kernel<T, TOK, TURNED, VEC, SUM>;
    if (smem > 48 * 1024) NK_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)));
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(unsigned(tiles * split));
    cfg.blockDim = dim3(FEW_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = unsigned(split);
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = split > 1 ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
    if (e != cudaSuccess) return nk_cuda_fail(ctx, e, "nk_gated_few_kernel");
    return nk_after_launch(ctx, "nk_gated_few_kernel");
}
template <class T, int TOK, bool SUM>
int few_route(nk_ctx* ctx, const FewCall& p) {
    const bool turned = p.w[0].rs == 1 && p.w[1].rs == 1 && p.w[0].cs != 1;
    if (turned) {
        // (the slices start at multiples of FEW_SLICE: only K itself and the weights decide whether vectors fit)
        if (p.K % few_v<T> == 0 && few_aligned<T>(p.w[0], false) && few_aligned<T>(p.w[1], false)) return few_launch<T, TOK, true, true, SUM>(ctx, p);
        return few_launch<T, TOK, true, false, SUM>(ctx, p);
    }
    if (p.N % few_v<T> == 0 && few_aligned<T>(p.w[0], true) && few_aligned<T>(p.w[1], true)) return few_launch<T, TOK, false, true, SUM>(ctx, p);
    return few_launch<T, TOK, false, false, SUM>(ctx, p);
}
template <class T, bool SUM>
int few_tokens(nk_ctx* ctx, const FewCall& p) {
    if (p.tokens == 1) return few_route<T, 1, SUM>(ctx, p);
    if (p.tokens <= 4) return few_route<T, 4, SUM>(ctx, p);
    return few_route<T, FEW_MAX, SUM>(ctx, p);
}
template <class T, int TOK>
int outer_launch(nk_ctx* ctx, const OuterCall& p) {
    constexpr int COLS = 32 * few_v<T>;
    const int64_t tiles_h = (p.H + COLS - 1) / COLS, grid = tiles_h * ((p.D + OUTER_ROWS - 1) / OUTER_ROWS);
    if (grid > 0x7fffffffLL) return nk_fail(ctx, NK_ERR_UNSUPPORTED, "nk_gated_grad: weights of %lld x %lld elements are too large", (long long)p.D, (long long)p.H);
    bool vec = p.H % few_v<T> == 0;
    for (int b = 0; b < 2; b++) vec = vec && (!p.dw[b].ptr || few_aligned<T>(p.dw[b], true));
    if (vec) nk_gated_outer_kernel<T, TOK, true><<<unsigned(grid), FEW_THREADS, 0, ctx->stream>>>(p, tiles_h);
    else nk_gated_outer_kernel<T, TOK, false><<<unsigned(grid), FEW_THREADS, 0, ctx->stream>>>(p, tiles_h);
    return nk_after_launch(ctx, "nk_gated_outer_kernel");
}

}  // namespace

int64_t nk_gated_few_most() { return FEW_MAX; }

template <class T>
int nk_gated_few_forward(nk_ctx* ctx, const GatedCall& c) {
    FewCall p;
    memset(&p, 0, sizeof(p));
    p.fun = c.fun;
    p.tokens = int(c.T);
    p.N = c.H;
    p.K = c.D;
    p.x[0] = c.x;
    p.w[0] = c.w[0];
    p.w[1] = c.w[1];
    p.out = c.y;
    p.gate = c.gate;
    p.up = c.up;
    return few_tokens<T, false>(ctx, p);
}
template <class T>
int nk_gated_few_dx(nk_ctx* ctx, const GatedCall& c, const T* dg, const T* du) {
    FewCall p;
    memset(&p, 0, sizeof(p));
    p.tokens = int(c.T);
    p.N = c.D;
    p.K = c.H;
    p.x[0] = GatedMatrix{const_cast<T*>(dg), c.H, 1};
    p.x[1] = GatedMatrix{const_cast<T*>(du), c.H, 1};
    for (int b = 0; b < 2; b++) p.w[b] = GatedMatrix{c.w[b].ptr, c.w[b].cs, c.w[b].rs};
    p.out = c.dx;
    return few_tokens<T, true>(ctx, p);
}
template <class T>
int nk_gated_few_dw(nk_ctx* ctx, const GatedCall& c, const T* dg, const T* du) {
    OuterCall o;
    memset(&o, 0, sizeof(o));
    o.tokens = int(c.T);
    o.D = c.D;
    o.H = c.H;
    o.x = c.x;
    o.e[0] = dg;
    o.e[1] = du;
    for (int b = 0; b < 2; b++) o.dw[b] = c.dw[b];
    if (c.T == 1) return outer_launch<T, 1>(ctx, o);
    if (c.T <= 4) return outer_launch<T, 4>(ctx, o);
    return outer_launch<T, FEW_MAX>(ctx, o);
}
template int nk_gated_few_forward<float>(nk_ctx*, const GatedCall&);
template int nk_gated_few_forward<double>(nk_ctx*, const GatedCall&);
template int nk_gated_few_dx<float>(nk_ctx*, const GatedCall&, const float*, const float*);
template int nk_gated_few_dx<double>(nk_ctx*, const GatedCall&, const double*, const double*);
template int nk_gated_few_dw<float>(nk_ctx*, const GatedCall&, const float*, const float*);
template int nk_gated_few_dw<double>(nk_ctx*, const GatedCall&, const double*, const double*);
