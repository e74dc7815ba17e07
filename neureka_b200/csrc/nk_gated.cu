// The gated feed-forward block (no counterpart in the reference):
//   g = x Wg, u = x Wu, y = f(g) * u;   dg = e * u * f'(g), du = e * f(g), dx = dg Wg^T + du Wu^T, dWg = x^T dg, dWu = x^T du.
//
// Which kernels take a call:
//   F32  1 token, or a matrix with a side below 16 and at most 8 tokens: nk_gated_few.cu; 2 to 192 tokens: nk_gated_narrow.cu; more, of at least 64 x 64
//        weights and 2^20 multiply-adds: nk_gated_tc.cu; the rest: nk_gated_tile_kernel. dW is a sum over the tokens: at most 8 nk_gated_few.cu, up to 64
//        and 2^26 multiply-adds nk_gated_tile_kernel, else nk_gated_tc.cu;
//   F64  at most 8 tokens: nk_gated_few.cu; more: nk_gated_dmma_kernel.
// Both kernels below take any sizes and any strides; both products of a tile share the panel of x and end in the same thread, so the
// activation and the product with it need no further pass.
#include <cooperative_groups.h>

#include "nk_gated.cuh"
#include "nk_ptx.cuh"

namespace cg = cooperative_groups;

namespace {

// ---- the tile kernel -------------------------------------------------------------------------------------------------------------
// For what is too small for the tensor cores, or too narrow: bound by latency (200 x 128 x 256 forward would be 20 us, on the tensor cores 16).
// One running sum of K terms of one sign is 2e-8 sqrt(K) off (standard deviation; 2e-5 for a million terms, more than a product of the framework may be),
// and where the tiles are few and the sums long (dW of a narrow block: all tokens) the chip is idle. So k is split over the CTAs, and a second
// launch adds the parts in order: backward pass of 65536 x 32 x 32 7350 -> 119 us.
// FORWARD: C_i = A_0 B_i, out_0 = f(C_0) * C_1 (C_i kept where wanted).  TWO: out_i = A_0 B_i.  SUM: out_0 = A_0 B_0 + A_1 B_1.
enum { GATED_FORWARD, GATED_TWO, GATED_SUM };
struct GatedTile {
    int fun;
    int64_t M, N, K;
    GatedMatrix a[2], b[2], out[2];   // [M, K], [K, N], [M, N]
    void *gate, *up;                  // FORWARD: row-major [M, N] or null
    int splits;                       // parts that k is cut into; above 1 they go to
    void* parts;                      // [part][product][M][N]
};
constexpr int GT = 64, GK = 16;       // 64 x 64 of out, panels of 16 k; 256 threads with 4 x 4 elements of each product
constexpr int GT_LEAST = 32, GT_MOST = 256;   // panels of a part: at least so many that its way through memory costs little, at most 4096 terms

// element (m, n) of what is asked for, from its product or products
template <class T, int MODE>
__device__ __forceinline__ void gated_tile_store(const GatedTile& p, int64_t m, int64_t n, T v0, T v1) {
    if (MODE == GATED_FORWARD) {
        if (p.gate) {
            static_cast<T*>(p.gate)[m * p.N + n] = v0;
            static_cast<T*>(p.up)[m * p.N + n] = v1;
        }
        static_cast<T*>(p.out[0].ptr)[m * p.out[0].rs + n * p.out[0].cs] = gate_fun<T>(p.fun, false, v0) * v1;
    } else {
        if (p.out[0].ptr) static_cast<T*>(p.out[0].ptr)[m * p.out[0].rs + n * p.out[0].cs] = v0;
        if (MODE == GATED_TWO && p.out[1].ptr) static_cast<T*>(p.out[1].ptr)[m * p.out[1].rs + n * p.out[1].cs] = v1;
    }
}

// SPLIT: a part of k per CTA (a form of its own: the split's arithmetic makes whole sums an eighth slower)
template <class T, int MODE, bool SPLIT>
__global__ void __launch_bounds__(256) nk_gated_tile_kernel(const GatedTile p) {
    constexpr int NB = MODE == GATED_SUM ? 1 : 2, PHASES = MODE == GATED_SUM ? 2 : 1;
    __shared__ T As[GK][GT + 1], Bs[NB][GK][GT + 1];
    const int64_t tiles_n = (p.N + GT - 1) / GT, tile = SPLIT ? blockIdx.x / unsigned(p.splits) : blockIdx.x, part = SPLIT ? blockIdx.x % unsigned(p.splits) : 0;
    const int64_t m0 = (tile / tiles_n) * GT, n0 = (tile % tiles_n) * GT;
    int64_t first = 0, last = 0;   // this CTA's share of the panels of 16 k, of both phases of a SUM one after the other
    const int64_t phase_panels = SPLIT ? (p.K + GK - 1) / GK : 0;
    if (SPLIT) {
        first = part * (phase_panels * PHASES) / p.splits;
        last = (part + 1) * (phase_panels * PHASES) / p.splits;
    }
    const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
    T acc[NB][4][4];
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) acc[b][i][j] = T(0);
    for (int phase = 0; phase < PHASES; phase++) {
        const GatedMatrix& A = p.a[phase];
        const int64_t k_begin = SPLIT && first > phase * phase_panels ? (first - phase * phase_panels) * GK : 0;
        const int64_t k_end = SPLIT && last - phase * phase_panels < phase_panels ? (last - phase * phase_panels) * GK : p.K;
        for (int64_t k0 = k_begin; k0 < k_end; k0 += GK) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 4; i++) {   // lanes along the contiguous direction
                const int e = tid + i * 256, k = A.cs == 1 ? e & 15 : e >> 6, r = A.cs == 1 ? e >> 4 : e & 63;
                As[k][r] = m0 + r < p.M && k0 + k < p.K ? static_cast<const T*>(A.ptr)[(m0 + r) * A.rs + (k0 + k) * A.cs] : T(0);
            }
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const GatedMatrix& B = p.b[MODE == GATED_SUM ? phase : b];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int e = tid + i * 256, k = B.rs == 1 ? e & 15 : e >> 6, c = B.rs == 1 ? e >> 4 : e & 63;
                    Bs[b][k][c] = n0 + c < p.N && k0 + k < p.K ? static_cast<const T*>(B.ptr)[(k0 + k) * B.rs + (n0 + c) * B.cs] : T(0);
                }
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < GK; k++) {
                T a[4];
#pragma unroll
                for (int i = 0; i < 4; i++) a[i] = As[k][ty + 16 * i];
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const T v = Bs[b][k][tx + 16 * j];
#pragma unroll
                        for (int i = 0; i < 4; i++) acc[b][i][j] = fma(a[i], v, acc[b][i][j]);
                    }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int64_t m = m0 + ty + 16 * i;
        if (m >= p.M) continue;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int64_t n = n0 + tx + 16 * j;
            if (n >= p.N) continue;
            if (SPLIT) {
#pragma unroll
                for (int b = 0; b < NB; b++) static_cast<T*>(p.parts)[((part * NB + b) * p.M + m) * p.N + n] = acc[b][i][j];
            } else gated_tile_store<T, MODE>(p, m, n, acc[0][i][j], acc[NB - 1][i][j]);
        }
    }
}
// The parts of split sums, in a fixed order: 32 elements per CTA, warp w takes the parts w, w + 8, ...
template <class T, int MODE>
__global__ void __launch_bounds__(256) nk_gated_join_kernel(const GatedTile p) {
    constexpr int NB = MODE == GATED_SUM ? 1 : 2;
    __shared__ T sums[NB][8][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t size = p.M * p.N, e = int64_t(blockIdx.x) * 32 + lane;
    T v[NB];
#pragma unroll
    for (int b = 0; b < NB; b++) v[b] = T(0);
    if (e < size) {
#pragma unroll 4
        for (int s = warp; s < p.splits; s += 8)
#pragma unroll
            for (int b = 0; b < NB; b++) v[b] += static_cast<const T*>(p.parts)[(int64_t(s) * NB + b) * size + e];
    }
#pragma unroll
    for (int b = 0; b < NB; b++) sums[b][warp][lane] = v[b];
    __syncthreads();
    if (warp || e >= size) return;
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
        for (int w = 1; w < 8; w++) v[b] += sums[b][w][lane];
    gated_tile_store<T, MODE>(p, e / p.N, e % p.N, v[0], v[NB - 1]);
}
// ---- F64 on the FP64 matrix instructions -----------------------------------------------------------------------------------------
// mma.m8n8k4, 64 x 64 tiles of four warps with 32 x 32 each (nk_conv_gemm.cu: why). With two B operands the tile is 32 columns of each product and
// the blocks of eight columns alternate between the two, so that a thread holds both products of an element. k is split over the CTAs of a
// cluster where the tiles are few; the tile passes through shared memory at the end, where the cluster's parts meet in rank order.
// Panels are copied asynchronously, element by element (any strides), two ahead (held in registers between load and store, one ahead: 1000 x 1000 x
// 1000 forward 230 us against 217). Bound by the FP64 matrix instructions: 2000 x 1000 x 1000 forward 316 us (25 TFLOP/s; products of 2048^3
// reach 27), 300 x 512 x 1365 44 us, where the last wave and the first panels weigh more. 16 x 8 x 8 instructions take as long as 8 x 8 x 4 ones.
constexpr int GD_T = 64, GD_K = 16, GD_PITCH = 20;   // a panel's rows have a pitch of 20 doubles: the fragment loads of a half warp fall on 16 banks
constexpr int GD_RING = 3, GD_SMEM = GD_RING * 2 * GD_T * GD_PITCH * int(sizeof(double));
__device__ __forceinline__ void gd_mma(double (&c)[2], double a, double b) {
    asm volatile("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0, %1}, {%2}, {%3}, {%0, %1};" : "+d"(c[0]), "+d"(c[1]) : "d"(a), "d"(b));
}
template <int MODE>
__global__ void __launch_bounds__(128, 3) nk_gated_dmma_kernel(const GatedTile p) {
    constexpr int COLS = MODE == GATED_SUM ? GD_T : GD_T / 2;   // columns of an output that a tile covers
    extern __shared__ __align__(16) unsigned char gd_smem[];    // [buffer][A, B][row][k]; then the tile, [row][column]
    double* smem = reinterpret_cast<double*>(gd_smem);
    auto As = reinterpret_cast<double (*)[2][GD_T][GD_PITCH]>(smem);
    cg::cluster_group cluster = cg::this_cluster();
    const int size = int(cluster.num_blocks()), rank = int(cluster.block_rank());
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int64_t tiles_n = (p.N + COLS - 1) / COLS, t = blockIdx.x / unsigned(size);
    const int64_t m0 = (t / tiles_n) * GD_T, n0 = (t % tiles_n) * COLS;
    // panels of 16 k, of both phases of a SUM one after the other; this CTA's share of them
    const int64_t phase_panels = (p.K + GD_K - 1) / GD_K, panels = phase_panels * (MODE == GATED_SUM ? 2 : 1);
    const int64_t first = rank * panels / size, last = (rank + 1) * panels / size;
    // Element i of a thread's share of a panel, the operand's contiguous direction across the threads: k = tid % 16 and rows tid / 16 + 8 i where k is,
    // otherwise row tid % 64 and k = tid / 64 + 2 i. An element's address is one base per thread plus a constant step, moved on by a
    // panel at a time (worked out per element, the integer chains took longer than the products).
    struct Walk {
        const double* at;
        int64_t step, panel;
        unsigned rows;   // bit i: element i's row exists
    };
    bool a_kfast = false, b_kfast = false;
    Walk wa, wb[2];      // two B operands, k contiguous: the even elements' and the odd ones'
    auto walk = [&](const GatedMatrix& m, int64_t rs, int64_t ks, bool kfast, int64_t row0, int64_t rows, int stride, int n, int64_t k0) {
        Walk w;
        const int r = kfast ? tid >> 4 : tid & 63, k = kfast ? tid & 15 : tid >> 6;
        w.at = static_cast<const double*>(m.ptr) + (row0 + r) * rs + (k0 + k) * ks;
        w.step = kfast ? stride * rs : 2 * ks;
        w.panel = GD_K * ks;
        w.rows = 0;
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < n && row0 + r + (kfast ? stride * i : 0) < rows) w.rows |= 1u << i;
        return w;
    };
    auto start = [&](int phase, int64_t k0) {
        const GatedMatrix& A = p.a[phase];
        a_kfast = A.cs == 1;
        wa = walk(A, A.rs, A.cs, a_kfast, m0, p.M, 8, 8, k0);
        b_kfast = p.b[phase].rs == 1;
        if (MODE == GATED_SUM) {
            wb[0] = walk(p.b[phase], p.b[phase].cs, p.b[phase].rs, b_kfast, n0, p.N, 8, 8, k0);
        } else if (b_kfast) {   // rows tid / 16 + 8 i of the panel: column tid / 16 + 8 (i / 2) of operand i % 2
#pragma unroll
            for (int w = 0; w < 2; w++) wb[w] = walk(p.b[w], p.b[w].cs, p.b[w].rs, true, n0, p.N, 8, 4, k0);
        } else {                // row tid % 64: column 8 (row / 16) + row % 8 of operand (row / 8) % 2
            const int r = tid & 63;
            const GatedMatrix& B = p.b[(r >> 3) & 1];
            wb[0] = walk(B, B.cs, B.rs, false, n0 + (r >> 4) * 8 + (r & 7) - r, p.N, 8, 8, k0);
        }
    };
    const double *any_a = static_cast<const double*>(p.a[0].ptr), *any_b = static_cast<const double*>(p.b[0].ptr);   // (not read where there is no element: zeros)
    auto fetch = [&](int64_t panel, int buf) {
        const int phase = MODE == GATED_SUM && panel >= phase_panels;
        const int64_t k0 = (panel - phase * phase_panels) * GD_K;
        if (panel == first || (MODE == GATED_SUM && panel == phase_panels)) start(phase, k0);
        const int left = p.K - k0 < GD_K ? int(p.K - k0) : GD_K, ak = a_kfast ? tid & 15 : tid >> 6, bk = b_kfast ? tid & 15 : tid >> 6;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const bool in = ((wa.rows >> i) & 1u) && ak + (a_kfast ? 0 : 2 * i) < left;
            nk_cp_async_8(&As[buf][0][a_kfast ? (tid >> 4) + 8 * i : tid & 63][a_kfast ? tid & 15 : (tid >> 6) + 2 * i], in ? wa.at + i * wa.step : any_a, in ? 8 : 0);
        }
        wa.at += wa.panel;
        if (MODE != GATED_SUM && b_kfast) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const Walk& w = wb[i & 1];
                const bool in = ((w.rows >> (i >> 1)) & 1u) && bk < left;
                nk_cp_async_8(&As[buf][1][(tid >> 4) + 8 * i][tid & 15], in ? w.at + (i >> 1) * w.step : any_b, in ? 8 : 0);
            }
            wb[1].at += wb[1].panel;
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const bool in = ((wb[0].rows >> i) & 1u) && bk + (b_kfast ? 0 : 2 * i) < left;
                nk_cp_async_8(&As[buf][1][b_kfast ? (tid >> 4) + 8 * i : tid & 63][b_kfast ? tid & 15 : (tid >> 6) + 2 * i], in ? wb[0].at + i * wb[0].step : any_b, in ? 8 : 0);
            }
        }
        wb[0].at += wb[0].panel;
    };
    double acc[4][4][2];
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j][0] = acc[i][j][1] = 0.0;
    const int wm = (warp >> 1) * 32, wn = (warp & 1) * 32, fr = lane >> 2, fk = lane & 3;
#pragma unroll
    for (int q = 0; q < GD_RING - 1; q++) {
        if (first + q < last) fetch(first + q, q);
        nk_cp_async_commit();
    }
    int buf = 0;
    for (int64_t panel = first; panel < last; panel++) {
        nk_cp_async_wait<GD_RING - 2>();
        __syncthreads();   // the panel has landed for everyone, and everyone has read the one whose buffer is filled next
        if (panel + GD_RING - 1 < last) fetch(panel + GD_RING - 1, (buf + GD_RING - 1) % GD_RING);
        nk_cp_async_commit();
#pragma unroll
        for (int k = 0; k < GD_K; k += 4) {
            double a[4], b[4];
#pragma unroll
            for (int i = 0; i < 4; i++) a[i] = As[buf][0][wm + 8 * i + fr][k + fk];
#pragma unroll
            for (int j = 0; j < 4; j++) b[j] = As[buf][1][wn + 8 * j + fr][k + fk];
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) gd_mma(acc[i][j], a[i], b[j]);
        }
        buf = buf + 1 == GD_RING ? 0 : buf + 1;
    }
    nk_cp_async_wait<0>();
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) *reinterpret_cast<double2*>(smem + (wm + 8 * i + fr) * GD_T + wn + 8 * j + 2 * fk) = make_double2(acc[i][j][0], acc[i][j][1]);
    cluster.sync();   // (a CTA alone: a barrier)
    for (int e = rank * 128 + tid; e < GD_T * COLS; e += size * 128) {
        const int r = e / COLS, c = e % COLS;
        const int64_t m = m0 + r, n = n0 + c;
        if (m >= p.M || n >= p.N) continue;
        const int at = r * GD_T + (MODE == GATED_SUM ? c : (c >> 3) * 16 + (c & 7));
        double v[2] = {0.0, 0.0};
        for (int q = 0; q < size; q++) {
            const double* theirs = cluster.map_shared_rank(smem, q);
            v[0] += theirs[at];
            if (MODE != GATED_SUM) v[1] += theirs[at + 8];
        }
        if (MODE == GATED_FORWARD) {
            if (p.gate) {
                static_cast<double*>(p.gate)[m * p.N + n] = v[0];
                static_cast<double*>(p.up)[m * p.N + n] = v[1];
            }
            static_cast<double*>(p.out[0].ptr)[m * p.out[0].rs + n * p.out[0].cs] = gate_fun<double>(p.fun, false, v[0]) * v[1];
        } else {
#pragma unroll
            for (int b = 0; b < (MODE == GATED_SUM ? 1 : 2); b++)
                if (p.out[b].ptr) static_cast<double*>(p.out[b].ptr)[m * p.out[b].rs + n * p.out[b].cs] = v[b];
        }
    }
    if (size > 1) cluster.sync();   // nobody leaves while its part may still be read
}
template <int MODE>
int launch_dmma(nk_ctx* ctx, const GatedTile& p) {
    constexpr int COLS = MODE == GATED_SUM ? GD_T : GD_T / 2;
    const int64_t tiles = ((p.M + GD_T - 1) / GD_T) * ((p.N + COLS - 1) / COLS), panels = (p.K + GD_K - 1) / GD_K * (MODE == GATED_SUM ? 2 : 1);
    // k is split, in parts of at least 64, where that evens out the SMs' shares. Three CTAs fit an SM and share its FP64 units, one by itself leaves half of
    // them idle, and a part costs about two panels of its own. 1000 x 1000 x 1000 forward, 512 tiles: whole 217 us, in four parts 185.
    const int64_t sms = ctx->prop.multiProcessorCount;
    int split = 1;
    int64_t best = 0;
    for (int s = 1; s <= 8 && (s == 1 || panels / s >= 4) && tiles < (int64_t(1) << 28); s *= 2) {
        const int64_t per_sm = (tiles * s + sms - 1) / sms, cost = (per_sm + (per_sm % 3 == 1)) * (panels / s + 2);
        if (s == 1 || cost < best) { split = s; best = cost; }
    }
    if (tiles * split > 0x7fffffffLL) return nk_fail(ctx, NK_ERR_UNSUPPORTED, "nk_gated: a result of %lld x %lld elements is too large", (long long)p.M, (long long)p.N);
    NK_CUDA(ctx, cudaFuncSetAttribute(nk_gated_dmma_kernel<MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, GD_SMEM));
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(unsigned(tiles * split));
    cfg.blockDim = dim3(128);
    cfg.dynamicSmemBytes = GD_SMEM;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = unsigned(split);
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = split > 1 ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, nk_gated_dmma_kernel<MODE>, p);
    if (e != cudaSuccess) return nk_cuda_fail(ctx, e, "nk_gated_dmma_kernel");
    return nk_after_launch(ctx, "nk_gated_dmma_kernel");
}

template <class T, int MODE>
int launch_tiles(nk_ctx* ctx, GatedTile p) {
    if constexpr (sizeof(T) == 8) return launch_dmma<MODE>(ctx, p);
    else {
        const int64_t tiles = ((p.M + GT - 1) / GT) * ((p.N + GT - 1) / GT), panels = (p.K + GK - 1) / GK * (MODE == GATED_SUM ? 2 : 1);
        if (tiles > 0x7fffffffLL) return nk_fail(ctx, NK_ERR_UNSUPPORTED, "nk_gated: a result of %lld x %lld elements is too large", (long long)p.M, (long long)p.N);
        int64_t splits = int64_t(ctx->prop.multiProcessorCount) * 2 / tiles;   // what fits the chip, two CTAs per SM
        if (splits > panels / GT_LEAST) splits = panels / GT_LEAST;
        if (splits < (panels + GT_MOST - 1) / GT_MOST) splits = (panels + GT_MOST - 1) / GT_MOST;
        if (tiles * splits > 0x7fffffffLL) return nk_fail(ctx, NK_ERR_UNSUPPORTED, "nk_gated: sums of %lld terms are too long", (long long)p.K);
        p.splits = int(splits);
        NkWorkspace ws(ctx);
        int st;
        if (p.splits > 1 && (st = ws.get(size_t(p.splits) * (MODE == GATED_SUM ? 1 : 2) * p.M * p.N * sizeof(T)))) return st;
        p.parts = ws.ptr;
        if (p.splits == 1) {
            nk_gated_tile_kernel<T, MODE, false><<<unsigned(tiles), 256, 0, ctx->stream>>>(p);
            return nk_after_launch(ctx, "nk_gated_tile_kernel");
        }
        nk_gated_tile_kernel<T, MODE, true><<<unsigned(tiles * p.splits), 256, 0, ctx->stream>>>(p);
        if ((st = nk_after_launch(ctx, "nk_gated_tile_kernel"))) return st;
        nk_gated_join_kernel<T, MODE><<<unsigned((p.M * p.N + 31) / 32), 256, 0, ctx->stream>>>(p);
        return nk_after_launch(ctx, "nk_gated_join_kernel");
    }
}

// dg and du, row-major [T, H]
template <class T>
__global__ void __launch_bounds__(256) nk_gated_errors_kernel(const GatedCall p, T* __restrict__ dg, T* __restrict__ du) {
    const int64_t total = p.T * p.H;
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < total; i += int64_t(gridDim.x) * 256) {
        const int64_t t = i / p.H, h = i - t * p.H;
        const T e = static_cast<const T*>(p.err.ptr)[t * p.err.rs + h * p.err.cs], g = static_cast<const T*>(p.gate)[i], u = static_cast<const T*>(p.up)[i];
        dg[i] = e * u * gate_fun<T>(p.fun, true, g);
        du[i] = e * gate_fun<T>(p.fun, false, g);
    }
}

GatedMatrix turned(const GatedMatrix& m) { return GatedMatrix{m.ptr, m.cs, m.rs}; }

template <class T>
int forward(nk_ctx* ctx, const GatedCall& c) {
    if constexpr (sizeof(T) == 4) {
        if (c.T > 1 && nk_gated_narrow(ctx, c)) return nk_gated_narrow_forward(ctx, c);
        bool handled = false;
        const int st = nk_gated_tc_forward(ctx, c, &handled);
        if (st || handled) return st;
    }
    if (c.T <= nk_gated_few_most()) return nk_gated_few_forward<T>(ctx, c);
    GatedTile p;
    memset(&p, 0, sizeof(p));
    p.fun = c.fun;
    p.M = c.T; p.N = c.H; p.K = c.D;
    p.a[0] = c.x;
    p.b[0] = c.w[0]; p.b[1] = c.w[1];
    p.out[0] = c.y;
    p.gate = c.gate; p.up = c.up;
    return launch_tiles<T, GATED_FORWARD>(ctx, p);
}
template <class T>
int backward(nk_ctx* ctx, const GatedCall& c) {
    if (sizeof(T) == 4) {
        bool handled = false;
        const int st = nk_gated_tc_backward(ctx, c, &handled);
        if (st || handled) return st;
    }
    NkWorkspace ws(ctx);
    int st = ws.get(size_t(c.T) * c.H * 2 * sizeof(T));
    if (st) return st;
    T *dg = static_cast<T*>(ws.ptr), *du = dg + c.T * c.H;
    nk_gated_errors_kernel<T><<<nk_grid_for(ctx, c.T * c.H, 256, 8), 256, 0, ctx->stream>>>(c, dg, du);
    if ((st = nk_after_launch(ctx, "nk_gated_errors_kernel"))) return st;
    if (c.T <= nk_gated_few_most()) {
        if (c.dx.ptr) {
            if constexpr (sizeof(T) == 4) st = c.T > 1 && nk_gated_narrow(ctx, c) ? nk_gated_narrow_dx(ctx, c, dg, du) : nk_gated_few_dx<T>(ctx, c, dg, du);
            else st = nk_gated_few_dx<T>(ctx, c, dg, du);
            if (st) return st;
        }
        return c.dw[0].ptr || c.dw[1].ptr ? nk_gated_few_dw<T>(ctx, c, dg, du) : int(NK_OK);
    }
    const GatedMatrix mg{dg, c.H, 1}, mu{du, c.H, 1};
    GatedTile p;
    memset(&p, 0, sizeof(p));
    bool narrow = false;
    if constexpr (sizeof(T) == 4) {
        narrow = c.dx.ptr && nk_gated_narrow(ctx, c);
        if (narrow && (st = nk_gated_narrow_dx(ctx, c, dg, du))) return st;
    }
    if (c.dx.ptr && !narrow) {
        p.M = c.T; p.N = c.D; p.K = c.H;
        p.a[0] = mg; p.a[1] = mu;
        p.b[0] = turned(c.w[0]); p.b[1] = turned(c.w[1]);
        p.out[0] = c.dx;
        if ((st = launch_tiles<T, GATED_SUM>(ctx, p))) return st;
    }
    if (!c.dw[0].ptr && !c.dw[1].ptr) return NK_OK;
    p.M = c.D; p.N = c.H; p.K = c.T;
    p.a[0] = turned(c.x);
    p.b[0] = mg; p.b[1] = mu;
    p.out[0] = c.dw[0]; p.out[1] = c.dw[1];
    return launch_tiles<T, GATED_TWO>(ctx, p);
}

// One of a call's matrices: a view of rank 2, T / D / H filled in or compared.
int gated_matrix(nk_ctx* ctx, const char* who, const char* what, nk_buf* buf, const int32_t* cfg, int32_t dtype, bool drain, int64_t* rows, int64_t* cols, GatedMatrix* out) {
    NkView v;
    int st;
    if ((st = nk_view_parse(ctx, who, buf, cfg, 2, dtype, &v))) return st;
    if (drain && (st = nk_check_drain(ctx, who, v))) return st;
    if (*rows == 0) *rows = v.shape[0];
    if (*cols == 0) *cols = v.shape[1];
    if (v.shape[0] != *rows || v.shape[1] != *cols)
        return nk_fail(ctx, NK_ERR_BAD_ARG, "%s: %s is [%lld, %lld], expected [%lld, %lld]", who, what, (long long)v.shape[0], (long long)v.shape[1], (long long)*rows, (long long)*cols);
    out->ptr = static_cast<char*>(buf->ptr) + v.base * int64_t(nk_dtype_size(dtype));
    out->rs = v.estride[0];
    out->cs = v.estride[1];
    return NK_OK;
}
int gated_kept(nk_ctx* ctx, const char* who, nk_buf* kept, int32_t dtype, GatedCall* c) {
    if (kept->magic != 0x4e4b4246) return nk_fail(ctx, NK_ERR_BAD_ARG, "%s: invalid handle of the kept products' buffer", who);
    if (kept->dtype != dtype || kept->device != ctx->device) return nk_fail(ctx, NK_ERR_BAD_ARG, "%s: the kept products' buffer is of another type or device", who);
    if (kept->n_elems / 2 / c->H < c->T)
        return nk_fail(ctx, NK_ERR_BOUNDS, "%s: the kept products need 2 * %lld * %lld elements, the buffer holds %lld", who, (long long)c->T, (long long)c->H, (long long)kept->n_elems);
    c->gate = kept->ptr;
    c->up = static_cast<char*>(kept->ptr) + size_t(c->T) * c->H * nk_dtype_size(dtype);
    return NK_OK;
}
int gated_check(nk_ctx* ctx, const char* who, int32_t fun, int32_t dtype) {
    if (dtype != NK_F32 && dtype != NK_F64) return nk_fail(ctx, NK_ERR_UNSUPPORTED, "%s: dtype %d not supported (F32/F64 only)", who, dtype);
    if (fun < 0 || fun >= NK_FUN_COUNT) return nk_fail(ctx, NK_ERR_BAD_ARG, "%s: unknown function id %d", who, fun);
    if (fun != NK_FUN_SIG && fun != NK_FUN_SILU && fun != NK_FUN_GELU && fun != NK_FUN_RELU && fun != NK_FUN_TANH && fun != NK_FUN_IDY)
        return nk_fail(ctx, NK_ERR_UNSUPPORTED, "%s: function id %d is no gate (sig, silu, gelu, relu, tanh, idy)", who, fun);
    return NK_OK;
}

}  // namespace

extern "C" int nk_gated(nk_ctx* ctx, int32_t fun, int32_t dtype, nk_buf* drn, const int32_t* cfg0, nk_buf* src, const int32_t* cfg1, nk_buf* w_gate,
                        const int32_t* cfg_gate, nk_buf* w_up, const int32_t* cfg_up, nk_buf* kept) {
    NK_CHECK_CTX(ctx);
    int st;
    if ((st = gated_check(ctx, "nk_gated", fun, dtype))) return st;
    GatedCall c;
    memset(&c, 0, sizeof(c));
    c.fun = fun;
    if ((st = gated_matrix(ctx, "nk_gated(src)", "src", src, cfg1, dtype, false, &c.T, &c.D, &c.x))) return st;
    if ((st = gated_matrix(ctx, "nk_gated(w_gate)", "w_gate", w_gate, cfg_gate, dtype, false, &c.D, &c.H, &c.w[0]))) return st;
    if ((st = gated_matrix(ctx, "nk_gated(w_up)", "w_up", w_up, cfg_up, dtype, false, &c.D, &c.H, &c.w[1]))) return st;
    if ((st = gated_matrix(ctx, "nk_gated(drain)", "the drain", drn, cfg0, dtype, true, &c.T, &c.H, &c.y))) return st;
    if (kept && (st = gated_kept(ctx, "nk_gated", kept, dtype, &c))) return st;
    return dtype == NK_F32 ? forward<float>(ctx, c) : forward<double>(ctx, c);
}

extern "C" int nk_gated_grad(nk_ctx* ctx, int32_t fun, int32_t dtype, nk_buf* dsrc, const int32_t* cfg_dsrc, nk_buf* dw_gate, const int32_t* cfg_dgate, nk_buf* dw_up,
                             const int32_t* cfg_dup, nk_buf* err, const int32_t* cfg_err, nk_buf* src, const int32_t* cfg1, nk_buf* w_gate, const int32_t* cfg_gate,
                             nk_buf* w_up, const int32_t* cfg_up, nk_buf* kept) {
    NK_CHECK_CTX(ctx);
    int st;
    if ((st = gated_check(ctx, "nk_gated_grad", fun, dtype))) return st;
    if (!kept) return nk_fail(ctx, NK_ERR_BAD_ARG, "nk_gated_grad: the products that the forward call kept are needed");
    GatedCall c;
    memset(&c, 0, sizeof(c));
    c.fun = fun;
    if ((st = gated_matrix(ctx, "nk_gated_grad(src)", "src", src, cfg1, dtype, false, &c.T, &c.D, &c.x))) return st;
    if ((st = gated_matrix(ctx, "nk_gated_grad(w_gate)", "w_gate", w_gate, cfg_gate, dtype, false, &c.D, &c.H, &c.w[0]))) return st;
    if ((st = gated_matrix(ctx, "nk_gated_grad(w_up)", "w_up", w_up, cfg_up, dtype, false, &c.D, &c.H, &c.w[1]))) return st;
    if ((st = gated_matrix(ctx, "nk_gated_grad(err)", "err", err, cfg_err, dtype, false, &c.T, &c.H, &c.err))) return st;
    if (dsrc && (st = gated_matrix(ctx, "nk_gated_grad(dsrc)", "dsrc", dsrc, cfg_dsrc, dtype, true, &c.T, &c.D, &c.dx))) return st;
    if (dw_gate && (st = gated_matrix(ctx, "nk_gated_grad(dw_gate)", "dw_gate", dw_gate, cfg_dgate, dtype, true, &c.D, &c.H, &c.dw[0]))) return st;
    if (dw_up && (st = gated_matrix(ctx, "nk_gated_grad(dw_up)", "dw_up", dw_up, cfg_dup, dtype, true, &c.D, &c.H, &c.dw[1]))) return st;
    if ((st = gated_kept(ctx, "nk_gated_grad", kept, dtype, &c))) return st;
    if (!dsrc && !dw_gate && !dw_up) return NK_OK;
    return dtype == NK_F32 ? backward<float>(ctx, c) : backward<double>(ctx, c);
}
