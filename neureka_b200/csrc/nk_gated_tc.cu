// The gated block for many tokens in F32 on the tensor cores (3xTF32, nk_tc.cuh).
//
// Forward: nk_tc_split_kernel lays out x [T, D] and both weights [H, D] as hi / lo panels, then one product with two B operands: a tile is 256 tokens x
// 128 hidden features of both products (pairs of CTAs; 128 x 64 for lone ones), so that a thread of the epilogue holds g and u of the same
// elements and stores f(g) * u (and g and u, where a backward pass follows) straight from its registers.
// Backward: nk_gated_errors_split_kernel reads e, g and u once and leaves dg = e u f'(g) and du = e f(g) as panels in both directions they are needed in:
// [T, dg | du] for dx = [dg | du] [Wg | Wu]^T, one product over 2 H, and [H, T] each for dWg | dWu = x^T [dg | du], the product with two B
// operands again. These panels are 32 bytes per element of T x H (dx or dW alone: 16), those of the forward pass 8 per element of x and the weights.
#include "nk_gated.cuh"
#include "nk_tc.cuh"

namespace {

// eight values of a row: one 32-byte store fills its sector (rows of a tile are apart, so two of 16 bytes reach L2 as two halves)
__device__ __forceinline__ void store8(float* at, const float* v) {
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"l"(at), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]),
                 "f"(v[7]) : "memory");
}
// 16 columns of a warp's 32 rows, a lane per row, into rows of memory that no vector fits (their length is odd, or their base): stored as they are, every
// access would touch 32 rows, so the two 16 x 16 halves are turned first, after which an access covers 16 columns of two rows. 1023 x 777 x 2051
// forward: the product 51 -> 41 us, dW 70 -> 50 us.
__device__ __forceinline__ void store_turned(float* base, int64_t rs, int64_t m, int64_t n0, int64_t M, int64_t N, float (&v)[16]) {
    const int lane = threadIdx.x & 31, c = lane & 15;
#pragma unroll
    for (int s = 8; s > 0; s >>= 1) {
        const bool up = lane & s;
#pragma unroll
        for (int j = 0; j < 16; j++) {
            if (j & s) continue;
            const float got = __shfl_xor_sync(0xffffffffu, up ? v[j] : v[j | s], s);
            if (up) v[j] = got;
            else v[j | s] = got;
        }
    }
    const int64_t first = m - c;   // the row of the first lane of this half
    float* at = base + first * rs + n0 + c;
    if (n0 + c >= N) return;
#pragma unroll
    for (int j = 0; j < 16; j++)
        if (first + j < M) at[j * rs] = v[j];
}
// ... whatever the layout (called by whole warps; rows from M on are not there)
__device__ __forceinline__ void store16(float* base, int64_t rs, int64_t cs, int vec, int64_t m, int64_t n0, int64_t M, int64_t N, float (&v)[16]) {
    if (n0 >= N) return;
    if (cs == 1 && !vec) store_turned(base, rs, m, n0, M, N, v);
    else if (m >= M) return;
    else if (vec && n0 + 16 <= N) {
        store8(base + m * rs + n0, v);
        store8(base + m * rs + n0 + 8, v + 8);
    } else {
#pragma unroll
        for (int i = 0; i < 16; i++)
            if (n0 + i < N) base[m * rs + (n0 + i) * cs] = v[i];
    }
}
// f(g) * u, and g and u where they are kept
template <int FUN>
struct GatedDrain {
    static constexpr bool DUAL = true;
    float *y, *gate, *up;
    int64_t M, N, rs, cs;
    int vec, kept_vec;   // 32-byte stores: the rows of y; of gate and up
    template <int EC>
    __device__ __forceinline__ void store(int64_t m, int64_t n0, float (&sum)[EC]) const {
        constexpr int HC = EC / 2;
#pragma unroll
        for (int j = 0; j < HC; j += 16) {
            float v[16];
#pragma unroll
            for (int i = 0; i < 16; i++) v[i] = gate_fun32(FUN, false, sum[j + i]) * sum[HC + j + i];
            store16(y, rs, cs, vec, m, n0 + j, M, N, v);
        }
        if (!gate) return;
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
            for (int j = 0; j < HC; j += 16) {
                float v[16];
#pragma unroll
                for (int i = 0; i < 16; i++) v[i] = sum[b * HC + j + i];
                store16(b ? up : gate, N, 1, kept_vec, m, n0 + j, M, N, v);
            }
    }
};
// both products as they are; either may be unwanted
struct TwoDrain {
    static constexpr bool DUAL = true;
    float* out[2];
    int64_t M, N, rs[2], cs[2];
    int vec[2];          // 32-byte stores along the rows
    template <int EC>
    __device__ __forceinline__ void store(int64_t m, int64_t n0, float (&sum)[EC]) const {
        constexpr int HC = EC / 2;
#pragma unroll
        for (int b = 0; b < 2; b++) {
            if (!out[b]) continue;
#pragma unroll
            for (int j = 0; j < HC; j += 16) {
                float v[16];
#pragma unroll
                for (int i = 0; i < 16; i++) v[i] = sum[b * HC + j + i];
                store16(out[b], rs[b], cs[b], vec[b], m, n0 + j, M, N, v);
            }
        }
    }
};
// one product
struct OneDrain {
    static constexpr bool DUAL = false;
    float* out;
    int64_t M, N, rs, cs;
    int vec;
    template <int EC>
    __device__ __forceinline__ void store(int64_t m, int64_t n0, float (&sum)[EC]) const {
#pragma unroll
        for (int j = 0; j < EC; j += 16) {
            float v[16];
#pragma unroll
            for (int i = 0; i < 16; i++) v[i] = sum[j + i];
            store16(out, rs, cs, vec, m, n0 + j, M, N, v);
        }
    }
};

struct ErrorPanels {
    float *a_hi, *a_lo;         // [T][2 Hp], dg then du; null: not wanted
    float *t_hi[2], *t_lo[2];   // [H][Tp] of dg and of du; null: not wanted
    int64_t Hp, Tp;
    int err_vec, kept_vec;      // 16-byte loads along the rows
    int* tickets;               // cleared
    int n_tickets;
};
// 32 tokens x 128 hidden features per CTA: 12 bytes read and 32 written per element, four elements per thread and access.
template <int FUN>
__global__ void __launch_bounds__(256) nk_gated_errors_split_kernel(const GatedCall c, const ErrorPanels p, int64_t tiles_h) {
    __shared__ float tile[2][32][129];
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i < p.n_tickets; i += 256) p.tickets[i] = 0;
    const int64_t t0 = (blockIdx.x / tiles_h) * 32, h0 = (blockIdx.x % tiles_h) * 128;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float *err = static_cast<const float*>(c.err.ptr), *gate = static_cast<const float*>(c.gate), *up = static_cast<const float*>(c.up);
    const int64_t h = h0 + lane * 4;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int64_t t = t0 + warp + 8 * i;
        float e[4], g[4], u[4], d[2][4];
        const bool whole = t < c.T && h + 4 <= c.H;
        if (whole && p.err_vec) *reinterpret_cast<float4*>(e) = __ldcs(reinterpret_cast<const float4*>(err + t * c.err.rs + h));
        else {
#pragma unroll
            for (int j = 0; j < 4; j++) e[j] = t < c.T && h + j < c.H ? err[t * c.err.rs + (h + j) * c.err.cs] : 0.0f;
        }
        if (whole && p.kept_vec) {
            *reinterpret_cast<float4*>(g) = __ldcs(reinterpret_cast<const float4*>(gate + t * c.H + h));
            *reinterpret_cast<float4*>(u) = __ldcs(reinterpret_cast<const float4*>(up + t * c.H + h));
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const bool in = t < c.T && h + j < c.H;
                g[j] = in ? gate[t * c.H + h + j] : 0.0f;
                u[j] = in ? up[t * c.H + h + j] : 0.0f;
            }
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            d[0][j] = e[j] * u[j] * gate_fun32(FUN, true, g[j]);
            d[1][j] = e[j] * gate_fun32(FUN, false, g[j]);
#pragma unroll
            for (int b = 0; b < 2; b++) tile[b][warp + 8 * i][lane * 4 + j] = d[b][j];
        }
        if (p.a_hi && t < c.T && h < p.Hp) {
#pragma unroll
            for (int b = 0; b < 2; b++) {
                float hi[4], lo[4];
#pragma unroll
                for (int j = 0; j < 4; j++) tc_split(d[b][j], &hi[j], &lo[j]);
                const int64_t at = t * 2 * p.Hp + b * p.Hp + h;
                *reinterpret_cast<float4*>(p.a_hi + at) = make_float4(hi[0], hi[1], hi[2], hi[3]);
                *reinterpret_cast<float4*>(p.a_lo + at) = make_float4(lo[0], lo[1], lo[2], lo[3]);
            }
        }
    }
    __syncthreads();
    const int64_t t = t0 + (lane & 7) * 4;
    if (t >= p.Tp) return;   // Tp is a multiple of 16: whole vectors
#pragma unroll
    for (int b = 0; b < 2; b++) {
        if (!p.t_hi[b]) continue;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = (lane >> 3) + 4 * (warp + 8 * i);
            if (h0 + r >= c.H) continue;
            float hi[4], lo[4];
#pragma unroll
            for (int j = 0; j < 4; j++) tc_split(tile[b][(lane & 7) * 4 + j][r], &hi[j], &lo[j]);
            const int64_t at = (h0 + r) * p.Tp + t;
            *reinterpret_cast<float4*>(p.t_hi[b] + at) = make_float4(hi[0], hi[1], hi[2], hi[3]);
            *reinterpret_cast<float4*>(p.t_lo[b] + at) = make_float4(lo[0], lo[1], lo[2], lo[3]);
        }
    }
}

bool wide_rows(const GatedMatrix& m) { return m.cs == 1 && m.rs % 8 == 0 && reinterpret_cast<uintptr_t>(m.ptr) % 32 == 0; }
bool vec_rows(const GatedMatrix& m) { return m.cs == 1 && m.rs % 4 == 0 && reinterpret_cast<uintptr_t>(m.ptr) % 16 == 0; }
// [R, K] of a matrix's view: rows at row_stride, k at k_stride
TcOperand operand(const void* src, int64_t R, int64_t sR, int64_t K, int64_t sK) {
    TcOperand o;
    memset(&o, 0, sizeof(o));
    o.src = static_cast<const float*>(src);
    o.R = R; o.sR = sR; o.K = K; o.sK = sK;
    return o;
}
// consecutive pieces of one block, on 1024-byte boundaries
struct Pieces {
    size_t bytes = 0;
    size_t take(size_t b) {
        const size_t at = bytes;
        bytes += (b + 1023) / 1024 * 1024;
        return at;
    }
};
int split(nk_ctx* ctx, const TcSplit& sp) {
    int64_t tiles = 0;
    for (int i = 0; i < TC_OPERANDS; i++) tiles += sp.op[i].tiles;
    if (tiles > 0x7fffffffLL) return nk_fail(ctx, NK_ERR_UNSUPPORTED, "nk_gated: operands of more than 2^31 tiles");
    nk_tc_split_kernel<<<unsigned(tiles), 256, 0, ctx->stream>>>(sp);
    return nk_after_launch(ctx, "nk_tc_split_kernel");
}
// Chunks of 128 k leave a result 1.8e-6 off (2-norm, normal operands; the accumulator truncates), chunks of 64 k 0.9e-6, whatever the length of the
// sum; a sum of F32 multiply-adds is 2.7e-8 sqrt(K) off. So sums of up to 4096 take the shorter chunks, which cost a tenth of the time (accumulators
// are read out twice as often, and a tile's stores hide behind half as much: 4096 x 2048 x 8192 forward 1.18 -> 1.30 ms, 2048 x 4096 x 2048 0.35 -> 0.37), and longer ones lose
// nothing by the longer ones. Small calls take chunks of 32 (200 x 256 x 300 forward 20.5 -> 21.2 us, backward 48.8 -> 50.5).
template <class Drain>
int product(nk_ctx* ctx, const GatedCall& c, const TcShape& shape, int64_t Kp, const TcPanels& a, const TcPanels& b0, const TcPanels& b1, TcParams tp, const Drain& drain) {
    if (gated_small(c)) tp.chunk = TC_KC / 4;
    else if (Kp <= 4096) tp.chunk = TC_KC / 2;
    const int st = shape.pair ? tc_launch<2, 256>(ctx, "nk_conv_tc_kernel<3xtf32,pair>", Kp, a, b0, b1, tp, drain)
                              : tc_launch<1, 128>(ctx, "nk_conv_tc_kernel<3xtf32>", Kp, a, b0, b1, tp, drain);
    return st == -1 ? nk_fail(ctx, NK_ERR_CUDA, "nk_gated: the driver has no tensor-map encoder") : st;
}
// sizes that the tensor-core path takes
bool fits(nk_ctx* ctx, const GatedCall& c) {
    if (c.T <= nk_gated_few_most() || c.H < 64 || c.D < 64 || double(c.T) * double(c.D) * double(c.H) < double(1 << 20)) return false;
    const int64_t most = (int64_t(1) << 21) - 32;
    return c.T < most && c.D < most && c.H < most / 2 && size_t(TcCfg<2, 256>::SMEM_BYTES) <= size_t(ctx->prop.sharedMemPerBlockOptin);
}

}  // namespace

int nk_gated_tc_forward(nk_ctx* ctx, const GatedCall& c, bool* handled) {
    *handled = false;
    if (!fits(ctx, c)) return NK_OK;
    const int64_t Kp = tc_round_k(c.D);
    const TcShape shape = tc_shape(c.T, c.H, Kp, true, ctx->prop.multiProcessorCount);
    Pieces pieces;
    const size_t x_bytes = size_t(c.T) * Kp * 4, w_bytes = size_t(c.H) * Kp * 4;
    const size_t x_hi = pieces.take(x_bytes), x_lo = pieces.take(x_bytes), g_hi = pieces.take(w_bytes), g_lo = pieces.take(w_bytes), u_hi = pieces.take(w_bytes),
                 u_lo = pieces.take(w_bytes), parts = pieces.take(tc_part_bytes(shape)), tickets = pieces.take(tc_ticket_bytes(shape));
    NkWorkspace ws(ctx);
    int st = ws.get(pieces.bytes);
    if (st) return st;
    auto at = [&](size_t o) { return reinterpret_cast<float*>(static_cast<char*>(ws.ptr) + o); };
    TcSplit sp;
    memset(&sp, 0, sizeof(sp));
    sp.op[0] = operand(c.x.ptr, c.T, c.x.rs, c.D, c.x.cs);
    tc_operand_layout(&sp.op[0], c.x.cs == 1, at(x_hi), at(x_lo), Kp);
    for (int b = 0; b < 2; b++) {
        sp.op[1 + b] = operand(c.w[b].ptr, c.H, c.w[b].cs, c.D, c.w[b].rs);
        tc_operand_layout(&sp.op[1 + b], c.w[b].rs == 1, at(b ? u_hi : g_hi), at(b ? u_lo : g_lo), Kp);
    }
    sp.tickets = reinterpret_cast<int*>(at(tickets));
    sp.n_tickets = int(tc_ticket_bytes(shape) / sizeof(int));
    if ((st = split(ctx, sp))) return st;
    const TcParams tp = tc_params(shape, c.T, Kp, at(parts), sp.tickets, ctx->tma_status_dev);
    const TcPanels a{at(x_hi), at(x_lo), c.T}, b0{at(g_hi), at(g_lo), c.H}, b1{at(u_hi), at(u_lo), c.H};
    const int kept_vec = c.H % 8 == 0 && reinterpret_cast<uintptr_t>(c.gate) % 32 == 0 && reinterpret_cast<uintptr_t>(c.up) % 32 == 0;
#define NK_CASE(FUN) st = product(ctx, c, shape, Kp, a, b0, b1, tp, GatedDrain<FUN>{static_cast<float*>(c.y.ptr), static_cast<float*>(c.gate), static_cast<float*>(c.up), c.T, c.H, c.y.rs, c.y.cs, wide_rows(c.y), kept_vec})
    NK_GATE_SWITCH(c.fun, NK_CASE)
#undef NK_CASE
    *handled = true;
    return st;
}

int nk_gated_tc_backward(nk_ctx* ctx, const GatedCall& c, bool* handled) {
    *handled = false;
    if (!fits(ctx, c)) return NK_OK;
    const bool dx = c.dx.ptr != nullptr, dw = c.dw[0].ptr || c.dw[1].ptr;
    // few tokens: dx straight from the weights as they lie (nk_gated_narrow.cu), and short sums for small dW by F32 multiply-adds, which need no panels
    // (both dW alone: 41 x 115 x 1269 15 us against 25 here, 16 x 1024 x 2048 20 against 27, 32 x 1024 x 2048 27 against 29, but 64 x 1024 x 2048 37 against 30)
    const bool narrow = nk_gated_narrow(ctx, c);
    if (narrow && c.T <= 64 && double(c.T) * double(c.D) * double(c.H) <= double(1 << 26)) return NK_OK;
    const int64_t Hp = narrow ? nk_gated_narrow_columns(c.H) : tc_round_k(c.H), Tp = tc_round_k(c.T), sms = ctx->prop.multiProcessorCount;
    const TcShape sx = tc_shape(c.T, c.D, 2 * Hp, false, sms), sw = tc_shape(c.D, c.H, Tp, true, sms);
    Pieces pieces;
    const size_t a_bytes = dx ? size_t(c.T) * 2 * Hp * 4 : 0, w_bytes = dx && !narrow ? size_t(c.D) * 2 * Hp * 4 : 0;
    const size_t e_bytes = dw ? size_t(c.H) * Tp * 4 : 0, x_bytes = dw ? size_t(c.D) * Tp * 4 : 0;
    const size_t a_hi = pieces.take(a_bytes), a_lo = pieces.take(a_bytes), w_hi = pieces.take(w_bytes), w_lo = pieces.take(w_bytes);
    size_t e_at[2][2];
    for (int b = 0; b < 2; b++)
        for (int k = 0; k < 2; k++) e_at[b][k] = pieces.take(e_bytes);
    const size_t x_hi = pieces.take(x_bytes), x_lo = pieces.take(x_bytes);
    size_t px_bytes = tc_part_bytes(sx), tx_bytes = tc_ticket_bytes(sx);
    if (narrow) {
        int n;
        nk_gated_narrow_dx_needs(ctx, c, &px_bytes, &n);
        tx_bytes = size_t(n) * sizeof(int);
    }
    if (!dx) px_bytes = tx_bytes = 0;
    const size_t px = pieces.take(px_bytes), pw = pieces.take(dw ? tc_part_bytes(sw) : 0), tw_bytes = dw ? tc_ticket_bytes(sw) : 0;
    const size_t tickets = pieces.take(tx_bytes + tw_bytes);
    NkWorkspace ws(ctx);
    int st = ws.get(pieces.bytes);
    if (st) return st;
    auto at = [&](size_t o) { return reinterpret_cast<float*>(static_cast<char*>(ws.ptr) + o); };

    ErrorPanels ep;
    memset(&ep, 0, sizeof(ep));
    ep.Hp = Hp;
    ep.Tp = Tp;
    if (dx) { ep.a_hi = at(a_hi); ep.a_lo = at(a_lo); }
    for (int b = 0; b < 2 && dw; b++) { ep.t_hi[b] = at(e_at[b][0]); ep.t_lo[b] = at(e_at[b][1]); }
    ep.err_vec = vec_rows(c.err);
    ep.kept_vec = c.H % 4 == 0 && reinterpret_cast<uintptr_t>(c.gate) % 16 == 0 && reinterpret_cast<uintptr_t>(c.up) % 16 == 0;
    ep.tickets = reinterpret_cast<int*>(at(tickets));
    ep.n_tickets = int((tx_bytes + tw_bytes) / sizeof(int));
    const int64_t tiles_h = (Hp + 127) / 128, tiles = tiles_h * ((Tp + 31) / 32);
    if (tiles > 0x7fffffffLL) return nk_fail(ctx, NK_ERR_UNSUPPORTED, "nk_gated_grad: an error of more than 2^31 tiles");
#define NK_CASE(FUN) nk_gated_errors_split_kernel<FUN><<<unsigned(tiles), 256, 0, ctx->stream>>>(c, ep, tiles_h)
    NK_GATE_SWITCH(c.fun, NK_CASE)
#undef NK_CASE
    if ((st = nk_after_launch(ctx, "nk_gated_errors_split_kernel"))) return st;

    TcSplit sp;
    memset(&sp, 0, sizeof(sp));
    int ops = 0;
    for (int b = 0; b < 2 && dx && !narrow; b++) {   // [Wg | Wu]: rows d, k = h
        TcOperand& o = sp.op[ops++];
        o = operand(c.w[b].ptr, c.D, c.w[b].rs, c.H, c.w[b].cs);
        tc_operand_layout(&o, c.w[b].cs == 1, at(w_hi) + b * Hp, at(w_lo) + b * Hp, 2 * Hp);
    }
    if (dw) {   // x^T: rows d, k = t
        TcOperand& o = sp.op[ops++];
        o = operand(c.x.ptr, c.D, c.x.cs, c.T, c.x.rs);
        tc_operand_layout(&o, c.x.rs == 1, at(x_hi), at(x_lo), Tp);
    }
    if (ops && (st = split(ctx, sp))) return st;
    if (dx && narrow) {
        if ((st = nk_gated_narrow_dx_panels(ctx, c, at(a_hi), at(a_lo), at(px), ep.tickets))) return st;
    } else if (dx) {
        const OneDrain drain{static_cast<float*>(c.dx.ptr), c.T, c.D, c.dx.rs, c.dx.cs, wide_rows(c.dx)};
        const TcPanels a{at(a_hi), at(a_lo), c.T}, b{at(w_hi), at(w_lo), c.D};
        if ((st = product(ctx, c, sx, 2 * Hp, a, b, b, tc_params(sx, c.T, 2 * Hp, at(px), ep.tickets, ctx->tma_status_dev), drain))) return st;
    }
    if (dw) {
        TwoDrain drain;
        memset(&drain, 0, sizeof(drain));
        drain.M = c.D;
        drain.N = c.H;
        for (int b = 0; b < 2; b++) {
            drain.out[b] = static_cast<float*>(c.dw[b].ptr);
            drain.rs[b] = c.dw[b].rs;
            drain.cs[b] = c.dw[b].cs;
            drain.vec[b] = wide_rows(c.dw[b]);
        }
        const TcPanels a{at(x_hi), at(x_lo), c.D}, b0{at(e_at[0][0]), at(e_at[0][1]), c.H}, b1{at(e_at[1][0]), at(e_at[1][1]), c.H};
        st = product(ctx, c, sw, Tp, a, b0, b1, tc_params(sw, c.D, Tp, at(pw), ep.tickets + tx_bytes / sizeof(int), ctx->tma_status_dev), drain);
    }
    *handled = true;
    return st;
}
