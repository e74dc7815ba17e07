// Dropout from a counter-based generator (no counterpart in the reference). The mask of element i is a function of (seed, stream, i): word i % 4 of
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", SC 2011) for the counter (i / 4, stream) and
// the key seed. It is drawn where it is needed, forward and backward, and never stored.
//
// A thread takes four consecutive elements, the four words of one counter. Compiled with -fmad=false: the product and the residual's sum
// round one after the other, like the separate operators.
#include "nk_internal.h"

namespace {

struct DropPlan {
    int nd;
    int64_t total;
    int64_t ext[NK_MAX_RANK];
    int64_t s0[NK_MAX_RANK], s1[NK_MAX_RANK], s2[NK_MAX_RANK];   // drain, source, residual
    unsigned below;                                              // words below this are dropped
    unsigned key[2], stream[2];
};

__device__ __forceinline__ void philox(unsigned (&c)[4], unsigned k0, unsigned k1) {
#pragma unroll
    for (int r = 0; r < 10; r++) {
        const unsigned a_lo = c[0] * 0xD2511F53u, a_hi = __umulhi(c[0], 0xD2511F53u);
        const unsigned b_lo = c[2] * 0xCD9E8D57u, b_hi = __umulhi(c[2], 0xCD9E8D57u);
        c[0] = b_hi ^ c[1] ^ (k0 + unsigned(r) * 0x9E3779B9u);
        c[1] = b_lo;
        c[2] = a_hi ^ c[3] ^ (k1 + unsigned(r) * 0xBB67AE85u);
        c[3] = a_lo;
    }
}

// Every operand contiguous and 16-byte aligned: vectors of 16 bytes, two groups per trip with all their loads before the first store.
// Drawing the mask takes about 60 instructions per group, a third of what the SMs can issue in the time the memory needs for it. Bound by the
// memory: 8192 x 8192 F32 with a residual and its backward pass 245 us, 5.5 TB/s (element by element 582).
template <class T> struct DropVec { using type = float4; };
template <> struct DropVec<double> { using type = double2; };
template <class T, bool RES>
__global__ void __launch_bounds__(256) nk_dropout_linear_kernel(T* out, const T* src, const T* res, const DropPlan p, const T scale) {
    using V = typename DropVec<T>::type;
    constexpr int VW = 16 / int(sizeof(T)), NV = 4 / VW;   // vectors of a group
    const int64_t whole = p.total / 4, stride = int64_t(gridDim.x) * blockDim.x, tid = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
    for (int64_t g0 = tid; g0 < whole; g0 += 2 * stride) {
        T v[2][4], r[2][4];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int64_t g = g0 + u * stride;
            if (g >= whole) break;
#pragma unroll
            for (int k = 0; k < NV; k++) {
                *reinterpret_cast<V*>(&v[u][k * VW]) = __ldcs(reinterpret_cast<const V*>(src + g * 4) + k);
                if (RES) *reinterpret_cast<V*>(&r[u][k * VW]) = __ldcs(reinterpret_cast<const V*>(res + g * 4) + k);
            }
        }
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int64_t g = g0 + u * stride;
            if (g >= whole) break;
            unsigned c[4] = {unsigned(g), unsigned(uint64_t(g) >> 32), p.stream[0], p.stream[1]};
            philox(c, p.key[0], p.key[1]);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                v[u][j] = c[j] >= p.below ? v[u][j] * scale : T(0);
                if (RES) v[u][j] = r[u][j] + v[u][j];
            }
#pragma unroll
            for (int k = 0; k < NV; k++) __stcs(reinterpret_cast<V*>(out + g * 4) + k, *reinterpret_cast<V*>(&v[u][k * VW]));
        }
    }
    if (tid == 0 && whole * 4 < p.total) {   // the last one to three elements
        unsigned c[4] = {unsigned(whole), unsigned(uint64_t(whole) >> 32), p.stream[0], p.stream[1]};
        philox(c, p.key[0], p.key[1]);
        for (int64_t i = whole * 4; i < p.total; i++) {
            T v = c[i - whole * 4] >= p.below ? src[i] * scale : T(0);
            if (RES) v = res[i] + v;
            out[i] = v;
        }
    }
}

// Any views: the indices of the first element by division (I: 32 bits where the index fits), the next three by counting up.
template <class T, bool RES, class I>
__global__ void __launch_bounds__(256) nk_dropout_kernel(T* out, const T* src, const T* res, const DropPlan p, const T scale) {
    const int64_t groups = (p.total + 3) / 4, stride = int64_t(gridDim.x) * blockDim.x;
    for (int64_t g = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; g < groups; g += stride) {
        unsigned c[4] = {unsigned(g), unsigned(uint64_t(g) >> 32), p.stream[0], p.stream[1]};
        philox(c, p.key[0], p.key[1]);
        I idx[NK_MAX_RANK], rem = I(g * 4);
        int64_t o0 = 0, o1 = 0, o2 = 0;
#pragma unroll
        for (int k = NK_MAX_RANK - 1; k >= 0; k--) {
            if (k >= p.nd) continue;
            const I q = k ? rem / I(p.ext[k]) : I(0);
            idx[k] = rem - q * I(p.ext[k]);
            rem = q;
            o0 += int64_t(idx[k]) * p.s0[k]; o1 += int64_t(idx[k]) * p.s1[k]; o2 += int64_t(idx[k]) * p.s2[k];
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (g * 4 + j < p.total) {
                T v = c[j] >= p.below ? src[o1] * scale : T(0);
                if (RES) v = res[o2] + v;
                out[o0] = v;
            }
            bool carry = true;
#pragma unroll
            for (int k = NK_MAX_RANK - 1; k >= 0; k--) {
                if (k >= p.nd || !carry) continue;
                idx[k]++; o0 += p.s0[k]; o1 += p.s1[k]; o2 += p.s2[k];
                carry = idx[k] == I(p.ext[k]);
                if (carry) {
                    o0 -= p.ext[k] * p.s0[k]; o1 -= p.ext[k] * p.s1[k]; o2 -= p.ext[k] * p.s2[k];
                    idx[k] = 0;
                }
            }
        }
    }
}

template <class T> T* at(nk_buf* b, const NkView& v) { return static_cast<T*>(b->ptr) + v.base; }

template <class T, bool RES>
int launch(nk_ctx* ctx, T* out, const T* src, const T* res, const DropPlan& p, double prob) {
    const T scale = T(1.0 / (1.0 - prob));
    auto aligned = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0; };
    const bool linear = p.nd == 1 && p.s0[0] == 1 && p.s1[0] == 1 && (!RES || p.s2[0] == 1) && aligned(out) && aligned(src) && (!RES || aligned(res));
    const int grid = nk_grid_for(ctx, (p.total + 3) / 4, 256, 8);
    if (linear) {
        nk_dropout_linear_kernel<T, RES><<<grid, 256, 0, ctx->stream>>>(out, src, res, p, scale);
        return nk_after_launch(ctx, "nk_dropout_linear_kernel");
    }
    if (p.total < (int64_t(1) << 31)) nk_dropout_kernel<T, RES, unsigned><<<grid, 256, 0, ctx->stream>>>(out, src, res, p, scale);
    else nk_dropout_kernel<T, RES, int64_t><<<grid, 256, 0, ctx->stream>>>(out, src, res, p, scale);
    return nk_after_launch(ctx, "nk_dropout_kernel");
}

}  // namespace

extern "C" int nk_dropout(nk_ctx* ctx, int32_t dtype, int32_t rank, nk_buf* drn, const int32_t* cfg0, nk_buf* src, const int32_t* cfg1,
                          nk_buf* residual, const int32_t* cfg2, double prob, int64_t seed, int64_t stream) {
    NK_CHECK_CTX(ctx);
    if (dtype != NK_F32 && dtype != NK_F64) return nk_fail(ctx, NK_ERR_UNSUPPORTED, "nk_dropout: dtype %d not supported (F32/F64 only)", dtype);
    if (!(prob >= 0.0 && prob < 1.0)) return nk_fail(ctx, NK_ERR_BAD_ARG, "nk_dropout: probability %g outside [0, 1)", prob);
    NkView v0, v1, v2;
    int st;
    if ((st = nk_view_parse(ctx, "nk_dropout(drain)", drn, cfg0, rank, dtype, &v0))) return st;
    if ((st = nk_check_drain(ctx, "nk_dropout", v0))) return st;
    if ((st = nk_view_parse(ctx, "nk_dropout(src)", src, cfg1, rank, dtype, &v1))) return st;
    v2 = v1;
    if (residual && (st = nk_view_parse(ctx, "nk_dropout(residual)", residual, cfg2, rank, dtype, &v2))) return st;
    for (int k = 0; k < rank; k++)
        if (v0.shape[k] != v1.shape[k] || v0.shape[k] != v2.shape[k])
            return nk_fail(ctx, NK_ERR_BAD_ARG, "nk_dropout: shapes differ at dim %d (%lld, %lld, %lld)", k, (long long)v0.shape[k], (long long)v1.shape[k],
                           (long long)v2.shape[k]);
    // size-1 dims go, neighbours merge where every operand is linear across them; the row-major index of an element stays what it is
    DropPlan p;
    memset(&p, 0, sizeof(p));
    p.total = v0.size;
    for (int k = 0; k < rank; k++) {
        const int64_t e = v0.shape[k], a = v0.estride[k], b = v1.estride[k], c = residual ? v2.estride[k] : 0;
        if (e == 1) continue;
        const int l = p.nd - 1;
        if (l >= 0 && p.s0[l] == e * a && p.s1[l] == e * b && p.s2[l] == e * c) {
            p.ext[l] *= e;
            p.s0[l] = a; p.s1[l] = b; p.s2[l] = c;
        } else {
            p.ext[p.nd] = e;
            p.s0[p.nd] = a; p.s1[p.nd] = b; p.s2[p.nd] = c;
            p.nd++;
        }
    }
    if (p.nd == 0) { p.nd = 1; p.ext[0] = 1; }
    p.below = unsigned(prob * 4294967296.0);
    p.key[0] = unsigned(uint64_t(seed)); p.key[1] = unsigned(uint64_t(seed) >> 32);
    p.stream[0] = unsigned(uint64_t(stream)); p.stream[1] = unsigned(uint64_t(stream) >> 32);
    if (dtype == NK_F32)
        return residual ? launch<float, true>(ctx, at<float>(drn, v0), at<float>(src, v1), at<float>(residual, v2), p, prob)
                        : launch<float, false>(ctx, at<float>(drn, v0), at<float>(src, v1), nullptr, p, prob);
    return residual ? launch<double, true>(ctx, at<double>(drn, v0), at<double>(src, v1), at<double>(residual, v2), p, prob)
                    : launch<double, false>(ctx, at<double>(drn, v0), at<double>(src, v1), nullptr, p, prob);
}
