// The gated feed-forward block: what the kernel families behind nk_gated / nk_gated_grad share.
// f and f' are the framework's functions (nk_scalarfun.cuh: the units are compiled with -fmad=false, products say fma).
#pragma once
#include "nk_internal.h"
#include "nk_scalarfun.cuh"

// A matrix: element (r, c) at base[r * rs + c * cs].
struct GatedMatrix {
    void* ptr;      // null: not wanted
    int64_t rs, cs;
};

// One call. T tokens, D features of the model, H hidden ones.
struct GatedCall {
    int fun;
    int64_t T, D, H;
    GatedMatrix x, w[2];      // [T, D]; gate and up [D, H]
    GatedMatrix y;            // forward: [T, H]
    void *gate, *up;          // x @ w[0], x @ w[1], row-major [T, H]; forward: null where nobody keeps them
    GatedMatrix err;          // backward: [T, H]
    GatedMatrix dx, dw[2];    // backward
};
// Products that `@` computes with F32 multiply-adds (below 2^24 of them). The block takes them to the tensor cores all the same, with accumulation chunks so short
// that a sum is no further off: 2.0e-7 to 2.5e-7 (2-norm, also for terms of one sign; multiply-adds 1.1e-7 sqrt(K / 64) at 64 to 512 terms).
inline bool gated_small(const GatedCall& c) { return double(c.T) * double(c.D) * double(c.H) < double(1 << 24); }

// f(x) and f'(x). In F32 both are evaluated in F64 and rounded once: sig, silu, gelu, relu and idy are the framework's own values to the last bit; tanh and the
// derivatives too are right to the last bit, where the framework's formulas (the reference's: 1 - s, 2 / (1 + e) - 1) cancel.
__device__ __forceinline__ float gate_derivative(int f, float x) {
    const double a = (f == NK_FUN_GELU ? 1.702 : f == NK_FUN_TANH ? 2.0 : 1.0) * double(x), c = fmin(fmax(a, -700.0), 700.0);   // (beyond, e and its products are 0 in F32)
    const double e = nkf::nk_exp_reduced(-fabs(c)), t = 1.0 / (1.0 + e), both = e * t * t;   // both: s (1 - s)
    const double v = f == NK_FUN_SIG ? both : f == NK_FUN_TANH ? 4.0 * both : (c < 0.0 ? e * t : t) + c * both;
    return x != x ? x : float(v);
}
template <class T>
__device__ __forceinline__ T gate_fun(int f, bool derive, T x) {
    if constexpr (sizeof(T) == 4) {
        if (f != NK_FUN_RELU && f != NK_FUN_IDY) {
            if (derive) return gate_derivative(f, x);
            if (f == NK_FUN_TANH) return float(tanh(double(x)));
        }
    }
    switch (f) {
        case NK_FUN_SIG: return nkf::fun(NK_FUN_SIG, derive, x);
        case NK_FUN_SILU: return nkf::fun(NK_FUN_SILU, derive, x);
        case NK_FUN_GELU: return nkf::fun(NK_FUN_GELU, derive, x);
        case NK_FUN_RELU: return nkf::fun(NK_FUN_RELU, derive, x);
        case NK_FUN_TANH: return nkf::fun(NK_FUN_TANH, derive, x);
        default: return nkf::fun(NK_FUN_IDY, derive, x);
    }
}

// The same in F32, where the products come from the tensor cores: the sigmoid and what is left to 1 from e^-|x| <= 1, so that neither cancels, some 4
// units in the last place off, and x is a product that is off by more than that. At 64 F64 operations a clock an epilogue of 128 x 128 gates took 15,000
// cycles, twice as long as the next products hide (4096 x 2048 x 8192 forward 1.48 -> 1.30 ms), and that of some tokens, which nothing hides, a
// tenth of a small call (24 x 515 x 900 22.5 us, so 20.5). Where the products are F32 or F64 multiply-adds, memory or latency leaves room
// for gate_fun (1 x 2048 x 5461 26.6 us against 25.6, 300 x 30 x 500 13.0 against 11.3).
__device__ __forceinline__ float gate_sig(float x, float* rest) {
    const float e = expf(-fabsf(x)), t = __fdividef(1.0f, 1.0f + e), m = e * t;
    *rest = x < 0.0f ? t : m;
    return x < 0.0f ? m : t;
}
__device__ __forceinline__ float gate_fun32(int f, bool derive, float x) {
    if (f == NK_FUN_RELU || f == NK_FUN_IDY) return nkf::fun(f, derive, x);
    if (f == NK_FUN_TANH) {
        if (!derive) return tanhf(x);
        const float e = expf(-2.0f * fabsf(x)), t = __fdividef(1.0f, 1.0f + e);
        return 4.0f * e * t * t;
    }
    const float k = 1.702f;
    const bool gelu = f == NK_FUN_GELU;
    const float a = gelu ? k * x : x;
    float rest, s = gate_sig(a, &rest);
    if (gelu) {   // what the product's rounding (and that of 1.702) left out, to first order; where |a| is large the sigmoid is 0 or 1
        const float left = fabsf(x) < 64.0f ? fmaf(k, x, -a) + float(1.702 - double(1.702f)) * x : 0.0f, at = s;
        s = fmaf(s * rest, left, s);
        rest = fmaf(-at * rest, left, rest);
    }
    if (f == NK_FUN_SIG) return derive ? s * rest : s;
    return derive ? fmaf(fminf(fmaxf(a, -128.0f), 128.0f) * rest, s, s) : x * s;   // (rest or s is 0 beyond, and 1.702 x may be infinite)
}
__device__ __forceinline__ float gate_fun32(int f, float x) {   // of a call's function
    switch (f) {
        case NK_FUN_SIG: return gate_fun32(NK_FUN_SIG, false, x);
        case NK_FUN_SILU: return gate_fun32(NK_FUN_SILU, false, x);
        case NK_FUN_GELU: return gate_fun32(NK_FUN_GELU, false, x);
        case NK_FUN_RELU: return gate_fun32(NK_FUN_RELU, false, x);
        case NK_FUN_TANH: return gate_fun32(NK_FUN_TANH, false, x);
        default: return gate_fun32(NK_FUN_IDY, false, x);
    }
}
// CASE(FUN) for the function of a call
#define NK_GATE_SWITCH(fun, CASE)                 \
    switch (fun) {                                \
        case NK_FUN_SIG: CASE(NK_FUN_SIG); break;   \
        case NK_FUN_SILU: CASE(NK_FUN_SILU); break; \
        case NK_FUN_GELU: CASE(NK_FUN_GELU); break; \
        case NK_FUN_RELU: CASE(NK_FUN_RELU); break; \
        case NK_FUN_TANH: CASE(NK_FUN_TANH); break; \
        default: CASE(NK_FUN_IDY); break;           \
    }

// Many tokens in F32 on the tensor cores (nk_gated_tc.cu); *handled stays false where the call is not theirs.
int nk_gated_tc_forward(nk_ctx* ctx, const GatedCall& c, bool* handled);
int nk_gated_tc_backward(nk_ctx* ctx, const GatedCall& c, bool* handled);

// Few tokens, at most nk_gated_few_most(), both types (nk_gated_few.cu). dg and du: row-major [T, H].
int64_t nk_gated_few_most();
template <class T> int nk_gated_few_forward(nk_ctx* ctx, const GatedCall& c);
template <class T> int nk_gated_few_dx(nk_ctx* ctx, const GatedCall& c, const T* dg, const T* du);
template <class T> int nk_gated_few_dw(nk_ctx* ctx, const GatedCall& c, const T* dg, const T* du);

// Some tokens in F32 (nk_gated_narrow.cu). dx from dg and du, or from panels hi and lo [T][2 * nk_gated_narrow_columns(H)] of them, zero past H, and
// cleared tickets.
bool nk_gated_narrow(const nk_ctx* ctx, const GatedCall& c);
int nk_gated_narrow_forward(nk_ctx* ctx, const GatedCall& c);
int64_t nk_gated_narrow_columns(int64_t H);
void nk_gated_narrow_dx_needs(nk_ctx* ctx, const GatedCall& c, size_t* part_bytes, int* tickets);
int nk_gated_narrow_dx(nk_ctx* ctx, const GatedCall& c, const float* dg, const float* du);
int nk_gated_narrow_dx_panels(nk_ctx* ctx, const GatedCall& c, const float* hi, const float* lo, float* parts, int* tickets);
