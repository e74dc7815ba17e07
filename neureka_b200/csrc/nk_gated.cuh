// The gated feed-forward block: what the kernel families behind nk_gated / nk_gated_grad share.
// f and f' are the framework's functions: F64 as they are (nk_scalarfun.cuh: the units are compiled with -fmad=false, products say fma), F32 below.
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

// The sigmoid in F32 and what is left to 1, from e^-|x| <= 1, so that neither cancels: some 4 units in the last place. The framework's F32
// functions evaluate it in F64 to be right to the last bit; here x is a product that is off by more than that, and at 64 F64 operations a clock an
// epilogue of 128 x 128 of them took 15,000 cycles, twice as long as the next products hide: 4096 x 2048 x 8192 forward 1.48 -> 1.30 ms.
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
template <class T>
__device__ __forceinline__ T gate_fun(int f, bool derive, T x) {
    if constexpr (sizeof(T) == 4) {
        switch (f) {
            case NK_FUN_SIG: return gate_fun32(NK_FUN_SIG, derive, x);
            case NK_FUN_SILU: return gate_fun32(NK_FUN_SILU, derive, x);
            case NK_FUN_GELU: return gate_fun32(NK_FUN_GELU, derive, x);
            case NK_FUN_RELU: return gate_fun32(NK_FUN_RELU, derive, x);
            case NK_FUN_TANH: return gate_fun32(NK_FUN_TANH, derive, x);
            default: return gate_fun32(NK_FUN_IDY, derive, x);
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
