// The gated feed-forward block: what the kernel families behind nk_gated / nk_gated_grad share.
#pragma once
#include "nk_internal.h"

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
