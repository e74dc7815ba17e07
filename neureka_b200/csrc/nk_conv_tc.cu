// Tensor-core family for F32 contraction-shaped convolution calls ([M,K,1] x [1,K,N], `Tensor.convDot`, `@`, and the two
// gradients of such calls): O[m, n] = sum_k A[m, k] * B[k, n] on the 5th-generation tensor cores with the 3xTF32 split.
// Replaces what the reference runs for these shapes on a GPU, `fast_CM_MM_MxKxN`
// (src/main/java/neureka/backend/main/operations/linear/internal/opencl/CLGEMM.java:44-92); the semantics are those of
// AbstractCPUConvolution.java:245-316 (forward) / :319-408 (deconvolution) restricted to contraction-shaped calls.
//
// The split, the kernel and how it accumulates: nk_tc.cuh.
//
// Launch sequence (one stream, one scratch block):
//   1. nk_gemm_offsets_kernel  -- only when an index group of the views has several dims (or the drain is wider than its own
//      strides tell): the groups flattened into offset tables. A matrix product's groups are one stride each: no tables;
//   2. nk_tc_split_kernel      -- gathers both operands into dense K-major arrays hi[rows][Kp] and lo[rows][Kp] (Kp = K
//      rounded up to 16, zero padded); an operand whose rows are the contiguous direction is transposed on the way, so
//      both reach the tensor cores K-major. It also clears the tickets of a k-split product;
//   3. nk_conv_tc_kernel       -- persistent, warp-specialised: one producer thread issues cp.async.bulk.tensor (TMA,
//      64-byte swizzle, no multicast, this GPU's memory only) into a ring of {A_hi, A_lo, B_hi, B_lo} panels of 16 k each;
//      one thread issues tcgen05.mma (kind::tf32, K = 8; six per stage) into one of two F32 accumulators in tensor memory
//      and hands stages back with tcgen05.commit; sixteen warps read finished accumulators with tcgen05.ld and scatter the
//      tile through the drain's strides or tables.
#include "nk_gemm_plan.h"
#include "nk_tc.cuh"

int nk_conv_tc_try(nk_ctx* ctx, nk_buf* drn, nk_buf* s1, nk_buf* s2, const GemmPlan& p, bool* handled) {
    *handled = false;
    const bool forced = ctx->conv_path == NK_CONV_TC;
    // worth three extra launches and a pass over both operands only for real matrix products
    if (p.M < 64 || p.N < 64 || p.K < 32) return NK_OK;
    if (!forced && double(p.M) * double(p.N) * double(p.K) < double(1 << 24)) return NK_OK;
    if (p.K > (int64_t(1) << 21) - 32 || p.M >= (int64_t(1) << 31) || p.N >= (int64_t(1) << 31)) return NK_OK;
    const int64_t Kp = tc_round_k(p.K);
    if (((p.M + 127) / 128) * ((p.N + 127) / 128) > 0x7fffffffLL) return NK_OK;
    if (size_t(TcCfg<2, 256>::SMEM_BYTES) > size_t(ctx->prop.sharedMemPerBlockOptin)) return NK_OK;
    const TcShape shape = tc_shape(p.M, p.N, Kp, false, ctx->prop.multiProcessorCount);

    // scratch: [tables | A_hi | A_lo | B_hi | B_lo | parts | tickets], the arrays on 1024-byte boundaries
    const bool tables = p.m.n > 1 || p.n.n > 1 || p.k.n > 1;
    auto round = [](size_t b) { return ((b + 1023) / 1024) * 1024; };
    const size_t tab_bytes = tables ? round(size_t(2 * (p.M + p.N + p.K)) * sizeof(int64_t)) : 0;
    const size_t a_bytes = round(size_t(p.M) * Kp * 4), b_bytes = round(size_t(p.N) * Kp * 4);
    const size_t part_bytes = tc_part_bytes(shape), ticket_bytes = tc_ticket_bytes(shape);
    void* scratch = nullptr;
    int st = nk_scratch(ctx, tab_bytes + 2 * a_bytes + 2 * b_bytes + part_bytes + ticket_bytes + 1024, &scratch);
    if (st) return st;
    scratch = reinterpret_cast<void*>((reinterpret_cast<uintptr_t>(scratch) + 1023) & ~uintptr_t(1023));
    int64_t* tab = reinterpret_cast<int64_t*>(scratch);
    char* base = reinterpret_cast<char*>(scratch) + tab_bytes;
    float *Ahi = reinterpret_cast<float*>(base), *Alo = reinterpret_cast<float*>(base + a_bytes);
    float *Bhi = reinterpret_cast<float*>(base + 2 * a_bytes), *Blo = reinterpret_cast<float*>(base + 2 * a_bytes + b_bytes);
    char* rest = base + 2 * a_bytes + 2 * b_bytes;

    if (tables) {
        st = nk_gemm_build_tables(ctx, p, tab);
        if (st) return st;
    }
    TcSplit sp;
    memset(&sp, 0, sizeof(sp));
    sp.tickets = reinterpret_cast<int*>(rest + part_bytes);
    sp.n_tickets = int(ticket_bytes / sizeof(int));
    auto stride = [](const GemmDims& g, bool second) { return g.n == 1 ? (second ? g.sb[0] : g.sa[0]) : 0; };   // n == 0: extent 1
    TcOperand& A = sp.op[0];
    A.src = static_cast<const float*>(s1->ptr) + p.bA;
    A.sR = stride(p.m, false); A.sK = stride(p.k, false); A.R = p.M; A.K = p.K;
    TcOperand& B = sp.op[1];
    B.src = static_cast<const float*>(s2->ptr) + p.bB;
    B.sR = stride(p.n, false); B.sK = stride(p.k, true); B.R = p.N; B.K = p.K;
    if (tables) {   // [offA_m | offO_m | offB_n | offO_n | offA_k | offB_k]
        A.offR = tab; A.offK = tab + 2 * p.M + 2 * p.N;
        B.offR = tab + 2 * p.M; B.offK = tab + 2 * p.M + 2 * p.N + p.K;
    }
    // is k the contiguous direction of an operand? (the innermost dim of its k group has stride 1)
    tc_operand_layout(&A, p.k.n > 0 && p.k.sa[p.k.n - 1] == 1, Ahi, Alo, Kp);
    tc_operand_layout(&B, p.k.n > 0 && p.k.sb[p.k.n - 1] == 1, Bhi, Blo, Kp);
    if (A.tiles + B.tiles > 0x7fffffffLL) return NK_OK;
    nk_tc_split_kernel<<<unsigned(A.tiles + B.tiles), 256, 0, ctx->stream>>>(sp);
    if ((st = nk_after_launch(ctx, "nk_tc_split_kernel"))) return st;

    TcPlainDrain drain;
    memset(&drain, 0, sizeof(drain));
    drain.out = static_cast<float*>(drn->ptr);
    drain.M = p.M;
    drain.N = p.N;
    if (tables) { drain.offOm = tab + p.M; drain.offOn = tab + 2 * p.M + p.N; }
    drain.sOm = stride(p.m, true);
    drain.sOn = stride(p.n, true);
    drain.bO = p.bO;
    bool vec = p.n.n == 1 && p.n.sb[0] == 1 && (p.bO % 4) == 0 && (reinterpret_cast<uintptr_t>(drn->ptr) % 16) == 0;
    for (int d = 0; d < p.m.n && vec; d++) vec = (p.m.sb[d] % 4) == 0;
    drain.out_vec = vec ? 1 : 0;
    const TcParams tp = tc_params(shape, p.M, Kp, reinterpret_cast<float*>(rest), sp.tickets, ctx->tma_status_dev);
    const TcPanels a{Ahi, Alo, p.M}, b{Bhi, Blo, p.N};
    st = shape.pair ? tc_launch<2, 256>(ctx, "nk_conv_tc_kernel<3xtf32,pair>", Kp, a, b, b, tp, drain)
                    : tc_launch<1, 128>(ctx, "nk_conv_tc_kernel<3xtf32>", Kp, a, b, b, tp, drain);
    if (st == -1) return NK_OK;   // the FMA family takes the call
    if (st) return st;
    *handled = true;
    return NK_OK;
}
