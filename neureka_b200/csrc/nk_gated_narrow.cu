// The gated block in F32 for some tokens (more than the streaming kernels take, fewer than fill a tile's rows): tensor cores, with the weights read
// from memory once and never laid out anew.
//
//   forward:  R_b[n, t] = sum_k w_b[k, n] x[t, k], out = f(R_0) * R_1         dx ("SUM"):  R[n, t] = sum_b sum_k w_b[k, n] x_b[t, k], out = R
//
// The weights are the product's A operand: 128 columns n are the rows of the tensor core's tile, the tokens (padded to 16, 32 or 64) its columns.
// A 3xTF32 product needs hi and lo of every weight; writing them to memory and reading them back would move five times the weights' bytes
// (nk_gated_tc.cu does, where a panel is used by many tiles). Here a warp brings 32 columns x 16 k into shared memory (cp.async, two or three
// such patches ahead: loads into registers, two ahead, left the memory at a third of its rate), splits them in registers and stores hi
// and lo into tensor memory, from where tcgen05.mma takes its A operand. The tokens' panels are split before (they are small) and come by TMA.
// What is left is the stream of weights: 4 bytes per element against 6 multiply-adds per token. 16 tokens x 4096 x 8192 64 us, where the weights' bytes take
// 41; 64 tokens 80; 24 x 2048 x 5461 38 us (14): bound by the issue of the converters (split, store) and, from 64 tokens on, by the products.
//
// Roles, 18 warps: 0..15 converters in two groups, warp 16 fetches the tokens' panels, warp 17 issues the products. A stage is 32 k of both weights
// (SUM: 64 k of one); every converter splits 32 columns x 16 k of it, warp w for lanes 32 (w % 4) of the tile. Tensor memory: three (two)
// stages of 128 columns (4 x (16 hi + 16 lo)) and the accumulators. (Stages of half that size: the issuing warp's waits took as long as its products.)
// A product of 128 x up to 128 x 8 takes about 86 cycles here whatever its width, so the tokens' hi and lo panels lie side by side as one operand:
// hi x [hi | lo], then lo x hi onto the second half -- two products per 8 k instead of three, and the small terms have an accumulator of
// their own. The tensor core truncates when it accumulates (nk_tc.cuh): the accumulators are read out every 256 k (32 accumulations), in small
// calls every 64 (gated_small; 24 x 515 x 900 20.5 -> 22.5 us, 16 x 4096 x 8192 would take 71 for 64), and added
// up in shared memory, rounding to nearest; where tensor memory has room for two sets the products go on meanwhile.
// Units of 32 k of all tiles form one sequence that the CTAs share evenly; a tile that several CTAs have a part of is finished by the last of
// them to arrive, which adds the parts in order (nobody waits; the same bits every time).
// Waits are bounded as everywhere: on expiry all roles run to the end without waiting, nothing is stored and the host reports NK_ERR_TIMEOUT.
#include "nk_gated.cuh"
#include "nk_tc.cuh"

namespace {

constexpr int NW_THREADS = 576, NW_PITCH = 20;   // PITCH: floats per column of a turned patch (conflict-free reads)
enum { NW_COLUMNS, NW_COLUMNS_ODD, NW_TURNED, NW_TURNED_ODD };   // n is the contiguous direction (by 16-byte vectors; element by element, or neither is); k is

struct NarrowCall {
    int fun;
    int64_t T, N, K;
    GatedMatrix w[2];          // [K, N]
    GatedMatrix out;           // [T, N]
    float *gate, *up;          // forward: row-major [T, N] or null
    int units, tiles_t, tiles;   // units of a tile (SUM: both weights'), tiles along the tokens, all tiles
    int chunk;                 // units between two readings of the accumulators, at least 1
    int64_t total;             // units of all tiles
    int64_t Kq;                // SUM: columns of a panel per weight, a multiple of a unit
    const float *x_hi, *x_lo;  // the tokens' panels, [T][pitch], hi and lo; SUM: the second weight's from Kq on
    int64_t pitch;
    float* parts;              // [CTA][2][NB][NT][128]
    int* tickets;              // [tiles]
    int* status;
};
template <int NT, bool SUM>
struct NarrowCfg {
    static constexpr int NB = SUM ? 1 : 2;
    static constexpr int UNIT = SUM ? 64 : 32;                    // k of a unit of work, which is a stage
    static constexpr int PANEL = NT * 64;                         // NT tokens x 16 k
    static constexpr int RING_BYTES = UNIT / 16 * 2 * PANEL;      // hi and lo of a stage's k
    static constexpr int RING = SUM && NT == 64 ? 3 : 4;
    static constexpr int RES = NB * NT * 128;                     // sums of a tile
    static constexpr int AHEAD = NT == 64 ? 2 : 3;                // patches of weights on their way, per warp
    static constexpr int PATCH = 32 * NW_PITCH;                   // floats
    static constexpr int NEEDS = 1024 + RING * RING_BYTES + RES * 4 + 16 * AHEAD * PATCH * 4 + 512;
    static constexpr int SMEM = NEEDS < 120 * 1024 ? 120 * 1024 : NEEDS;   // one CTA per SM: each takes all of its tensor memory
    static_assert(SMEM <= 227 * 1024, "more shared memory than a CTA can have");
    static constexpr int ACC = NB * 2 * NT;                       // columns of tensor memory that a set of accumulators takes
    static constexpr int AST = ACC <= 128 ? 3 : 2;                // stages of weights in tensor memory
    static constexpr int A0 = 512 - AST * 128;                    // their first column
    static constexpr int SETS = 2 * ACC <= A0 ? 2 : 1;
    static constexpr uint32_t ONE = (1u << 4) | (2u << 7) | (2u << 10) | (uint32_t(NT >> 3) << 17) | (uint32_t(128 >> 4) << 24);   // x lo or hi
    static constexpr uint32_t TWO = ONE + (uint32_t(NT >> 3) << 17);                                                                // x [hi | lo]
};
// the first unit of a CTA, and the CTA that has unit u
__device__ __forceinline__ int64_t nw_begin(int64_t cta, int64_t total, int64_t grid) { return cta * total / grid; }
__device__ __forceinline__ int64_t nw_cta(int64_t c, int64_t total, int64_t grid) { return ((c + 1) * grid - 1) / total; }

// Called by a whole warp, issued by one lane of it: the operands stay in uniform registers (from a branch of a single lane each product
// took 100 cycles to issue).
__device__ __forceinline__ void nw_mma(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n .reg .pred p, e;\n setp.ne.b32 p, %4, 0;\n elect.sync _|e, 0xffffffff;\n @e tcgen05.mma.cta_group::1.kind::tf32 [%0], [%1], %2, %3, p;\n}\n"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void nw_commit(uint64_t* bar) {
    unsigned a = (unsigned)__cvta_generic_to_shared(bar);
    asm volatile("{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(a) : "memory");
}
__device__ __forceinline__ void nw_st16(uint32_t taddr, const float (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};\n"
                 ::"r"(taddr), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]), "f"(v[10]),
                 "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15]) : "memory");
}
__device__ __forceinline__ void nw_ld8(uint32_t taddr, float (&v)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]) : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
}
__device__ __forceinline__ void nw_sync() { asm volatile("bar.sync 1, 512;\n" ::: "memory"); }   // the converters

// Sums that came out as NaN because of an infinity (tc_again says how), taken again by F32 multiply-adds: a whole warp, token t, four columns from n on per lane, whose
// sums are res[0..3] and (two products) res[second + 0..3].
template <bool SUM>
__device__ __noinline__ void nw_again(const NarrowCall& p, float* res, int second, int64_t t, int64_t n) {
    const int lane = threadIdx.x & 31;
    const float *hi = p.x_hi + t * p.pitch, *lo = p.x_lo + t * p.pitch;
    bool found = false;   // a NaN of the token's own spoils all its sums
    for (int64_t k = lane; k < (SUM ? p.Kq + p.K : p.K); k += 32) found = found || hi[k] != hi[k];
    if (__any_sync(0xffffffffu, found)) return;
    for (int i = 0; i < (SUM ? 4 : 8); i++) {   // sum by sum: what lives across the call in the caller's registers counts for more than the time of such calls
        float* at = res + (i & 3) + (i >> 2) * second;
        const int64_t c = n + (i & 3);
        const bool lost = c < p.N && *at != *at;
        if (!__any_sync(0xffffffffu, lost)) continue;
        float v = 0.0f;
        for (int b = SUM ? 0 : i >> 2; b < (SUM ? 2 : (i >> 2) + 1); b++) {
            const GatedMatrix& w = p.w[b];
            const float *column = static_cast<const float*>(w.ptr) + (lost ? c : 0) * w.cs, *x_hi = hi + (SUM && b ? p.Kq : 0), *x_lo = lo + (SUM && b ? p.Kq : 0);
            for (int64_t k0 = 0; k0 < p.K && __any_sync(0xffffffffu, lost && v == v); k0 += 64) {   // (NaN it is, else)
                const int kc = p.K - k0 < 64 ? int(p.K - k0) : 64;
#pragma unroll 4
                for (int k = 0; k < kc; k++) v = fmaf(x_hi[k0 + k] + x_lo[k0 + k], column[(k0 + k) * w.rs], v);
            }
        }
        if (lost) *at = v;
    }
}

template <int NT, bool SUM, int LAYOUT>
__global__ void __launch_bounds__(NW_THREADS, 1)
nk_gated_narrow_kernel(const __grid_constant__ CUtensorMap map_hi, const __grid_constant__ CUtensorMap map_lo, const __grid_constant__ NarrowCall p) {
    using C = NarrowCfg<NT, SUM>;
    extern __shared__ unsigned char nw_raw[];
    unsigned char* smem = nw_raw + ((1024u - ((unsigned)__cvta_generic_to_shared(nw_raw) & 1023u)) & 1023u);
    float* res = reinterpret_cast<float*>(smem + C::RING * C::RING_BYTES);       // [NB][NT][128]
    float* patches = res + C::RES;                                               // [converter warp][AHEAD]: columns [16 k][32], turned [32][NW_PITCH]
    uint64_t* bars = reinterpret_cast<uint64_t*>(patches + 16 * C::AHEAD * C::PATCH);
    uint64_t *b_full = bars, *b_free = bars + C::RING;                           // the tokens' panels
    uint64_t *a_full = bars + 2 * C::RING, *a_free = a_full + C::AST;            // [stage % AST]
    uint64_t *acc_full = a_free + C::AST, *acc_free = acc_full + 2;                   // [set]
    uint64_t* drain_bar = acc_free + 2;
    volatile int* abort_word = reinterpret_cast<volatile int*>(drain_bar + 1);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain_bar + 2);
    volatile int* last_word = reinterpret_cast<volatile int*>(drain_bar + 3);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < C::RING; i++) { nk_mbar_init(&b_full[i], 1); nk_mbar_init(&b_free[i], 1); }
        for (int i = 0; i < C::AST; i++) { nk_mbar_init(&a_full[i], 16); nk_mbar_init(&a_free[i], 1); }
        for (int i = 0; i < 2; i++) { nk_mbar_init(&acc_full[i], 1); nk_mbar_init(&acc_free[i], 16); }
        nk_mbar_init(drain_bar, 1);
        *abort_word = 0;
        nk_fence_barrier_init();
        nk_fence_proxy_async();
    }
    if (warp == 17) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"((unsigned)__cvta_generic_to_shared(tmem_slot)), "r"(TC_TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;   // set s of the accumulators at ACC s (of weight b: + 2 NT b), stage s at A0 + 128 (s % AST), 32 columns for each of four groups of warps

    bool dead = false;   // a wait ran out, here or elsewhere: this thread waits no more
    auto wait = [&](uint64_t* bar, unsigned parity) {
        if (dead) return false;
        const int r = nk_mbar_wait_bounded(bar, parity, NK_WAIT_LIMIT_NS, abort_word);
        if (r < 0) {
            *abort_word = 1;
            if (p.status) atomicExch(p.status, 1);
        }
        dead = r <= 0;
        return r > 0;
    };
    const int64_t u_begin = nw_begin(blockIdx.x, p.total, gridDim.x);
    const int count = int(nw_begin(int64_t(blockIdx.x) + 1, p.total, gridDim.x) - u_begin);   // units of this CTA
    // its units of one tile, [first, end), and of one chunk of them, [from, to)
    auto tile_end = [&](int first) {
        const unsigned u = unsigned(u_begin) + unsigned(first), e = (u / unsigned(p.units) + 1) * unsigned(p.units) - unsigned(u_begin);
        return e < unsigned(count) ? int(e) : count;
    };

    if (warp == 16) {
        if (lane == 0) {
            // ---- the tokens' panels, stage by stage (split by the launch before, beside which the weights' way may begin) ----
            asm volatile("griddepcontrol.wait;\n" ::: "memory");
            bool ok = true;
            int it = 0, tile = int(u_begin / p.units), j = int(u_begin % p.units), t0 = (tile % p.tiles_t) * NT;
            const int half = p.units / 2;
            for (int r = 0, phase = 1; it < count; it++) {
                ok = wait(&b_free[r], unsigned(phase));
                if (!ok) break;
                unsigned char* st = smem + r * C::RING_BYTES;
                nk_mbar_expect_tx(&b_full[r], C::RING_BYTES);
                const int k = SUM && j >= half ? int(p.Kq) + (j - half) * C::UNIT : j * C::UNIT;
                for (int h = 0; h < C::UNIT / 16; h++) {
                    nk_tma_load_2d(st + h * 2 * C::PANEL, &map_hi, &b_full[r], k + 16 * h, t0);
                    nk_tma_load_2d(st + h * 2 * C::PANEL + C::PANEL, &map_lo, &b_full[r], k + 16 * h, t0);
                }
                if (++r == C::RING) { r = 0; phase ^= 1; }
                if (++j == p.units) {
                    j = 0;
                    t0 = (++tile % p.tiles_t) * NT;
                }
            }
            if (!ok || *abort_word)   // copies already requested still land in shared memory
                for (int i = it > C::RING ? it - C::RING : 0; i < it; i++) nk_mbar_wait_bounded(&b_full[i % C::RING], (unsigned(i) / C::RING) & 1u, NK_WAIT_LIMIT_NS, nullptr);
        }
    } else if (warp == 17) {
        // ---- products, by the whole warp ----
        bool ok = true;
        unsigned chunk = 0, r = 0, r_phase = 0, as = 0, a_phase = 0;   // the slots of both rings that are due
        const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
        const uint64_t desc0 = tc_smem_desc((uint32_t)__cvta_generic_to_shared(smem));
        auto all_lanes = [&](bool mine) { return __all_sync(0xffffffffu, mine) != 0; };
        for (int first = 0, end; first < count && ok; first = end) {
            end = tile_end(first);
            for (int from = first; from < end && ok; from += p.chunk, chunk++) {
                const int to = from + p.chunk < end ? from + p.chunk : end;
                const unsigned set = C::SETS == 2 ? chunk & 1u : 0u, use = C::SETS == 2 ? chunk >> 1 : chunk;
                ok = all_lanes(wait(&acc_free[set], (use & 1u) ^ 1u));
#pragma unroll 1
                for (int s = from; s < to && ok; s++) {
                    ok = all_lanes(wait(&b_full[r], r_phase) && wait(&a_full[as], a_phase));
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t panels = desc0 + r * unsigned(C::RING_BYTES / 16);
                    const uint32_t a0 = tm + unsigned(C::A0) + 128u * as, acc0 = tm + set * unsigned(C::ACC);
#pragma unroll
                    for (int w = 0; w < 4; w++)       // the groups of warps: 2 g + b
#pragma unroll
                        for (int ks = 0; ks < 2; ks++) {
                            // w's 16 k among the stage's panels: forward g, of weight b; SUM 2 g + b, of the one weight
                            const uint32_t a = a0 + uint32_t(32 * w + 8 * ks), acc = acc0 + uint32_t(SUM ? 0 : (w & 1) * 2 * NT);
                            const uint64_t panel = panels + uint64_t(((SUM ? w : w >> 1) * 2 * C::PANEL + 32 * ks) / 16);
                            nw_mma(acc, a, panel, C::TWO, s > from || ks > 0 || w >= (SUM ? 1 : 2) ? 1u : 0u);
                            nw_mma(acc + uint32_t(NT), a + 16u, panel, C::ONE, 1u);
                        }
                    nw_commit(&a_free[as]);
                    nw_commit(&b_free[r]);
                    if (++as == unsigned(C::AST)) { as = 0; a_phase ^= 1u; }
                    if (++r == unsigned(C::RING)) { r = 0; r_phase ^= 1u; }
                    if (s == to - 1) nw_commit(&acc_full[set]);
                }
            }
        }
        if (!ok || *abort_word) {
            nw_commit(drain_bar);   // nothing may still run on the tensor cores at release time
            nk_mbar_wait_bounded(drain_bar, 0, NK_WAIT_LIMIT_NS, nullptr);
        }
    } else {
        // ---- converters ----
        bool waited = false;   // for the launch before: it clears the tickets
        const int g = warp >> 3, b = (warp >> 2) & 1, q = warp & 3;
        float* mine = patches + warp * C::AHEAD * C::PATCH;
        // What this warp fetches next: 32 columns x 16 k at `src`, k0 their first k, of unit `next`; worked out anew where a tile or a weight begins,
        // stepped along k in between. Element-wise: lane = column (turned: lanes across 16 k), sixteen accesses; by vectors four accesses,
        // across 32 columns of four k (turned: across 16 k of eight columns).
        const float* src = nullptr;
        int k0 = 0, next = 0, fresh_at = 0;   // fresh_at: the first unit that `src` does not lead to
        int64_t col0 = 0, along = 0, step_k = 0;   // the lane's first column; from access to access and from stage to stage
        const float* const src0 = static_cast<const float*>(p.w[0].ptr);   // an address for accesses that read nothing
        auto seek = [&]() {
            const unsigned u = unsigned(u_begin) + unsigned(next), tile = u / unsigned(p.units), j = u - tile * unsigned(p.units);
            const int half = p.units / 2, m = SUM ? int(j) >= half : b;
            const GatedMatrix& w = p.w[m];
            const int lane_col = LAYOUT == NW_COLUMNS ? (lane & 7) * 4 : LAYOUT == NW_COLUMNS_ODD ? lane : LAYOUT == NW_TURNED ? lane >> 2 : lane >> 4;
            const int lane_k = LAYOUT == NW_COLUMNS ? lane >> 3 : LAYOUT == NW_COLUMNS_ODD ? 0 : LAYOUT == NW_TURNED ? (lane & 3) * 4 : lane & 15;
            k0 = (SUM && m ? int(j) - half : int(j)) * C::UNIT + (SUM ? 2 * g + b : g) * 16 + lane_k;
            col0 = int64_t(tile / unsigned(p.tiles_t)) * 128 + 32 * q + lane_col;
            along = LAYOUT == NW_COLUMNS ? 4 * w.rs : LAYOUT == NW_COLUMNS_ODD ? w.rs : LAYOUT == NW_TURNED ? 8 * w.cs : 2 * w.cs;
            src = static_cast<const float*>(w.ptr) + col0 * w.cs + int64_t(k0) * w.rs;
            step_k = int64_t(C::UNIT) * w.rs;
            fresh_at = next + (SUM && !m ? half : p.units) - int(j);
        };
        // past the ends nothing is read and zeros arrive
        auto fetch = [&](float* to) {
            const float* at = src;
            if constexpr (LAYOUT == NW_COLUMNS) {
#pragma unroll
                for (int e = 0; e < 4; e++, at += along) {
                    const bool in = col0 < p.N && k0 + 4 * e < p.K;
                    nk_cp_async_16(to + (4 * e + (lane >> 3)) * 32 + (lane & 7) * 4, in ? at : src0, in ? 16 : 0);
                }
            } else if constexpr (LAYOUT == NW_COLUMNS_ODD) {
#pragma unroll
                for (int e = 0; e < 16; e++, at += along) {
                    const bool in = col0 < p.N && k0 + e < p.K;
                    nk_cp_async_4(to + e * 32 + lane, in ? at : src0, in ? 4 : 0);
                }
            } else if constexpr (LAYOUT == NW_TURNED) {
#pragma unroll
                for (int e = 0; e < 4; e++, at += along) {
                    const bool in = col0 + 8 * e < p.N && k0 < p.K;
                    nk_cp_async_16(to + (8 * e + (lane >> 2)) * NW_PITCH + (lane & 3) * 4, in ? at : src0, in ? 16 : 0);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 16; e++, at += along) {
                    const bool in = col0 + 2 * e < p.N && k0 < p.K;
                    nk_cp_async_4(to + (2 * e + (lane >> 4)) * NW_PITCH + (lane & 15), in ? at : src0, in ? 4 : 0);
                }
            }
            k0 += C::UNIT;
            src += step_k;
        };
        auto fetch_next = [&](float* to) {
            if (next < count) {
                if (next >= fresh_at) seek();
                fetch(to);
                next++;
            }
            nk_cp_async_commit();   // (an empty group where all is fetched: the waits count groups)
        };
#pragma unroll
        for (int a = 0; a < C::AHEAD; a++) fetch_next(mine + a * C::PATCH);
        int slot = 0, as = 0;      // the patch and the stage of tensor memory that are due
        unsigned a_phase = 1;
        // the next `n` stages
        auto convert = [&](int n) {
#pragma unroll 1
            for (; n > 0; n--) {
                float* patch = mine + slot * C::PATCH;
                nk_cp_async_wait<C::AHEAD - 1>();
                __syncwarp();
                float v[16];
                if constexpr (LAYOUT == NW_COLUMNS || LAYOUT == NW_COLUMNS_ODD) {
#pragma unroll
                    for (int e = 0; e < 16; e++) v[e] = patch[e * 32 + lane];
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float4 x = *reinterpret_cast<const float4*>(patch + lane * NW_PITCH + 4 * e);
                        v[4 * e] = x.x; v[4 * e + 1] = x.y; v[4 * e + 2] = x.z; v[4 * e + 3] = x.w;
                    }
                }
                __syncwarp();
                fetch_next(patch);
                slot = slot + 1 == C::AHEAD ? 0 : slot + 1;
                float hi[16], lo[16], check = 0.0f;
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    // to nearest, halves away from zero, like cvt.rna.tf32 -- which issues at a quarter of these operations' rate
                    hi[e] = __uint_as_float((__float_as_uint(v[e]) + 0x1000u) & 0xffffe000u);
                    const float rest = v[e] - hi[e];
                    check += rest;
                    lo[e] = __uint_as_float((__float_as_uint(rest) + 0x1000u) & 0xffffe000u);
                }
                if (!isfinite(check)) {   // something is not finite, or has been rounded past the largest finite value
#pragma unroll
                    for (int e = 0; e < 16; e++) tc_split(v[e], &hi[e], &lo[e]);
                }
                wait(&a_free[as], a_phase);
                __syncwarp();
                tc_fence_after();
                const uint32_t at = tmem + (uint32_t(32 * q) << 16) + uint32_t(C::A0 + 128 * as + 64 * g + 32 * b);
                nw_st16(at, hi);
                nw_st16(at + 16, lo);
                asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
                tc_fence_before();
                __syncwarp();
                if (lane == 0) nk_mbar_arrive(&a_full[as]);
                if (++as == C::AST) { as = 0; a_phase ^= 1u; }
            }
        };
        // A chunk's sums into shared memory, eight columns at a time; the four warps of a lane quarter share them.
        auto read_out = [&](unsigned chunk, bool fresh) {
            const unsigned set = C::SETS == 2 ? chunk & 1u : 0u, use = C::SETS == 2 ? chunk >> 1 : chunk;
            wait(&acc_full[set], use & 1u);
            __syncwarp();
            tc_fence_after();
#pragma unroll
            for (int k = 0; k < (C::NB * NT / 8 + 3) / 4; k++) {
                const int col = (4 * k + 2 * g + b) * 8;   // of NB * NT
                if (col >= C::NB * NT) break;
                const uint32_t at = tmem + (uint32_t(32 * q) << 16) + set * unsigned(C::ACC) + uint32_t(col / NT * 2 * NT + col % NT);
                float v[8], w[8];
                nw_ld8(at, v);
                nw_ld8(at + NT, w);
                float* to = res + col * 128 + 32 * q + lane;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float x = v[e] + w[e];
                    to[e * 128] = fresh ? x : to[e * 128] + x;
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) nk_mbar_arrive(&acc_free[set]);
        };
        // What is done with a tile when its last chunk of this CTA has been read out.
        auto close_tile = [&](int first, int end) {
            const int tile = int((u_begin + first) / p.units);
            // ---- the tile, or this CTA's part of it ----
            nw_sync();
            // four neighbouring columns of a token per access, VE of them per thread: e = t * 128 + n
            constexpr int VE = NT / 16;
            const int e0 = threadIdx.x * 4;
            const int64_t n0 = int64_t(tile / p.tiles_t) * 128;
            const int t0 = (tile % p.tiles_t) * NT;
            bool finish = end - first == p.units;
            if (!finish) {
                if (!waited) asm volatile("griddepcontrol.wait;\n" ::: "memory");
                waited = true;
                auto part_of = [&](int64_t cta) {   // a CTA's part of this tile: its first tile or not
                    return p.parts + (2 * cta + (nw_begin(cta, p.total, gridDim.x) / p.units == tile ? 0 : 1)) * int64_t(C::RES);
                };
                float* to = part_of(blockIdx.x);
#pragma unroll
                for (int k = 0; k < VE * C::NB; k++) *reinterpret_cast<float4*>(to + e0 + k * 2048) = *reinterpret_cast<const float4*>(res + e0 + k * 2048);
                const int64_t from = nw_cta(int64_t(tile) * p.units, p.total, gridDim.x), last = nw_cta((int64_t(tile) + 1) * p.units - 1, p.total, gridDim.x);
                __threadfence();
                nw_sync();
                if (threadIdx.x == 0) *last_word = atomicAdd(&p.tickets[tile], 1) == int(last - from);
                nw_sync();
                finish = *last_word;
                if (finish) {   // all parts, in order
                    __threadfence();
                    float4 v[VE * C::NB];
#pragma unroll
                    for (int k = 0; k < VE * C::NB; k++) v[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    for (int64_t cta = from; cta <= last; cta++) {
                        const float* part = part_of(cta);
                        float4 w[VE * C::NB];
#pragma unroll
                        for (int k = 0; k < VE * C::NB; k++) w[k] = __ldcg(reinterpret_cast<const float4*>(part + e0 + k * 2048));
#pragma unroll
                        for (int k = 0; k < VE * C::NB; k++) { v[k].x += w[k].x; v[k].y += w[k].y; v[k].z += w[k].z; v[k].w += w[k].w; }
                    }
#pragma unroll
                    for (int k = 0; k < VE * C::NB; k++) *reinterpret_cast<float4*>(res + e0 + k * 2048) = v[k];   // (this thread's own elements)
                }
            }
            if (__all_sync(0xffffffffu, finish && !*abort_word)) {   // (one answer per warp)
#pragma unroll 1
                for (int k = 0; k < VE; k++) {
                    const int e = e0 + k * 2048;
                    const int64_t t = t0 + (e >> 7), n = n0 + (e & 127);
                    if (t >= p.T) break;   // (a warp has one token)
                    bool lost = false;
#pragma unroll
                    for (int j = 0; j < 4; j++) lost = lost || (n + j < p.N && (res[e + j] != res[e + j] || (!SUM && res[C::RES / 2 + e + j] != res[C::RES / 2 + e + j])));
                    if (__any_sync(0xffffffffu, lost)) {
                        if (!waited) asm volatile("griddepcontrol.wait;\n" ::: "memory");   // for the panels
                        waited = true;
                        nw_again<SUM>(p, res + e, C::RES / 2, t, n);
                    }
                    float* o = static_cast<float*>(p.out.ptr) + t * p.out.rs + n * p.out.cs;
#pragma unroll 1
                    for (int j = 0; j < 4 && n + j < p.N; j++) {
                        const float v0 = res[e + j], v1 = SUM ? 0.0f : res[C::RES / 2 + e + j];
                        o[j * p.out.cs] = SUM ? v0 : gate_fun32(p.fun, v0) * v1;
                        if (!SUM && p.gate) { p.gate[t * p.N + n + j] = v0; p.up[t * p.N + n + j] = v1; }
                    }
                }
            }
            nw_sync();   // the sums have been read
        };
        // Chunk by chunk: the first two stages are delivered before the chunk before is read out, so that its last products and this work overlap.
        unsigned chunk = 0;
        int before_first = 0, before_end = 0;   // the tile of the chunk before, where that was its last one
        bool before_fresh = false;
        for (int first = 0, end; first < count; first = end) {
            end = tile_end(first);
            for (int from = first; from < end; from += p.chunk, chunk++) {
                const int to = from + p.chunk < end ? from + p.chunk : end;
                const int n = to - from, head = n < 2 ? n : 2;
                convert(head);
                if (chunk > 0) {
                    read_out(chunk - 1, before_fresh);
                    if (before_end > 0) close_tile(before_first, before_end);
                }
                convert(n - head);
                before_fresh = from == first;
                before_first = first;
                before_end = to == end ? end : 0;
            }
        }
        read_out(chunk - 1, before_fresh);
        close_tile(before_first, before_end);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 17) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(TC_TMEM_COLS) : "memory");
    }
}

int narrow_tokens(int64_t T) { return T <= 16 ? 16 : T <= 32 ? 32 : 64; }
int narrow_unit(bool sum) { return sum ? NarrowCfg<16, true>::UNIT : NarrowCfg<16, false>::UNIT; }
void narrow_tiles(NarrowCall* p, bool sum, bool small) {
    const int64_t nt = narrow_tokens(p->T);
    const int64_t unit = narrow_unit(sum);
    p->units = int((p->K + unit - 1) / unit) * (sum ? 2 : 1);
    p->tiles_t = int((p->T + nt - 1) / nt);
    p->tiles = int((p->N + 127) / 128) * p->tiles_t;
    p->total = int64_t(p->tiles) * p->units;
    p->chunk = int((small ? 64 : 256) / unit);
    p->Kq = (p->K + unit - 1) / unit * unit;
}
// at least four units per CTA: a tile's parts cost what there are of them
int narrow_grid(const nk_ctx* ctx, const NarrowCall& p) {
    const int64_t most = (p.total + 3) / 4;
    return int(most < ctx->prop.multiProcessorCount ? most : ctx->prop.multiProcessorCount);
}
size_t narrow_part_bytes(const nk_ctx* ctx, const NarrowCall& p, bool sum) { return size_t(narrow_grid(ctx, p)) * 2 * (sum ? 1 : 2) * narrow_tokens(p.T) * 128 * 4; }

template <int NT, bool SUM, int LAYOUT>
int narrow_launch(nk_ctx* ctx, NarrowCall p, const float* hi, const float* lo, int64_t cols) {
    using C = NarrowCfg<NT, SUM>;
    CUtensorMap map_hi, map_lo;
    if (nk_tma_encode_2d_f32(hi, uint64_t(p.T), uint64_t(cols), uint64_t(cols) * 4, 16, NT, 2, &map_hi) ||
        nk_tma_encode_2d_f32(lo, uint64_t(p.T), uint64_t(cols), uint64_t(cols) * 4, 16, NT, 2, &map_lo))
        return nk_fail(ctx, NK_ERR_CUDA, "nk_gated: the driver has no tensor-map encoder");
    auto* kern = nk_gated_narrow_kernel<NT, SUM, LAYOUT>;
    NK_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    p.x_hi = hi;
    p.x_lo = lo;
    p.pitch = cols;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(unsigned(narrow_grid(ctx, p)));
    cfg.blockDim = dim3(NW_THREADS);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, map_hi, map_lo, p);
    if (e != cudaSuccess) return nk_cuda_fail(ctx, e, "nk_gated_narrow_kernel");
    return nk_after_launch(ctx, "nk_gated_narrow_kernel");
}
template <int NT, bool SUM>
int narrow_layout(nk_ctx* ctx, const NarrowCall& p, const float* hi, const float* lo, int64_t cols) {
    bool turned = true, vec_n = p.N % 4 == 0, vec_k = p.K % 4 == 0;
    for (const GatedMatrix& w : p.w) {
        const bool aligned = reinterpret_cast<uintptr_t>(w.ptr) % 16 == 0;
        turned = turned && w.rs == 1 && w.cs != 1;
        vec_n = vec_n && aligned && w.cs == 1 && w.rs % 4 == 0;
        vec_k = vec_k && aligned && w.rs == 1 && w.cs % 4 == 0;
    }
    if (turned) return vec_k ? narrow_launch<NT, SUM, NW_TURNED>(ctx, p, hi, lo, cols) : narrow_launch<NT, SUM, NW_TURNED_ODD>(ctx, p, hi, lo, cols);
    return vec_n ? narrow_launch<NT, SUM, NW_COLUMNS>(ctx, p, hi, lo, cols) : narrow_launch<NT, SUM, NW_COLUMNS_ODD>(ctx, p, hi, lo, cols);
}
template <bool SUM>
int narrow(nk_ctx* ctx, const NarrowCall& p, const float* hi, const float* lo, int64_t cols) {
    switch (narrow_tokens(p.T)) {
        case 16: return narrow_layout<16, SUM>(ctx, p, hi, lo, cols);
        case 32: return narrow_layout<32, SUM>(ctx, p, hi, lo, cols);
        default: return narrow_layout<64, SUM>(ctx, p, hi, lo, cols);
    }
}

}  // namespace

bool nk_gated_narrow(const nk_ctx* ctx, const GatedCall& c) {
    // Up to three tiles of 64 tokens: every tile reads the weights again (64 tokens 80 us at 4096 x 8192), where panels of them (nk_gated_tc.cu) cost
    // their split, 150 us there, and 1.1 us per token.
    if (c.T > 192 || c.D < 16 || c.H < 16) return false;
    const int64_t most = int64_t(1) << 30;
    return c.D < most && c.H < most && double(c.D) * double(c.H) < 4e12 && size_t(NarrowCfg<64, false>::SMEM) <= size_t(ctx->prop.sharedMemPerBlockOptin);
}

int nk_gated_narrow_forward(nk_ctx* ctx, const GatedCall& c) {
    NarrowCall p;
    memset(&p, 0, sizeof(p));
    p.fun = c.fun;
    p.T = c.T;
    p.N = c.H;
    p.K = c.D;
    p.w[0] = c.w[0];
    p.w[1] = c.w[1];
    p.out = c.y;
    p.gate = static_cast<float*>(c.gate);
    p.up = static_cast<float*>(c.up);
    p.status = ctx->tma_status_dev;
    narrow_tiles(&p, false, gated_small(c));
    const int64_t Kp = tc_round_k(c.D);
    auto pad = [](size_t b) { return (b + 1023) / 1024 * 1024; };
    const size_t x_bytes = pad(size_t(c.T) * Kp * 4), part_bytes = pad(narrow_part_bytes(ctx, p, false));
    NkWorkspace ws(ctx);
    int st = ws.get(2 * x_bytes + part_bytes + size_t(p.tiles) * sizeof(int));
    if (st) return st;
    char* base = static_cast<char*>(ws.ptr);
    float *hi = reinterpret_cast<float*>(base), *lo = reinterpret_cast<float*>(base + x_bytes);
    p.parts = reinterpret_cast<float*>(base + 2 * x_bytes);
    p.tickets = reinterpret_cast<int*>(base + 2 * x_bytes + part_bytes);
    TcSplit sp;
    memset(&sp, 0, sizeof(sp));
    sp.op[0].src = static_cast<const float*>(c.x.ptr);
    sp.op[0].R = c.T; sp.op[0].sR = c.x.rs; sp.op[0].K = c.D; sp.op[0].sK = c.x.cs;
    tc_operand_layout(&sp.op[0], c.x.cs == 1, hi, lo, Kp);
    sp.tickets = p.tickets;
    sp.n_tickets = p.tiles;
    nk_tc_split_kernel<<<unsigned(sp.op[0].tiles), 256, 0, ctx->stream>>>(sp);
    if ((st = nk_after_launch(ctx, "nk_tc_split_kernel"))) return st;
    return narrow<false>(ctx, p, hi, lo, Kp);
}

int64_t nk_gated_narrow_columns(int64_t H) { return (H + narrow_unit(true) - 1) / narrow_unit(true) * narrow_unit(true); }
static NarrowCall narrow_dx_call(nk_ctx* ctx, const GatedCall& c) {
    NarrowCall p;
    memset(&p, 0, sizeof(p));
    p.T = c.T;
    p.N = c.D;
    p.K = c.H;
    for (int b = 0; b < 2; b++) p.w[b] = GatedMatrix{c.w[b].ptr, c.w[b].cs, c.w[b].rs};
    p.out = c.dx;
    p.status = ctx->tma_status_dev;
    narrow_tiles(&p, true, gated_small(c));
    return p;
}
void nk_gated_narrow_dx_needs(nk_ctx* ctx, const GatedCall& c, size_t* part_bytes, int* tickets) {
    const NarrowCall p = narrow_dx_call(ctx, c);
    *part_bytes = narrow_part_bytes(ctx, p, true);
    *tickets = p.tiles;
}
int nk_gated_narrow_dx_panels(nk_ctx* ctx, const GatedCall& c, const float* hi, const float* lo, float* parts, int* tickets) {
    NarrowCall p = narrow_dx_call(ctx, c);
    p.parts = parts;
    p.tickets = tickets;
    return narrow<true>(ctx, p, hi, lo, 2 * p.Kq);
}
int nk_gated_narrow_dx(nk_ctx* ctx, const GatedCall& c, const float* dg, const float* du) {
    const NarrowCall p = narrow_dx_call(ctx, c);
    auto pad = [](size_t b) { return (b + 1023) / 1024 * 1024; };
    const size_t e_bytes = pad(size_t(c.T) * 2 * p.Kq * 4), part_bytes = pad(narrow_part_bytes(ctx, p, true));
    NkWorkspace ws(ctx);
    int st = ws.get(2 * e_bytes + part_bytes + size_t(p.tiles) * sizeof(int));
    if (st) return st;
    char* base = static_cast<char*>(ws.ptr);
    float *hi = reinterpret_cast<float*>(base), *lo = reinterpret_cast<float*>(base + e_bytes);
    int* tickets = reinterpret_cast<int*>(base + 2 * e_bytes + part_bytes);
    TcSplit sp;
    memset(&sp, 0, sizeof(sp));
    int64_t tiles = 0;
    for (int b = 0; b < 2; b++) {
        TcOperand& o = sp.op[b];
        o.src = b ? du : dg;
        o.R = c.T; o.sR = c.H; o.K = c.H; o.sK = 1;
        tc_operand_layout(&o, true, hi + b * p.Kq, lo + b * p.Kq, 2 * p.Kq, p.Kq);
        tiles += o.tiles;
    }
    sp.tickets = tickets;
    sp.n_tickets = p.tiles;
    nk_tc_split_kernel<<<unsigned(tiles), 256, 0, ctx->stream>>>(sp);
    if ((st = nk_after_launch(ctx, "nk_tc_split_kernel"))) return st;
    return nk_gated_narrow_dx_panels(ctx, c, hi, lo, reinterpret_cast<float*>(base + 2 * e_bytes), tickets);
}
