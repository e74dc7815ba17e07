// The gated block in F32 for some tokens (more than the streaming kernels take, fewer than fill a tile's rows): tensor cores, with the weights read
// from memory once and never laid out anew.
//
//   forward:  R_b[n, t] = sum_k w_b[k, n] x[t, k], out = f(R_0) * R_1         dx ("SUM"):  R[n, t] = sum_b sum_k w_b[k, n] x_b[t, k], out = R
//
// The weights are the product's A operand: 128 columns n are the rows of the tensor core's tile, the tokens (padded to 16, 32 or 64) its columns.
// A 3xTF32 product needs hi and lo of every weight; writing them to memory and reading them back would move five times the weights' bytes
// (nk_gated_tc.cu does, where a panel is used by many tiles). Here a warp loads 32 columns x 16 k into registers, splits them there and stores hi
// and lo into tensor memory, from where tcgen05.mma takes its A operand; shared memory only carries the tokens' panels (TMA, split before:
// they are small). What is left is the stream of weights: 4 bytes per element against 6 multiply-adds per token.
//
// Roles, 18 warps: 0..15 converters in two groups, warp 16 fetches the tokens' panels, warp 17 issues the products. A group works on every second
// chunk of 128 k. Within a group, warp w serves lanes 32 (w % 4) of the tile; its two halves take the two weights (forward), or the two halves of a
// stage's 32 k (SUM). A stage is 64 columns of tensor memory (2 x (16 hi + 16 lo)), two per group; loads run two stages ahead in registers.
// The tensor core truncates when it accumulates (nk_tc.cuh), so an accumulator is read out after every chunk and added up in shared memory, rounding
// to nearest. Chunks of all tiles form one sequence that the CTAs share evenly; a tile that several CTAs have a part of is finished by the
// last of them to arrive, which adds the parts in order (nobody waits; the same bits every time).
// Waits are bounded as everywhere: on expiry all roles run to the end without waiting, nothing is stored and the host reports NK_ERR_TIMEOUT.
#include "nk_gated.cuh"
#include "nk_tc.cuh"

namespace {

constexpr int NW_THREADS = 576, NW_CONV = 512, NW_RING = 4, NW_PITCH = 20;   // PITCH: of a row in a warp's transposing buffer
constexpr int NW_CHUNK = 128;
enum { NW_COLUMNS, NW_TURNED, NW_TURNED_ODD };   // n is the contiguous direction, or neither; k is, in 16-byte vectors; k is, element by element

struct NarrowCall {
    int fun;
    int64_t T, N, K;
    GatedMatrix w[2];          // [K, N]
    GatedMatrix out;           // [T, N]
    float *gate, *up;          // forward: row-major [T, N] or null
    int chunks, tiles_t, tiles;   // chunks of a tile (SUM: both weights'), tiles along the tokens, all tiles
    int64_t total;             // chunks of all tiles
    int64_t Kq;                // SUM: columns of a panel per weight, a multiple of NW_CHUNK
    float* parts;              // [CTA][2][NB][NT][128]
    int* tickets;              // [tiles]
    int* status;
};
template <int NT, bool SUM>
struct NarrowCfg {
    static constexpr int NB = SUM ? 1 : 2;
    static constexpr int STAGES = SUM ? 4 : 8;                    // of a chunk
    static constexpr int PANEL = NT * 64;                         // NT tokens x 16 k
    static constexpr int RING_BYTES = (SUM ? 4 : 2) * PANEL;      // hi and lo of 16 (SUM: 32) k
    static constexpr int RES = NB * NT * 128;                     // sums of a tile
    static constexpr int NEEDS = 1024 + NW_RING * RING_BYTES + 2 * RES * 4 + 16 * 32 * NW_PITCH * 4 + 512;
    static constexpr int SMEM = NEEDS < 120 * 1024 ? 120 * 1024 : NEEDS;   // one CTA per SM: each takes all of its tensor memory
    static constexpr uint32_t IDESC = (1u << 4) | (2u << 7) | (2u << 10) | (uint32_t(NT >> 3) << 17) | (uint32_t(128 >> 4) << 24);
};
// the CTA that has chunk c, and the first chunk of a CTA
__device__ __forceinline__ int64_t nw_begin(int64_t cta, int64_t total, int64_t grid) { return cta * total / grid; }
__device__ __forceinline__ int64_t nw_cta(int64_t c, int64_t total, int64_t grid) { return ((c + 1) * grid - 1) / total; }

__device__ __forceinline__ void nw_mma(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::tf32 [%0], [%1], %2, %3, p;\n}\n"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void nw_st16(uint32_t taddr, const float (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};\n"
                 ::"r"(taddr), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]), "f"(v[10]),
                 "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15]) : "memory");
}
__device__ __forceinline__ void nw_sync() { asm volatile("bar.sync 1, 512;\n" ::: "memory"); }   // the converters

template <int NT, bool SUM, int LAYOUT>
__global__ void __launch_bounds__(NW_THREADS, 1)
nk_gated_narrow_kernel(const __grid_constant__ CUtensorMap map_hi, const __grid_constant__ CUtensorMap map_lo, const __grid_constant__ NarrowCall p) {
    using C = NarrowCfg<NT, SUM>;
    extern __shared__ unsigned char nw_raw[];
    unsigned char* smem = nw_raw + ((1024u - ((unsigned)__cvta_generic_to_shared(nw_raw) & 1023u)) & 1023u);
    float* res = reinterpret_cast<float*>(smem + NW_RING * C::RING_BYTES);       // [group][NB][NT][128]
    float* turn = res + 2 * C::RES;                                              // [converter warp][32][NW_PITCH]
    uint64_t* bars = reinterpret_cast<uint64_t*>(turn + 16 * 32 * NW_PITCH);
    uint64_t *b_full = bars, *b_free = bars + NW_RING;                           // the tokens' panels
    uint64_t *a_full = bars + 2 * NW_RING, *a_free = a_full + 4;                 // [group][stage]
    uint64_t *acc_full = a_free + 4, *drain_bar = acc_full + 2;                  // [group]
    volatile int* abort_word = reinterpret_cast<volatile int*>(drain_bar + 1);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain_bar + 2);
    volatile int* last_word = reinterpret_cast<volatile int*>(drain_bar + 3);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < NW_RING; i++) { nk_mbar_init(&b_full[i], 1); nk_mbar_init(&b_free[i], 1); }
        for (int i = 0; i < 4; i++) { nk_mbar_init(&a_full[i], 8); nk_mbar_init(&a_free[i], 1); }
        for (int i = 0; i < 2; i++) nk_mbar_init(&acc_full[i], 1);
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
    const uint32_t tmem = *tmem_slot;   // group g: accumulators at 256 g (+ NT for the second), stage s at 256 g + 128 + 64 s

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
    const int64_t c_begin = nw_begin(blockIdx.x, p.total, gridDim.x);
    const int count = int(nw_begin(int64_t(blockIdx.x) + 1, p.total, gridDim.x) - c_begin);   // chunks of this CTA
    // its chunks of one tile, [first, end): the groups take them in turn, beginning with group 0 (all roles step through the same pairs)
    auto tile_end = [&](int first) {
        const int64_t e = ((c_begin + first) / p.chunks + 1) * p.chunks - c_begin;
        return e < count ? int(e) : count;
    };

    if (warp == 16) {
        if (lane == 0) {
            // ---- the tokens' panels, in the order the products need them ----
            bool ok = true;
            int it = 0;
            for (int first = 0, end; first < count && ok; first = end) {
                end = tile_end(first);
                for (int step = 0; step < (end - first + 1) / 2 * C::STAGES && ok; step++) {
                    const int pair = first + 2 * (step / C::STAGES), s = step % C::STAGES;
                    for (int i = pair; i < pair + 2 && i < end && ok; i++, it++) {
                        const int r = it % NW_RING;
                        ok = wait(&b_free[r], ((unsigned(it) / NW_RING) & 1u) ^ 1u);
                        if (!ok) break;
                        const int64_t c = c_begin + i;
                        const int tile = int(c / p.chunks), j = int(c % p.chunks), t0 = (tile % p.tiles_t) * NT;
                        unsigned char* st = smem + r * C::RING_BYTES;
                        nk_mbar_expect_tx(&b_full[r], C::RING_BYTES);
                        if (SUM) {
                            const int half = p.chunks / 2, k0 = (j >= half ? int(p.Kq) + (j - half) * NW_CHUNK : j * NW_CHUNK) + s * 32;
                            for (int h = 0; h < 2; h++) {
                                nk_tma_load_2d(st + h * 2 * C::PANEL, &map_hi, &b_full[r], k0 + 16 * h, t0);
                                nk_tma_load_2d(st + h * 2 * C::PANEL + C::PANEL, &map_lo, &b_full[r], k0 + 16 * h, t0);
                            }
                        } else {
                            nk_tma_load_2d(st, &map_hi, &b_full[r], j * NW_CHUNK + s * 16, t0);
                            nk_tma_load_2d(st + C::PANEL, &map_lo, &b_full[r], j * NW_CHUNK + s * 16, t0);
                        }
                    }
                }
            }
            if (!ok || *abort_word)   // copies already requested still land in shared memory
                for (int i = it > NW_RING ? it - NW_RING : 0; i < it; i++) nk_mbar_wait_bounded(&b_full[i % NW_RING], (unsigned(i) / NW_RING) & 1u, NK_WAIT_LIMIT_NS, nullptr);
        }
    } else if (warp == 17) {
        if (lane == 0) {
            // ---- products: per stage two blocks of 16 k (of the two weights, or of one), each 2 x 8 k, three products (small terms first) ----
            bool ok = true;
            int it = 0, stage[2] = {0, 0};
            for (int first = 0, end; first < count && ok; first = end) {
                end = tile_end(first);
                for (int step = 0; step < (end - first + 1) / 2 * C::STAGES && ok; step++) {
                    const int pair = first + 2 * (step / C::STAGES), s = step % C::STAGES;
                    for (int i = pair; i < pair + 2 && i < end && ok; i++, it++) {
                        const int g = i - pair, r = it % NW_RING, as = stage[g] & 1;
                        ok = wait(&b_full[r], (unsigned(it) / NW_RING) & 1u) && wait(&a_full[2 * g + as], (unsigned(stage[g]) >> 1) & 1u);
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t sb = (uint32_t)__cvta_generic_to_shared(smem + r * C::RING_BYTES), a0 = tmem + uint32_t(256 * g + 128 + 64 * as);
#pragma unroll
                        for (int b = 0; b < 2; b++) {
                            const uint32_t acc = tmem + uint32_t(256 * g + (SUM ? 0 : b * NT));
#pragma unroll
                            for (int ks = 0; ks < 2; ks++) {
                                const uint32_t a = a0 + uint32_t(32 * b + 8 * ks), panel = sb + uint32_t((SUM ? b * 2 * C::PANEL : 0) + 32 * ks);
                                const uint64_t hi = tc_smem_desc(panel), lo = tc_smem_desc(panel + C::PANEL);
                                nw_mma(acc, a + 16, hi, C::IDESC, (s > 0 || ks > 0 || (SUM && b > 0)) ? 1u : 0u);
                                nw_mma(acc, a, lo, C::IDESC, 1u);
                                nw_mma(acc, a, hi, C::IDESC, 1u);
                            }
                        }
                        tc_commit<1>(&a_free[2 * g + as]);
                        tc_commit<1>(&b_free[r]);
                        if (s == C::STAGES - 1) tc_commit<1>(&acc_full[g]);
                        stage[g]++;
                    }
                }
            }
            if (!ok || *abort_word) {
                tc_commit<1>(drain_bar);   // nothing may still run on the tensor cores at release time
                nk_mbar_wait_bounded(drain_bar, 0, NK_WAIT_LIMIT_NS, nullptr);
            }
        }
    } else {
        // ---- converters ----
        const int g = warp >> 3, b = (warp >> 2) & 1, q = warp & 3;
        float* buf = turn + warp * 32 * NW_PITCH;
        float pf[2][16];
        // 32 columns x 16 k of stage s of chunk i: columns: lane = column, one k per element; turned: see below
        auto fetch = [&](int i, int s, float (&v)[16]) {
            const int64_t c = c_begin + i;
            const int tile = int(c / p.chunks), j = int(c % p.chunks);
            int m, k0;
            if (SUM) {
                m = j >= p.chunks / 2;
                k0 = (m ? j - p.chunks / 2 : j) * NW_CHUNK + s * 32 + b * 16;
            } else {
                m = b;
                k0 = j * NW_CHUNK + s * 16;
            }
            const int64_t n = int64_t(tile / p.tiles_t) * 128 + 32 * q;
            const GatedMatrix& w = p.w[m];
            const float* src = static_cast<const float*>(w.ptr);
            if constexpr (LAYOUT == NW_COLUMNS) {
                const float* at = src + (n + lane) * w.cs + int64_t(k0) * w.rs;
                if (n + lane < p.N && k0 + 16 <= p.K) {
#pragma unroll
                    for (int e = 0; e < 16; e++, at += w.rs) v[e] = __ldcs(at);
                } else {
#pragma unroll
                    for (int e = 0; e < 16; e++) v[e] = n + lane < p.N && k0 + e < p.K ? __ldcs(at + e * w.rs) : 0.0f;
                }
            } else if constexpr (LAYOUT == NW_TURNED) {   // four lanes across 16 k, eight columns per access
                const int k = k0 + (lane & 3) * 4;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int64_t col = n + 8 * e + (lane >> 2);
                    const float4 x = col < p.N && k < p.K ? __ldcs(reinterpret_cast<const float4*>(src + col * w.cs + k)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    v[4 * e] = x.x; v[4 * e + 1] = x.y; v[4 * e + 2] = x.z; v[4 * e + 3] = x.w;
                }
            } else {                                      // sixteen lanes across 16 k, two columns per access
                const int k = k0 + (lane & 15);
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const int64_t col = n + 2 * e + (lane >> 4);
                    v[e] = col < p.N && k < p.K ? __ldcs(src + col * w.cs + k) : 0.0f;
                }
            }
        };
        // ... to lane = column
        auto arrange = [&](float (&v)[16]) {
            if constexpr (LAYOUT == NW_COLUMNS) return;
            __syncwarp();
            if constexpr (LAYOUT == NW_TURNED) {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    *reinterpret_cast<float4*>(buf + (8 * e + (lane >> 2)) * NW_PITCH + (lane & 3) * 4) = make_float4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
            } else {
#pragma unroll
                for (int e = 0; e < 16; e++) buf[(2 * e + (lane >> 4)) * NW_PITCH + (lane & 15)] = v[e];
            }
            __syncwarp();
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float4 x = *reinterpret_cast<const float4*>(buf + lane * NW_PITCH + 4 * e);
                v[4 * e] = x.x; v[4 * e + 1] = x.y; v[4 * e + 2] = x.z; v[4 * e + 3] = x.w;
            }
        };
        // this group's stages, one after the other; the fetches run ahead of the tile that is being worked on
        int next_end = tile_end(0), next = g, next_stage = 0, next_first = 0;
        auto skip = [&] {   // to a tile that has a chunk for this group
            while (next >= next_end && next_end < count) {
                next_first = next_end;
                next_end = tile_end(next_first);
                next = next_first + g;
            }
        };
        skip();
        auto fetch_next = [&](float (&v)[16]) {
            if (next >= next_end) return;   // all fetched
            fetch(next, next_stage, v);
            if (++next_stage == C::STAGES) {
                next_stage = 0;
                next += 2;
                skip();
            }
        };
        fetch_next(pf[0]);
        fetch_next(pf[1]);
        int step = 0, chunk = 0;   // stages and chunks of this group so far
        for (int first = 0, end; first < count; first = end) {
            end = tile_end(first);
            const int tile = int((c_begin + first) / p.chunks);
            for (int i = first + g; i < end; i += 2, chunk++) {
#pragma unroll 1
                for (int s = 0; s < C::STAGES; s += 2) {
#pragma unroll
                    for (int u = 0; u < 2; u++, step++) {
                        arrange(pf[u]);
                        float hi[16], lo[16], check = 0.0f;
#pragma unroll
                        for (int e = 0; e < 16; e++) {
                            unsigned h, l;
                            asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(h) : "f"(pf[u][e]));
                            hi[e] = __uint_as_float(h);
                            asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(l) : "f"(pf[u][e] - hi[e]));
                            lo[e] = __uint_as_float(l);
                            check += lo[e];
                        }
                        if (!isfinite(check)) {   // something is not finite, or rounds past the largest finite value
#pragma unroll
                            for (int e = 0; e < 16; e++) tc_split(pf[u][e], &hi[e], &lo[e]);
                        }
                        fetch_next(pf[u]);
                        wait(&a_free[2 * g + u], ((unsigned(step) >> 1) & 1u) ^ 1u);
                        __syncwarp();
                        tc_fence_after();
                        const uint32_t at = tmem + (uint32_t(32 * q) << 16) + uint32_t(256 * g + 128 + 64 * u + 32 * b);
                        nw_st16(at, hi);
                        nw_st16(at + 16, lo);
                        asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) nk_mbar_arrive(&a_full[2 * g + u]);
                    }
                }
                // the chunk's sums into shared memory (SUM: the group's halves share the one accumulator's columns)
                wait(&acc_full[g], unsigned(chunk) & 1u);
                __syncwarp();
                tc_fence_after();
                constexpr int DC = SUM && NT >= 32 ? NT / 2 : NT;
                if (!SUM || NT >= 32 || b == 0) {
                    const bool fresh = i < first + 2;   // the group's first chunk of this tile
#pragma unroll
                    for (int c0 = 0; c0 < DC; c0 += 16) {
                        uint32_t v[16];
                        const int col = SUM ? (NT >= 32 ? b * DC : 0) + c0 : c0;
                        tc_ld16(tmem + (uint32_t(32 * q) << 16) + uint32_t(256 * g + (SUM ? 0 : b * NT) + col), v);
                        float* to = res + g * C::RES + ((SUM ? 0 : b * NT) + col) * 128 + 32 * q + lane;
#pragma unroll
                        for (int e = 0; e < 16; e++) to[e * 128] = fresh ? __uint_as_float(v[e]) : to[e * 128] + __uint_as_float(v[e]);
                    }
                }
                tc_fence_before();
            }
            // ---- the tile, or this CTA's part of it ----
            nw_sync();
            auto sum_at = [&](int e) { return end - first >= 2 ? res[e] + res[C::RES + e] : res[e]; };
            const int64_t n0 = int64_t(tile / p.tiles_t) * 128;
            const int t0 = (tile % p.tiles_t) * NT;
            auto store = [&](int e, float v0, float v1) {   // element e = t * 128 + n of the tile
                const int64_t t = t0 + (e >> 7), n = n0 + (e & 127);
                if (t >= p.T || n >= p.N) return;
                float* o = static_cast<float*>(p.out.ptr) + t * p.out.rs + n * p.out.cs;
                if (SUM) { *o = v0; return; }
                *o = gate_fun<float>(p.fun, false, v0) * v1;
                if (p.gate) { p.gate[t * p.N + n] = v0; p.up[t * p.N + n] = v1; }
            };
            if (end - first == p.chunks) {
                if (!*abort_word)
                    for (int e = threadIdx.x; e < NT * 128; e += NW_CONV) store(e, sum_at(e), SUM ? 0.0f : sum_at(C::RES - NT * 128 + e));
            } else {
                auto slot = [&](int64_t cta) {   // a CTA's part of this tile: its first tile or not
                    return p.parts + (2 * cta + (nw_begin(cta, p.total, gridDim.x) / p.chunks == tile ? 0 : 1)) * int64_t(C::RES);
                };
                float* mine = slot(blockIdx.x);
                for (int e = threadIdx.x; e < C::RES; e += NW_CONV) mine[e] = sum_at(e);
                const int64_t from = nw_cta(int64_t(tile) * p.chunks, p.total, gridDim.x), to = nw_cta((int64_t(tile) + 1) * p.chunks - 1, p.total, gridDim.x);
                __threadfence();
                nw_sync();
                if (threadIdx.x == 0) *last_word = atomicAdd(&p.tickets[tile], 1) == int(to - from);
                nw_sync();
                if (*last_word && !*abort_word) {
                    __threadfence();
                    for (int e = threadIdx.x; e < NT * 128; e += NW_CONV) {
                        float v0 = 0.0f, v1 = 0.0f;
                        for (int64_t cta = from; cta <= to; cta++) {
                            const float* part = slot(cta);
                            v0 += __ldcg(part + e);
                            if (!SUM) v1 += __ldcg(part + NT * 128 + e);
                        }
                        store(e, v0, v1);
                    }
                }
            }
            nw_sync();   // the sums have been read
        }
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
void narrow_tiles(NarrowCall* p, bool sum) {
    const int64_t nt = narrow_tokens(p->T);
    p->chunks = int((p->K + NW_CHUNK - 1) / NW_CHUNK) * (sum ? 2 : 1);
    p->tiles_t = int((p->T + nt - 1) / nt);
    p->tiles = int((p->N + 127) / 128) * p->tiles_t;
    p->total = int64_t(p->tiles) * p->chunks;
    p->Kq = (p->K + NW_CHUNK - 1) / NW_CHUNK * NW_CHUNK;
}
int narrow_grid(const nk_ctx* ctx, const NarrowCall& p) { return int(p.total < ctx->prop.multiProcessorCount ? p.total : ctx->prop.multiProcessorCount); }
size_t narrow_part_bytes(const nk_ctx* ctx, const NarrowCall& p, bool sum) { return size_t(narrow_grid(ctx, p)) * 2 * (sum ? 1 : 2) * narrow_tokens(p.T) * 128 * 4; }

template <int NT, bool SUM, int LAYOUT>
int narrow_launch(nk_ctx* ctx, const NarrowCall& p, const float* hi, const float* lo, int64_t cols) {
    using C = NarrowCfg<NT, SUM>;
    CUtensorMap map_hi, map_lo;
    if (nk_tma_encode_2d_f32(hi, uint64_t(p.T), uint64_t(cols), uint64_t(cols) * 4, 16, NT, 2, &map_hi) ||
        nk_tma_encode_2d_f32(lo, uint64_t(p.T), uint64_t(cols), uint64_t(cols) * 4, 16, NT, 2, &map_lo))
        return nk_fail(ctx, NK_ERR_CUDA, "nk_gated: the driver has no tensor-map encoder");
    auto* kern = nk_gated_narrow_kernel<NT, SUM, LAYOUT>;
    NK_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    kern<<<narrow_grid(ctx, p), NW_THREADS, C::SMEM, ctx->stream>>>(map_hi, map_lo, p);
    return nk_after_launch(ctx, "nk_gated_narrow_kernel");
}
template <int NT, bool SUM>
int narrow_layout(nk_ctx* ctx, const NarrowCall& p, const float* hi, const float* lo, int64_t cols) {
    bool turned = true, vec = p.K % 4 == 0;
    for (const GatedMatrix& w : p.w) {
        turned = turned && w.rs == 1 && w.cs != 1;
        vec = vec && w.cs % 4 == 0 && reinterpret_cast<uintptr_t>(w.ptr) % 16 == 0;
    }
    if (!turned) return narrow_launch<NT, SUM, NW_COLUMNS>(ctx, p, hi, lo, cols);
    return vec ? narrow_launch<NT, SUM, NW_TURNED>(ctx, p, hi, lo, cols) : narrow_launch<NT, SUM, NW_TURNED_ODD>(ctx, p, hi, lo, cols);
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
    if (c.T > 64) return false;
    const int64_t most = int64_t(1) << 30;
    return c.D < most && c.H < most && size_t(NarrowCfg<64, false>::SMEM) <= size_t(ctx->prop.sharedMemPerBlockOptin);
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
    narrow_tiles(&p, false);
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

int64_t nk_gated_narrow_columns(int64_t H) { return (H + NW_CHUNK - 1) / NW_CHUNK * NW_CHUNK; }
static NarrowCall narrow_dx_call(nk_ctx* ctx, const GatedCall& c) {
    NarrowCall p;
    memset(&p, 0, sizeof(p));
    p.T = c.T;
    p.N = c.D;
    p.K = c.H;
    for (int b = 0; b < 2; b++) p.w[b] = GatedMatrix{c.w[b].ptr, c.w[b].cs, c.w[b].rs};
    p.out = c.dx;
    p.status = ctx->tma_status_dev;
    narrow_tiles(&p, true);
    return p;
}
void nk_gated_narrow_dx_needs(nk_ctx* ctx, const GatedCall& c, size_t* part_bytes, int* tickets) {
    const NarrowCall p = narrow_dx_call(ctx, c);
    *part_bytes = narrow_part_bytes(ctx, p, true);
    *tickets = p.tiles;
}
int nk_gated_narrow_dx(nk_ctx* ctx, const GatedCall& c, const float* hi, const float* lo, float* parts, int* tickets) {
    NarrowCall p = narrow_dx_call(ctx, c);
    p.parts = parts;
    p.tickets = tickets;
    return narrow<true>(ctx, p, hi, lo, 2 * p.Kq);
}
