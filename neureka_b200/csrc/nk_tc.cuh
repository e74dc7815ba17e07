// F32 products on the 5th-generation tensor cores with the 3xTF32 split: the machinery of nk_conv_tc.cu (contraction-shaped convolutions) and
// nk_gated_tc.cu (the gated block). Every unit that includes it instantiates what it launches.
//
// 3xTF32. A TF32 operand keeps 11 significant bits, an F32 value 24. Every operand element v is split once into
// hi = tf32(v) (round to nearest) and lo = tf32(v - hi) (v - hi is exact in F32), and the product sum is evaluated as
// sum(lo_a*hi_b) + sum(hi_a*lo_b) + sum(hi_a*hi_b) with F32 accumulation in tensor memory: the dropped lo*lo term and
// the rounding of lo are below 2^-21 of |a||b| per term, inside the 1e-5 * sum|a||b| tolerance of the path. Sums with infinite operands: tc_again.
//
// Two shapes of the kernel, chosen by estimated time (tc_shape):
//   * pairs of CTAs (cta_group::2), tile 256 x 256: each CTA stages 128 rows of A and 128 of B, 32 KiB per 16 k where a lone
//     CTA with a 128 x 256 tile stages 48. Six products of 128 x 256 x 8 take 768 cycles; the lone CTA moved 48 KiB in and
//     72 KiB out of its shared memory per stage in that time, more than the 128 bytes per cycle there are, the pair 32 + 48.
//     4096^3: 554 us, lone CTAs 596;
//   * lone CTAs, tile 128 x 128, for products with too few large tiles to fill the chip; where even these are too few, k is
//     split over several CTAs per tile: each warp leaves its part of the tile in scratch and takes a ticket, the warp that
//     draws the last one adds the parts in split order (nobody waits; the result does not depend on the order of arrival).
//
// Accumulation. The tensor core adds each product block into the accumulator with truncation (measured: a sum of K
// same-signed terms came out low by K/8 * 3 * 2^-25 relative, 9e-5 at K = 8192). A tile's sum over k is therefore cut
// into chunks of 128 k (48 accumulations, bias below 1.5e-6; a caller may ask for shorter ones): the two accumulators alternate chunk by chunk, and the
// sixteen epilogue warps add every finished chunk into per-thread F32 running sums with ordinary round-to-nearest adds
// while the next chunk's products already run into the other accumulator. The running sums of a tile (a quarter of its
// columns per thread) go to the drain after its last chunk.
// Eighteen warps leave 96 registers a thread (five warps share a register file). A thread of the pair form holds 64 sums, and its store spills: 4 bytes a
// thread for the plain drain, 200 to 680 for the block's, once per tile; the lone form fits.
// Every mbarrier wait is bounded (nk_mbar_wait_bounded); on expiry the waiter raises the CTA's abort word and the
// host-visible status, all roles leave their loops, outstanding copies and tensor-core work are waited for (bounded),
// tensor memory is released and the kernel returns; the host then reports NK_ERR_TIMEOUT.
#pragma once
#include <cuda.h>

#include "nk_internal.h"
#include "nk_ptx.cuh"

int nk_tma_encode_2d_f32(const void* base, uint64_t rows, uint64_t cols, uint64_t pitch_bytes, int box_cols, int box_rows, int swizzle,
                         CUtensorMap* out);

namespace {

constexpr int TC_BM = 128, TC_BK = 16;                        // rows of A a CTA stages, k per stage
constexpr int TC_THREADS = 576;                              // warp 0 producer, warp 1 tensor-core issue, warps 2..17 epilogue
constexpr unsigned TC_TMEM_COLS = 512;                       // all of it: two accumulators of up to 128 x 256 F32 per CTA
constexpr int TC_KC = 8;                                     // k blocks (of 16) per accumulation chunk (a caller may want fewer)
constexpr int TC_MAX_SPLITS = 16;

// CG: CTAs that share a tile (1 or 2); BN: columns of the tile
template <int CG, int BN>
struct TcCfg {
    static constexpr int TM = TC_BM * CG;                    // rows of the tile
    static constexpr int B_ROWS = BN / CG;                   // rows of B (columns of the tile) a CTA stages
    static constexpr int A_PART = TC_BM * TC_BK * 4;         // 8 KiB: one of A_hi / A_lo for a stage
    static constexpr int B_PART = B_ROWS * TC_BK * 4;
    static constexpr int STAGE_BYTES = 2 * A_PART + 2 * B_PART;   // 32 KiB for both shapes in use
    static constexpr int STAGES = 192 * 1024 / STAGE_BYTES;
    static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 1024 /* alignment slack */ + 256 /* barriers */;
    static constexpr int EPI_COLS = BN / 4;                  // accumulator columns an epilogue warp owns (4 warps per lane quarter)
    // Instruction descriptor: F32 accumulate, TF32 x TF32, both operands K-major
    static constexpr uint32_t IDESC = (1u << 4) | (2u << 7) | (2u << 10) | (uint32_t(BN >> 3) << 17) | (uint32_t(TM >> 4) << 24);
};

// ---- split: v -> hi = tf32(v), lo = tf32(v - hi) ------------------------------------------------------------------------
__device__ __forceinline__ void tc_split(float v, float* hi, float* lo) {
    unsigned h;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(h) : "f"(v));
    float fh = __uint_as_float(h);
    if (!isfinite(fh)) fh = isfinite(v) ? __uint_as_float(__float_as_uint(v) & 0xffffe000u) : v;   // rounded past the largest finite value
    float r = isfinite(v) ? v - fh : 0.0f;
    unsigned l;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(l) : "f"(r));
    *hi = fh;
    *lo = __uint_as_float(l);
}

// One operand of the split: element (r, k) is src[offR(r) + offK(k)], the offsets a stride or (index groups of several dims) a table.
struct TcOperand {
    const float* src;             // the view's base
    const int64_t *offR, *offK;   // null: r * sR, k * sK
    int64_t sR, sK, R, K, Kp;     // Kp: columns of the panel, a multiple of 16, zero from K on
    int64_t pitch;                // of a row of hi and lo; Kp unless several operands lie side by side along k
    int64_t tiles;                // CTAs for this operand
    int kfast;                    // consecutive k are consecutive in memory
    int vec;                      // 16-byte loads along the contiguous direction are legal (and there are no tables)
    float *hi, *lo;
};
constexpr int TC_OPERANDS = 3;
struct TcSplit {
    TcOperand op[TC_OPERANDS];    // tiles = 0: none
    int* tickets;
    int n_tickets;
};
inline int64_t tc_round_k(int64_t k) { return (k + TC_BK - 1) / TC_BK * TC_BK; }
// src, offsets, strides, R and K are there; the rest follows. kfast: the operand's contiguous direction is k. columns: Kp, where more of a panel than
// up to the next multiple of 16 has to be zero.
inline void tc_operand_layout(TcOperand* o, bool kfast, float* hi, float* lo, int64_t pitch, int64_t columns = 0) {
    o->Kp = columns ? columns : tc_round_k(o->K);
    o->pitch = pitch;
    o->hi = hi;
    o->lo = lo;
    o->kfast = kfast;
    o->tiles = kfast ? ((o->R + 31) / 32) * ((o->Kp + 127) / 128) : ((o->R + 127) / 128) * ((o->Kp + 31) / 32);
    const int64_t fast = kfast ? o->sK : o->sR, slow = kfast ? o->sR : o->sK;
    o->vec = !o->offR && fast == 1 && slow % 4 == 0 && (reinterpret_cast<uintptr_t>(o->src) % 16) == 0;
}
// Gathers the operands into hi / lo [R][pitch], zero for K <= k < Kp. A CTA takes 32 x 128 elements, 128 along the operand's contiguous
// direction (rows x k, or -- turned through shared memory on the way -- k x rows), four 16-byte loads per thread in flight
// and 16-byte stores; operands that 16-byte loads do not fit are read element by element. All operands in one launch: the
// second's tiles follow the first's. Bound by memory: 12 bytes move per element.
// 4096^2 operands, two per product: 62 us (58 is the floor); two launches of 32 x 32 tiles with 4-byte accesses: 87 to 114.
__global__ void __launch_bounds__(256) nk_tc_split_kernel(const TcSplit p) {
    __shared__ float tile[32][129];
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");   // a launch that allows it may begin what does not need these panels
    int which = 0;
    int64_t t = blockIdx.x;
    while (which + 1 < TC_OPERANDS && t >= p.op[which].tiles) t -= p.op[which++].tiles;
    const TcOperand& o = p.op[which];
    if (p.n_tickets && blockIdx.x == 0)
        for (int i = threadIdx.x; i < p.n_tickets; i += 256) p.tickets[i] = 0;
    const int64_t tiles_k = (o.Kp + (o.kfast ? 127 : 31)) / (o.kfast ? 128 : 32);
    const int64_t k0 = (t % tiles_k) * (o.kfast ? 128 : 32), r0 = (t / tiles_k) * (o.kfast ? 32 : 128);
    auto at = [&](int64_t r, int64_t k) { return (o.offR ? o.offR[r] : r * o.sR) + (o.offK ? o.offK[k] : k * o.sK); };
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float v[4][4];
    // lane: 4 consecutive elements of the contiguous direction; warp + 8 i: the other direction
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int64_t slow = (o.kfast ? r0 : k0) + warp + 8 * i, fast = (o.kfast ? k0 : r0) + lane * 4;
        const int64_t slow_end = o.kfast ? o.R : o.K, fast_end = o.kfast ? o.K : o.R;
        if (o.vec && slow < slow_end && fast + 4 <= fast_end) {
            *reinterpret_cast<float4*>(v[i]) = __ldcs(reinterpret_cast<const float4*>(o.src + (o.kfast ? at(slow, fast) : at(fast, slow))));
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) v[i][e] = slow < slow_end && fast + e < fast_end ? o.src[o.kfast ? at(slow, fast + e) : at(fast + e, slow)] : 0.0f;
        }
    }
    int64_t row[4], k;
    if (o.kfast) {
        k = k0 + lane * 4;
#pragma unroll
        for (int i = 0; i < 4; i++) row[i] = r0 + warp + 8 * i;
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) tile[warp + 8 * i][lane * 4 + e] = v[i][e];
        __syncthreads();
        // eight lanes cover the 32 k of a row, four rows per warp and step
        k = k0 + (lane & 7) * 4;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = (lane >> 3) + 4 * (warp + 8 * i);
            row[i] = r0 + r;
#pragma unroll
            for (int e = 0; e < 4; e++) v[i][e] = tile[(lane & 7) * 4 + e][r];
        }
    }
    if (k >= o.Kp) return;   // Kp is a multiple of 16: whole vectors from here on
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (row[i] >= o.R) continue;
        float h[4], l[4];
#pragma unroll
        for (int e = 0; e < 4; e++) tc_split(v[i][e], &h[e], &l[e]);
        *reinterpret_cast<float4*>(o.hi + row[i] * o.pitch + k) = make_float4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<float4*>(o.lo + row[i] * o.pitch + k) = make_float4(l[0], l[1], l[2], l[3]);
    }
}

// ---- tcgen05 wrappers ------------------------------------------------------------------------------------------------
// Shared-memory operand descriptor, K-major, 64-byte swizzle: rows of 64 bytes (16 F32), 8-row groups 512 bytes apart.
__device__ __forceinline__ uint64_t tc_smem_desc(uint32_t saddr) {
    uint64_t d = 0;
    d |= uint64_t((saddr & 0x3ffffu) >> 4);     // start address, 16-byte units
    d |= uint64_t(1) << 16;                     // leading byte offset: not used by swizzled K-major layouts
    d |= uint64_t(512 >> 4) << 32;              // stride byte offset between 8-row groups
    d |= uint64_t(1) << 46;                     // descriptor version of this architecture
    d |= uint64_t(4) << 61;                     // layout type: 64-byte swizzle
    return d;
}
template <int CG>
__device__ __forceinline__ void tc_mma(uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accumulate) {
    if (CG == 2)
        asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::tf32 [%0], %1, %2, %3, p;\n}\n"
                     ::"r"(tmem_d), "l"(da), "l"(db), "r"(idesc), "r"(accumulate) : "memory");
    else
        asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::tf32 [%0], %1, %2, %3, p;\n}\n"
                     ::"r"(tmem_d), "l"(da), "l"(db), "r"(idesc), "r"(accumulate) : "memory");
}
// Arrives on the mbarrier (of both CTAs of a pair) once every tcgen05.mma issued so far by this thread has completed.
template <int CG>
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
    unsigned a = (unsigned)__cvta_generic_to_shared(bar);
    if (CG == 2)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n"
                     ::"r"(a), "h"((unsigned short)3) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(a) : "memory");
}
// the shared::cluster address of an mbarrier's counterpart in the pair's first CTA, which issues the products
__device__ __forceinline__ unsigned tc_leader_bar(uint64_t* bar) {
    unsigned a = (unsigned)__cvta_generic_to_shared(bar), r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;\n" : "=r"(r) : "r"(a));
    return r;
}
__device__ __forceinline__ void tc_arrive_cluster(unsigned bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(bar) : "memory");
}
// 2-D tile load of one CTA of a pair into its own shared memory, reporting to the leader's mbarrier
__device__ __forceinline__ void tc_load_pair(void* smem, const void* tensor_map, unsigned leader_bar, int c0, int c1) {
    unsigned d = (unsigned)__cvta_generic_to_shared(smem);
    unsigned long long m = reinterpret_cast<unsigned long long>(tensor_map);
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n"
                 ::"r"(d), "l"(m), "r"(c0), "r"(c1), "r"(leader_bar) : "memory");
}
__device__ __forceinline__ void tc_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
// 16 consecutive accumulator columns of this thread's lane (32 lanes x 32 bits per warp and column)
__device__ __forceinline__ void tc_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                   "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
}

struct TcParams {
    int64_t M;
    int k_blocks;                  // Kp / 16
    int tiles_m;
    int64_t units;                 // tiles * splits; unit u is part u % splits of tile u / splits
    int splits, kb_per;            // k blocks per part
    int chunk;                     // k blocks per accumulation chunk
    const float *a[2], *b[4];      // the panels, hi and lo of A and of each B, rows of Kp: what tc_again reads
    int64_t N, Kp;                 // rows of B
    float* parts;                  // splits > 1: [tile][part][warp of 16][columns / 4][32 rows x 4]
    int* tickets;                  // splits > 1: [tile][warp of 16]
    int* status;                   // host-mapped word, set non-zero when a bounded wait ran out
};
// The operands' tensor maps: hi and lo of A, then of each B.
template <bool DUAL>
struct TcMaps {
    CUtensorMap a[2], b[DUAL ? 4 : 2];
};

// What becomes of a tile's sums. A drain is called by whole warps (rows past
// the last among them). One with DUAL = false takes a thread's row m and 32-column groups of its EC columns from n0 on. With
// DUAL = true there are two B operands of one shape, a tile is BN / 2 columns of each product, and a thread holds its row's columns [n0, n0 + EC / 2)
// of the first product and then of the second.
struct TcPlainDrain {
    static constexpr bool DUAL = false;
    float* out;
    int64_t M, N;
    const int64_t *offOm, *offOn;  // null: m * sOm, n * sOn
    int64_t sOm, sOn, bO;
    int out_vec;                   // the drain's n index is its contiguous direction and every row starts 16-byte aligned
    template <int EC>
    __device__ __forceinline__ void store(int64_t m, int64_t n0, const float (&sum)[EC]) const {
        if (m >= M) return;
        const int64_t row = bO + (offOm ? offOm[m] : m * sOm);
#pragma unroll
        for (int c = 0; c < EC / 32; c++) {
            const int64_t n = n0 + c * 32;
            if (n >= N) continue;
            if (out_vec && n + 32 <= N) {
                float4* dst = reinterpret_cast<float4*>(out + row + n);
#pragma unroll
                for (int j = 0; j < 8; j++) dst[j] = make_float4(sum[c * 32 + 4 * j], sum[c * 32 + 4 * j + 1], sum[c * 32 + 4 * j + 2], sum[c * 32 + 4 * j + 3]);
            } else {
#pragma unroll
                for (int j = 0; j < 32; j++)
                    if (n + j < N) out[row + (offOn ? offOn[n + j] : (n + j) * sOn)] = sum[c * 32 + j];
            }
        }
    }
};

// An infinity's lo is 0 and its products with the other operand's low bits are NaN (0) or of either sign, so three products give NaN where the sum of
// hi + lo is infinite. Sums that come out as NaN are taken again, by F32 multiply-adds over the panels: sum[j] of a thread is that of its row m and column n0 + j
// (two B operands: the first half of the second one's). Called by a whole warp, which shares the work of each; rows and columns with a NaN
// of their own, which spoil all their sums, are found first.
template <int EC, bool DUAL>
__device__ __noinline__ void tc_again(const TcParams& p, float* sum, int64_t m, int64_t n0) {
    constexpr int COLS = DUAL ? EC / 2 : EC;
    const int lane = threadIdx.x & 31;
    auto has_nan = [&](const float* row) {
        bool found = false;
        for (int64_t k = lane * 4; k - lane * 4 < p.Kp && !found; k += 128) {
            const float4 v = k < p.Kp ? *reinterpret_cast<const float4*>(row + k) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            found = __any_sync(0xffffffffu, v.x != v.x || v.y != v.y || v.z != v.z || v.w != v.w);
        }
        return found;
    };
    auto columns = [&](int j) { return n0 + j % COLS < p.N; };
    bool mine = false;
    for (int j = 0; j < EC; j++) mine = mine || (columns(j) && sum[j] != sum[j]);
    mine = mine && m < p.M;
    for (unsigned rows = __ballot_sync(0xffffffffu, mine); rows; rows &= rows - 1) {
        const int r = __ffs(int(rows)) - 1;
        const bool spoilt = has_nan(p.a[0] + __shfl_sync(0xffffffffu, m, r) * p.Kp);
        if (lane == r) mine = !spoilt;
    }
    for (int j = 0; j < EC; j++) {
        unsigned rows = __ballot_sync(0xffffffffu, mine && columns(j) && sum[j] != sum[j]);
        if (!rows) continue;
        const int which = DUAL ? 2 * (j / COLS) : 0;
        const int64_t column = (n0 + j % COLS) * p.Kp;
        const float *b_hi = p.b[which] + column, *b_lo = p.b[which + 1] + column;
        if (has_nan(b_hi)) continue;
        for (; rows; rows &= rows - 1) {
            const int r = __ffs(int(rows)) - 1;
            const int64_t row = __shfl_sync(0xffffffffu, m, r) * p.Kp;
            const float *a_hi = p.a[0] + row, *a_lo = p.a[1] + row;
            float v = 0.0f;
            bool done = false;
            for (int64_t k0 = 0; k0 < p.Kp && !done; k0 += 128) {
                const int64_t k = k0 + lane * 4;
                if (k < p.Kp) {   // (Kp is a multiple of 16)
                    const float4 x = *reinterpret_cast<const float4*>(a_hi + k), y = *reinterpret_cast<const float4*>(a_lo + k);
                    const float4 z = *reinterpret_cast<const float4*>(b_hi + k), w = *reinterpret_cast<const float4*>(b_lo + k);
                    v = fmaf(x.x + y.x, z.x + w.x, v);
                    v = fmaf(x.y + y.y, z.y + w.y, v);
                    v = fmaf(x.z + y.z, z.z + w.z, v);
                    v = fmaf(x.w + y.w, z.w + w.w, v);
                }
                done = __any_sync(0xffffffffu, v != v);   // (NaN it is)
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
            if (lane == r) sum[j] = v;
        }
    }
}

template <int CG, int BN, class Drain>
__global__ void __launch_bounds__(TC_THREADS, 1)
nk_conv_tc_kernel(const __grid_constant__ TcMaps<Drain::DUAL> maps, const __grid_constant__ TcParams p, const __grid_constant__ Drain drain) {
    constexpr bool DUAL = Drain::DUAL;
    constexpr int COLS = DUAL ? BN / 2 : BN;   // columns of a drain that a tile covers
    using C = TcCfg<CG, BN>;
    constexpr int STAGES = C::STAGES, EC = C::EPI_COLS;
    extern __shared__ unsigned char tc_smem_raw[];
    // stages must start on a 1024-byte boundary (swizzle pattern = function of the address bits); the dynamic block of both CTAs
    // of a pair starts at the same offset, so the pair's panels and barriers lie at the same offsets too
    unsigned char* smem = tc_smem_raw + ((1024u - ((unsigned)__cvta_generic_to_shared(tc_smem_raw) & 1023u)) & 1023u);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + STAGES * C::STAGE_BYTES);
    uint64_t* full_bar = bars;                      // [STAGES] a stage's panels have landed (a pair's: in both CTAs; the leader's is used)
    uint64_t* empty_bar = bars + STAGES;            // [STAGES] the products reading a stage have completed
    uint64_t* acc_full = bars + 2 * STAGES;         // [2] an accumulator holds a finished chunk
    uint64_t* acc_empty = bars + 2 * STAGES + 2;    // [2] the epilogue (of both CTAs) has read it out; the leader's is used
    uint64_t* drain_bar = bars + 2 * STAGES + 4;    // only on the abort path: all issued products have completed
    volatile int* abort_word = reinterpret_cast<volatile int*>(bars + 2 * STAGES + 5);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 6);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = CG == 2 ? int(blockIdx.x & 1u) : 0;              // the cluster is (2, 1, 1): rank = index inside it
    const int64_t unit0 = CG == 2 ? blockIdx.x >> 1 : blockIdx.x, unit_step = CG == 2 ? gridDim.x >> 1 : gridDim.x;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; s++) { nk_mbar_init(&full_bar[s], 1); nk_mbar_init(&empty_bar[s], 1); }
        for (int b = 0; b < 2; b++) { nk_mbar_init(&acc_full[b], 1); nk_mbar_init(&acc_empty[b], 16 * CG); }
        nk_mbar_init(drain_bar, 1);
        *abort_word = 0;
        nk_fence_barrier_init();
        nk_fence_proxy_async();
    }
    if (warp == 1) {   // one warp allocates all of the SM's tensor memory (one CTA per SM: 192 KiB of shared memory each)
        unsigned slot = (unsigned)__cvta_generic_to_shared(tmem_slot);
        if (CG == 2) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(slot), "r"(TC_TMEM_COLS) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(slot), "r"(TC_TMEM_COLS) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
        }
    }
    tc_fence_before();
    __syncthreads();
    if (CG == 2) tc_cluster_sync();   // the peer's barriers are initialised and both allocations made
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    auto wait_or_abort = [&](uint64_t* bar, unsigned parity) -> bool {
        const int r = nk_mbar_wait_bounded(bar, parity, NK_WAIT_LIMIT_NS, abort_word);
        if (r < 0) {
            *abort_word = 1;
            if (p.status) atomicExch(p.status, 1);
        }
        return r > 0;
    };
    // the k blocks of a unit
    auto range = [&](int64_t u, int* kb_begin, int* kb_end) {
        const int part = p.splits > 1 ? int(u % p.splits) : 0;
        *kb_begin = part * p.kb_per;
        *kb_end = *kb_begin + p.kb_per < p.k_blocks ? *kb_begin + p.kb_per : p.k_blocks;
    };

    if (warp == 0) {
        if (lane == 0) {
            // ---- producer: four (two B operands in a lone CTA: six) tensor copies per stage; of a pair, each CTA's producer fetches its own rows ----
            int it = 0;
            bool ok = true;
            for (int64_t u = unit0; u < p.units && ok; u += unit_step) {
                const int64_t t = p.splits > 1 ? u / p.splits : u;
                int kb_begin, kb_end;
                range(u, &kb_begin, &kb_end);
                const int m0 = int(t % p.tiles_m) * C::TM + rank * TC_BM, n0 = int(t / p.tiles_m) * COLS + (DUAL ? 0 : rank * C::B_ROWS);
                for (int kb = kb_begin; kb < kb_end && ok; kb++, it++) {
                    const int s = it % STAGES;
                    ok = wait_or_abort(&empty_bar[s], ((unsigned(it) / STAGES) & 1u) ^ 1u);
                    if (!ok) break;
                    unsigned char* st = smem + size_t(s) * C::STAGE_BYTES;
                    if (rank == 0) nk_mbar_expect_tx(&full_bar[s], unsigned(CG * C::STAGE_BYTES));
                    const int k0 = kb * TC_BK;
                    unsigned char* sb = st + 2 * C::A_PART;
                    if (CG == 2) {
                        // two B operands: the pair's first CTA stages the first one's columns, the second CTA the second one's
                        const unsigned bar = tc_leader_bar(&full_bar[s]);
                        tc_load_pair(st, &maps.a[0], bar, k0, m0);
                        tc_load_pair(st + C::A_PART, &maps.a[1], bar, k0, m0);
                        tc_load_pair(sb, &maps.b[DUAL ? 2 * rank : 0], bar, k0, n0);
                        tc_load_pair(sb + C::B_PART, &maps.b[DUAL ? 2 * rank + 1 : 1], bar, k0, n0);
                    } else {
                        nk_tma_load_2d(st, &maps.a[0], &full_bar[s], k0, m0);
                        nk_tma_load_2d(st + C::A_PART, &maps.a[1], &full_bar[s], k0, m0);
                        nk_tma_load_2d(sb, &maps.b[0], &full_bar[s], k0, n0);
                        nk_tma_load_2d(sb + C::B_PART, &maps.b[1], &full_bar[s], k0, n0);
                        if constexpr (DUAL) {   // half the rows from either
                            nk_tma_load_2d(sb + C::B_PART / 2, &maps.b[2], &full_bar[s], k0, n0);
                            nk_tma_load_2d(sb + C::B_PART + C::B_PART / 2, &maps.b[3], &full_bar[s], k0, n0);
                        }
                    }
                }
            }
            if ((!ok || *abort_word) && rank == 0) {
                // copies already requested still land in shared memory: wait for them (bounded); of a pair, the leader's
                // barriers count both CTAs' bytes and neither leaves before the cluster barrier at the end
                for (int j = (it > STAGES ? it - STAGES : 0); j < it; j++)
                    nk_mbar_wait_bounded(&full_bar[j % STAGES], (unsigned(j) / STAGES) & 1u, NK_WAIT_LIMIT_NS, nullptr);
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            // ---- tensor-core issue: per stage two k-steps of 8, three products each (small terms first); a new
            // accumulator every p.chunk stages ----
            int it = 0, ch = 0;
            bool ok = true;
            for (int64_t u = unit0; u < p.units && ok; u += unit_step) {
                int kb_begin, kb_end;
                range(u, &kb_begin, &kb_end);
                for (int kb0 = kb_begin; kb0 < kb_end && ok; kb0 += p.chunk, ch++) {
                    const int b = ch & 1;
                    ok = wait_or_abort(&acc_empty[b], ((unsigned(ch) >> 1) & 1u) ^ 1u);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t acc = tmem_base + uint32_t(b) * BN;
                    const int kb1 = kb0 + p.chunk < kb_end ? kb0 + p.chunk : kb_end;
                    for (int kb = kb0; kb < kb1 && ok; kb++, it++) {
                        const int s = it % STAGES;
                        ok = wait_or_abort(&full_bar[s], (unsigned(it) / STAGES) & 1u);
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t sa = (uint32_t)__cvta_generic_to_shared(smem + size_t(s) * C::STAGE_BYTES);
#pragma unroll
                        for (int ks = 0; ks < TC_BK / 8; ks++) {
                            const uint32_t koff = uint32_t(ks) * 32u;   // 8 F32 further along the 64-byte row
                            const uint64_t a_hi = tc_smem_desc(sa + koff), a_lo = tc_smem_desc(sa + C::A_PART + koff);
                            const uint64_t b_hi = tc_smem_desc(sa + 2 * C::A_PART + koff), b_lo = tc_smem_desc(sa + 2 * C::A_PART + C::B_PART + koff);
                            tc_mma<CG>(acc, a_lo, b_hi, C::IDESC, (kb > kb0 || ks != 0) ? 1u : 0u);
                            tc_mma<CG>(acc, a_hi, b_lo, C::IDESC, 1u);
                            tc_mma<CG>(acc, a_hi, b_hi, C::IDESC, 1u);
                        }
                        tc_commit<CG>(&empty_bar[s]);   // the stage goes back to the producer(s) when these products are done
                    }
                    if (ok) tc_commit<CG>(&acc_full[b]);    // ... and the chunk to the epilogue(s)
                }
            }
            if (!ok || *abort_word) {
                tc_commit<CG>(drain_bar);           // nothing of this CTA may still run on the tensor cores at release time
                nk_mbar_wait_bounded(drain_bar, 0, NK_WAIT_LIMIT_NS, nullptr);
            }
        }
    } else {
        // ---- epilogue: warps 2..17; warp w reads the 32 accumulator lanes of its quarter (w % 4) and the columns of
        // part (w - 2) / 4, adds every finished chunk into its running sums and stores them after the tile's last chunk ----
        const int q = warp & 3, quarter = (warp - 2) >> 2;
        const unsigned empty_leader[2] = {CG == 2 ? tc_leader_bar(&acc_empty[0]) : 0u, CG == 2 ? tc_leader_bar(&acc_empty[1]) : 0u};
        int ch = 0;
        bool ok = true;
        for (int64_t u = unit0; u < p.units && ok; u += unit_step) {
            const int64_t t = p.splits > 1 ? u / p.splits : u;
            int kb_begin, kb_end;
            range(u, &kb_begin, &kb_end);
            const int64_t m = int64_t(t % p.tiles_m) * C::TM + rank * TC_BM + q * 32 + lane;
            const int64_t n0 = int64_t(t / p.tiles_m) * COLS + quarter * (DUAL ? EC / 2 : EC);
            float sum[EC];
            for (int kb0 = kb_begin; kb0 < kb_end && ok; kb0 += p.chunk, ch++) {
                const int b = ch & 1;
                ok = __all_sync(0xffffffffu, wait_or_abort(&acc_full[b], (unsigned(ch) >> 1) & 1u));   // the lanes go on, or leave, together
                if (!ok) break;
                tc_fence_after();
                const uint32_t src = tmem_base + (uint32_t(q * 32) << 16) + uint32_t(b) * BN + uint32_t(quarter) * (DUAL ? EC / 2 : EC);
#pragma unroll
                for (int c = 0; c < EC / 16; c++) {
                    uint32_t v[16];
                    tc_ld16(src + uint32_t(c) * 16u + (DUAL && c >= EC / 32 ? uint32_t(COLS - EC / 2) : 0u), v);
                    if (kb0 == kb_begin) {
#pragma unroll
                        for (int j = 0; j < 16; j++) sum[c * 16 + j] = __uint_as_float(v[j]);
                    } else {
#pragma unroll
                        for (int j = 0; j < 16; j++) sum[c * 16 + j] += __uint_as_float(v[j]);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (CG == 2) tc_arrive_cluster(empty_leader[b]);
                    else nk_mbar_arrive(&acc_empty[b]);
                }
            }
            if (!ok) continue;
            if (CG == 1 && p.splits > 1) {   // (pairs never split k)
                // this warp's part of the tile into scratch (lanes side by side), then a ticket; the last one adds all parts
                const int64_t block = int64_t(32) * EC;
                const int64_t first = ((t * p.splits) * 16 + (warp - 2)) * block;
                float4* mine = reinterpret_cast<float4*>(p.parts + first + int64_t(u % p.splits) * 16 * block);
#pragma unroll
                for (int c = 0; c < EC / 4; c++) mine[c * 32 + lane] = make_float4(sum[4 * c], sum[4 * c + 1], sum[4 * c + 2], sum[4 * c + 3]);
                __threadfence();
                __syncwarp();
                int drawn = 0;
                if (lane == 0) drawn = atomicAdd(&p.tickets[t * 16 + (warp - 2)], 1);
                drawn = __shfl_sync(0xffffffffu, drawn, 0);
                if (drawn != p.splits - 1) continue;
                __threadfence();
                for (int part = 0; part < p.splits; part++) {
                    const float4* src = reinterpret_cast<const float4*>(p.parts + first + int64_t(part) * 16 * block);
#pragma unroll
                    for (int c = 0; c < EC / 4; c++) {
                        const float4 v = __ldcg(src + c * 32 + lane);
                        if (part == 0) { sum[4 * c] = v.x; sum[4 * c + 1] = v.y; sum[4 * c + 2] = v.z; sum[4 * c + 3] = v.w; }
                        else { sum[4 * c] += v.x; sum[4 * c + 1] += v.y; sum[4 * c + 2] += v.z; sum[4 * c + 3] += v.w; }
                    }
                }
            }
            bool lost = false;
#pragma unroll
            for (int j = 0; j < EC; j++) lost = lost || sum[j] != sum[j];
            if (__any_sync(0xffffffffu, lost)) {
                float again[EC];
#pragma unroll
                for (int j = 0; j < EC; j++) again[j] = sum[j];
                tc_again<EC, DUAL>(p, again, m, n0);
#pragma unroll
                for (int j = 0; j < EC; j++) sum[j] = again[j];
            }
            drain.store(m, n0, sum);
        }
    }

    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (CG == 2) tc_cluster_sync();   // the peer's products read this CTA's shared memory and write its tensor memory
    if (warp == 1) {
        tc_fence_after();
        if (CG == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(tmem_base), "r"(TC_TMEM_COLS) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem_base), "r"(TC_TMEM_COLS) : "memory");
    }
}

// Which shape, and how k is split, for tiles of `cols` columns per 256 of the pair's shape (256, or 128 of each of two products).
struct TcShape {
    bool pair;
    int splits, kb_per;
    int64_t tiles_m, tiles;
};
inline TcShape tc_shape(int64_t M, int64_t N, int64_t Kp, bool dual, int64_t sms) {
    const int64_t wide = dual ? 128 : 256, narrow = wide / 2;
    const int kb = int(Kp / TC_BK);
    const int64_t m_pair = (M + 255) / 256, n_pair = (N + wide - 1) / wide, m_one = (M + 127) / 128, n_one = (N + narrow - 1) / narrow;
    // k split of the small tiles: as many parts as keep one wave of CTAs busy, each at least two accumulation chunks long
    int64_t splits = sms / (m_one * n_one);
    if (splits > kb / (2 * TC_KC)) splits = kb / (2 * TC_KC);
    if (splits > TC_MAX_SPLITS) splits = TC_MAX_SPLITS;
    if (splits < 1) splits = 1;
    const int64_t kb_per = (kb + splits - 1) / splits;
    splits = (kb + kb_per - 1) / kb_per;
    // Estimated cycles of either shape: waves x k blocks x cycles per stage (pairs: 768, the tensor cores' time for six 128 x 256 x 8
    // products; lone CTAs: 640, their shared-memory traffic of 80 KiB per stage).
    const int64_t est_pair = ((m_pair * n_pair + sms / 2 - 1) / (sms / 2)) * kb * 768;
    const int64_t est_one = ((m_one * n_one * splits + sms - 1) / sms) * kb_per * 640;
    TcShape s;
    s.pair = est_pair <= est_one;
    s.splits = s.pair ? 1 : int(splits);
    s.kb_per = s.splits > 1 ? int(kb_per) : kb;
    s.tiles_m = s.pair ? m_pair : m_one;
    s.tiles = s.pair ? m_pair * n_pair : m_one * n_one;
    return s;
}
inline size_t tc_part_bytes(const TcShape& s) { return s.splits > 1 ? size_t(s.tiles) * s.splits * 128 * 128 * 4 : 0; }
inline size_t tc_ticket_bytes(const TcShape& s) { return s.splits > 1 ? size_t(s.tiles) * 16 * sizeof(int) : 0; }
inline TcParams tc_params(const TcShape& s, int64_t M, int64_t Kp, float* parts, int* tickets, int* status) {
    TcParams p;
    memset(&p, 0, sizeof(p));
    p.M = M;
    p.k_blocks = int(Kp / TC_BK);
    p.tiles_m = int(s.tiles_m);
    p.units = s.tiles * s.splits;
    p.splits = s.splits;
    p.kb_per = s.kb_per;
    p.chunk = TC_KC;
    p.parts = parts;
    p.tickets = tickets;
    p.status = status;
    return p;
}

// rows x Kp panels of an operand, hi and lo
struct TcPanels {
    const float *hi, *lo;
    int64_t rows;
};
// -1: there is no tensor-map encoder
template <int CG, int BN, class Drain>
int tc_launch(nk_ctx* ctx, const char* name, int64_t Kp, const TcPanels& A, const TcPanels& B0, const TcPanels& B1, TcParams tp, const Drain& drain) {
    using C = TcCfg<CG, BN>;
    constexpr bool DUAL = Drain::DUAL;
    TcMaps<DUAL> maps;
    auto encode = [&](const TcPanels& x, int box_rows, CUtensorMap* to) {
        return nk_tma_encode_2d_f32(x.hi, uint64_t(x.rows), uint64_t(Kp), uint64_t(Kp) * 4, TC_BK, box_rows, 2, to) ||
               nk_tma_encode_2d_f32(x.lo, uint64_t(x.rows), uint64_t(Kp), uint64_t(Kp) * 4, TC_BK, box_rows, 2, to + 1);
    };
    constexpr int B_BOX = DUAL && CG == 1 ? C::B_ROWS / 2 : C::B_ROWS;
    if (encode(A, TC_BM, maps.a) || encode(B0, B_BOX, maps.b)) return -1;
    if constexpr (DUAL) {
        if (encode(B1, B_BOX, maps.b + 2)) return -1;
    }
    tp.a[0] = A.hi; tp.a[1] = A.lo;
    tp.b[0] = B0.hi; tp.b[1] = B0.lo; tp.b[2] = B1.hi; tp.b[3] = B1.lo;
    tp.N = B0.rows;
    tp.Kp = Kp;
    auto* kern = nk_conv_tc_kernel<CG, BN, Drain>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM_BYTES);
    if (e != cudaSuccess) return nk_cuda_fail(ctx, e, "cudaFuncSetAttribute(nk_conv_tc_kernel)");
    const int64_t slots = ctx->prop.multiProcessorCount / CG;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(unsigned((tp.units < slots ? tp.units : slots) * CG));
    cfg.blockDim = dim3(TC_THREADS);
    cfg.dynamicSmemBytes = C::SMEM_BYTES;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = CG;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, kern, maps, tp, drain);
    if (e != cudaSuccess) return nk_cuda_fail(ctx, e, "cudaLaunchKernelEx(nk_conv_tc_kernel)");
    return nk_after_launch(ctx, name);
}

}  // namespace
