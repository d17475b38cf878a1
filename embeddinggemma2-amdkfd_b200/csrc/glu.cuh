// Gated feed-forward projection and its gradient on the 5th-generation tensor
// cores, fp16 or bf16 operands, fp32 accumulators in tensor memory:
//
//   G = x Wg^T, U = x Wu^T, out = act(G) * U           (x [n][k], Wg, Wu [m][k], out [n][m])
//
// and, from dout = dL/dout, with G and U computed again from x:
//
//   dG = dout U act'(G), dU = dout act(G)              (GLU_DGRAD: rounded once to the operands' type,
//                                                       since the next products take them as operands)
//                                                       (in fp16 infinite above 65504); where they
//                                                       are few, what that leaves is kept too)
//   dx = dG Wg + dU Wu, dWg = dG^T x, dWu = dU^T x     (GLU_PRODUCTS)
//
// act is gelu_tanh(g) = g s(2 c (g + 0.044715 g^3)), c = sqrt(2/pi), or silu(g) =
// g s(g), with the logistic s(z) = 1 / (1 + exp(-z)): gelu's 0.5 (1 + tanh v) is
// s(2 v), which keeps its relative precision where tanh is near -1.
//
// Measured on B200, bf16: forward 16411 x 2048 x 8192 (1.10 TFLOP) 0.83 ms, 1.33
// PFLOP/s with the card at its power limit, tensor pipe active on 86 % of the
// cycles; backward 8203 x 2048 x 8192 (1.65 TFLOP) 1.35 ms, pipe 76 % (projections)
// and 86 % (products); backward of a 2048 x 512 x 2048 wave 40 us, a third of it the
// ramps and last epilogues of its three launches.  A 64-deep step of a 256 x 256
// tile takes 0.34 us with or without its loads, one of 256 x 128 no less.
//
// One kernel carries all of it.  A cluster of two CTAs (two SMs) owns one output
// tile of 256 rows x BN columns: each CTA loads its own 128 rows of A and half of
// B's columns, and one tcgen05.mma.cta_group::2 per 16 of K, issued by the even
// CTA, reads both halves, so each SM fetches 32 KB per 64 of K where a tile of its
// own (128 x 256) would fetch 48 KB: the L2-to-SM path is what such tiles run
// into first.  The gate and up projections are one product: the even CTA's half
// of B is the gate's weight rows, the odd one's the up projection's, and the
// accumulator holds a gate column and its up column BN / 2 apart in the same
// lane, where the epilogue pairs them.
//
// Operands arrive by TMA in boxes of 64 elements (128 bytes, 128-byte swizzle) x
// up to 64 rows; an operand whose K runs along the rows in memory (the weights in
// dx, everything in dW) is taken as it lies, as an MN-major operand.  What lies
// outside a tensor is filled with zeros on both sides of a product, and what
// lies outside the output is not stored, so n is free and k, m are multiples of 8
// (the 16-byte row pitch of a tensor map).
//
// Per CTA: warp 0 TMA producer, warp 1 MMA issuer (even CTA) and owner of tensor
// memory, warps 4..11 epilogue (lane quadrant = warp % 4, half of the columns
// each).  Two accumulators of BN columns, so that a tile's epilogue runs under
// the next tile's products.  Persistent; in GLU_PRODUCTS the clusters are shared out
// between dx's tiles (K = 2 m) and the weights' (K = n) by their lengths, or, where
// there are many of both, take dx's and then the weights' together, so that those
// running at one time share more of their operands in L2.
#pragma once
#include "typed.cuh"

namespace eg2 {

enum : int { GLU_FORWARD = 0, GLU_DGRAD = 1, GLU_PRODUCTS = 2 };
enum : int { ACT_GELU_TANH = 0, ACT_SILU = 1 };

template <int MODE, int BN_>
struct GluCfg {
    static constexpr int BN = BN_, BM = 256, BK = 64;  // one cluster's tile
    static constexpr int THREADS = 12 * 32, EPI_WARPS = 8;
    static constexpr int A_BYTES = 128 * BK * 2, B_BYTES = BN / 2 * BK * 2, STAGE = A_BYTES + B_BYTES;
    static constexpr int B_ROWS = BN / 2 < 64 ? BN / 2 : 64;  // rows of a weight box
    // An epilogue warp's own tile in shared memory: its 32 rows x ROW bytes (a
    // quarter of the columns, or 128 bytes of them at a time), two in GLU_DGRAD.
    static constexpr int ROW = MODE == GLU_PRODUCTS ? 128 : BN / 4 * 2, CHUNKS = ROW / 16;
    static constexpr int STAGING = 32 * ROW * (MODE == GLU_DGRAD ? 2 : 1);
    static constexpr int STAGES = MODE == GLU_DGRAD && BN == 256 ? 5 : 6;
    static constexpr size_t SMEM = 1024 + size_t(STAGES) * STAGE + EPI_WARPS * STAGING + 256;
};

struct GluMaps {
    CUtensorMap x, wg, wu, dg, du, dgl, dul;  // dg, du, and dgl, dul with halves = 2: GLU_PRODUCTS only
};
struct GluParams {
    int n, k, m;
    const void *dout;             // GLU_DGRAD
    long long dout_stride;
    void *low[2];                 // DGRAD below 256 columns: what dG's and dU's roundings left (null: not kept)
    int halves;                   // PRODUCTS: 2 where those are operands too, else 1
    void *out[3];                 // FORWARD: out; DGRAD: dG, dU; PRODUCTS: dx, dWg, dWu (null: not wanted)
    long long out_stride[3];
    int dw_f32, dw_accumulate;    // PRODUCTS: the weight gradients' type, and whether they are added to
    int tiles, dx_tiles, group;   // tiles in all; those of dx come first; row tiles walked together
    int splits;                   // PRODUCTS: dx's K in this many parts, a tile each; above 1 they are
    float *parts;                 // written here, [splits][n][k] in fp32, for glu_add_kernel
    int dx_clusters;              // PRODUCTS: clusters 0 .. dx_clusters - 1 take dx's tiles, the others the
                                  // weights'; below 0: all of them dx's and then the weights'
};

// ---------------------------------------------------------------- cluster pieces
__device__ __forceinline__ void bar_arrive_cluster(uint32_t addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
// 2-D tiled load into this CTA's shared memory that completes on a barrier of
// the pair; c0 is a multiple of 64 16-bit elements at every call.
__device__ __forceinline__ void tma_load_2d_pair(void *dst, const CUtensorMap *map, uint32_t bar, int c0, int c1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4}], "
        "[%2];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
        : "memory");
}
__device__ __forceinline__ void tmem_alloc_pair(uint32_t *dst_smem, uint32_t ncols) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst_smem)),
                 "r"(ncols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
// Arrives at the barrier at this offset in both CTAs once the MMAs issued so far completed.
__device__ __forceinline__ void tc_commit_pair(uint64_t *bar) {
    asm volatile(
        "{\n\t.reg .b16 both;\n\tmov.b16 both, 3;\n\t"
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], both;\n\t}" ::"r"(
            smem_u32(bar))
        : "memory");
}
__device__ __forceinline__ void mma_f16_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                             uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// ---------------------------------------------------------------- activation
// s(z) = 1 / (1 + 2^(-z log2 e)) from the approximate 2^x and reciprocal, each
// within a few 2^-23 of its value: far below the operands' types.
__device__ __forceinline__ float logistic(float z) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + ex2_approx(-1.4426950408889634f * z)));
    return r;
}
constexpr float GELU_A = 1.5957691216057308f, GELU_B = 0.071354816272600247f;  // 2 sqrt(2/pi) times 1 and 0.044715
template <int ACT>
__device__ __forceinline__ float glu_act(float g) {
    return ACT == ACT_SILU ? g * logistic(g) : g * logistic(g * fmaf(GELU_B * g, g, GELU_A));
}
// act(g) and act'(g) = s (1 + g z' (1 - s)).  gelu's slope is 0 or 1, and s too, to
// the last bit of fp32 beyond |g| = 32; held there (NaN stays NaN), since g z'
// overflows from |g| = 1.2e13 and 0 * inf would be NaN.
template <int ACT>
__device__ __forceinline__ float glu_act_grad(float g, float *act) {
    const float b = ACT == ACT_SILU || !(fabsf(g) > 32.0f) ? g : copysignf(32.0f, g), b2 = b * b;
    const float s = logistic(ACT == ACT_SILU ? b : b * fmaf(GELU_B, b2, GELU_A));
    const float dz = ACT == ACT_SILU ? 1.0f : fmaf(3.0f * GELU_B, b2, GELU_A);
    *act = g * s;
    return s * fmaf(b * dz, 1.0f - s, 1.0f);
}
// What rounding a pair to T left of it, rounded to T (nothing where it became infinite).
template <typename T>
__device__ __forceinline__ uint32_t rest2(float2 f, uint32_t rounded) {
    const T *h = reinterpret_cast<const T *>(&rounded);
    const float a = to_f32(h[0]), b = to_f32(h[1]);
    return pack2<T>(isinf(a) ? 0.0f : f.x - a, isinf(b) ? 0.0f : f.y - b);
}
// ---------------------------------------------------------------- tiles
// kind 0: the projections' tile or dx's; kinds 1 and 2: dWg's and dWu's.
struct GluTile {
    int kind, row0, col0, steps, step0, part;  // K steps step0 .. step0 + steps - 1
};
template <int MODE, int BN>
__device__ __forceinline__ GluTile glu_tile(const GluParams &p, int i) {
    const int steps_m = (p.m + 63) / 64;
    int kind = 0, rows = p.n, cols = p.m, bn = BN / 2, steps = (p.k + 63) / 64, step0 = 0, part = 0;
    if (MODE == GLU_PRODUCTS) {
        cols = p.k, bn = BN, steps = 2 * steps_m * p.halves;
        if (i < p.dx_tiles) {
            const int each = p.dx_tiles / p.splits;
            part = i / each, i -= part * each;
            step0 = int((long long)steps * part / p.splits);
            steps = int((long long)steps * (part + 1) / p.splits) - step0;
        } else {
            i -= p.dx_tiles;
            rows = p.m, steps = (p.n + 63) / 64 * p.halves;
            kind = p.out[1] ? 1 : 2;
            const int each = ((rows + 255) / 256) * ((cols + bn - 1) / bn);
            if (i >= each) i -= each, kind = 2;
        }
    }
    // `group` row tiles are walked together, column by column, so that the tiles
    // running at one time share their operands in L2.
    const int tm = (rows + 255) / 256, tn = (cols + bn - 1) / bn;
    const int band = i / (p.group * tn), r0 = band * p.group, height = min(p.group, tm - r0);
    const int j = i - band * p.group * tn;
    return {kind, (r0 + j % height) * 256, (j / height) * bn, steps, step0, part};
}

template <int MODE, int BN, typename T, int ACT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(GluCfg<MODE, BN>::THREADS, 1)
    glu_kernel(const __grid_constant__ GluMaps maps, const __grid_constant__ GluParams p) {
    using C = GluCfg<MODE, BN>;
    static_assert(sizeof(T) == 2, "16-bit operands");
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = align_smem_1024(smem_raw);
    uint8_t *staging = smem + size_t(C::STAGES) * C::STAGE;
    uint64_t *bars = reinterpret_cast<uint64_t *>(staging + C::EPI_WARPS * C::STAGING);
    uint64_t *full = bars, *empty = full + C::STAGES, *accfull = empty + C::STAGES, *accempty = accfull + 2;
    uint64_t *mdone = accempty + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(mdone + 1);
    volatile int *abort = reinterpret_cast<int *>(tmem_slot + 1);
    auto a_tile = [&](int s) { return smem + s * C::STAGE; };
    auto b_tile = [&](int s) { return smem + s * C::STAGE + C::A_BYTES; };

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = int(cluster_rank());
    // This cluster's tiles: first, first + step, ... below end.
    int first = blockIdx.x / 2, step = gridDim.x / 2, end = p.tiles;
    if (MODE == GLU_PRODUCTS && p.dx_clusters >= 0) {
        if (first < p.dx_clusters) step = p.dx_clusters, end = p.dx_tiles;
        else first += p.dx_tiles - p.dx_clusters, step -= p.dx_clusters;
    }
    if (threadIdx.x == 0) {
        tma_prefetch(&maps.x), tma_prefetch(&maps.wg), tma_prefetch(&maps.wu);
        *abort = 0;
        for (int s = 0; s < C::STAGES; ++s) bar_init(&full[s], 1), bar_init(&empty[s], 1);
        for (int b = 0; b < 2; ++b) bar_init(&accfull[b], 1), bar_init(&accempty[b], 2 * C::EPI_WARPS);
        bar_init(mdone, 1);
        fence_bar_init();
    }
    if (warp == 1) tmem_alloc_pair(tmem_slot, 512);
    tc_fence_before();
    cluster_sync_all();
    tc_fence_after();
    pdl_wait();
    pdl_trigger();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {
        // ------------------------------------------------------------ TMA producer
        if (lane == 0) {
            int it = 0;
            bool ok = true;
            for (int i = first; ok && i < end; i += step) {
                const GluTile t = glu_tile<MODE, BN>(p, i);
                for (int kb = 0; kb < t.steps; ++kb, ++it) {
                    const int s = it % C::STAGES;
                    if (!wait_bar(&empty[s], ((it / C::STAGES) & 1) ^ 1, abort)) {
                        ok = false;
                        break;
                    }
                    // The even CTA's barrier counts both CTAs' bytes.
                    if (rank == 0) bar_expect_tx(&full[s], 2 * C::STAGE);
                    const uint32_t bar = cluster_addr(0, &full[s]);
                    uint8_t *a = a_tile(s), *b = b_tile(s);
                    const int arow = t.row0 + rank * 128;
                    if (MODE != GLU_PRODUCTS) {
                        for (int j = 0; j < 2; ++j) tma_load_2d_pair(a + j * 8192, &maps.x, bar, kb * 64, arow + j * 64);
                        for (int j = 0; j < BN / 2 / C::B_ROWS; ++j)
                            tma_load_2d_pair(b + j * 8192, rank ? &maps.wu : &maps.wg, bar, kb * 64, t.col0 + j * 64);
                    } else {
                        const int bcol = t.col0 + rank * (BN / 2);
                        if (t.kind == 0) {
                            // K: dG's columns, dU's, and with two halves dG's and dU's rests.
                            const int per = (p.m + 63) / 64, ks = t.step0 + kb;
                            const int seg = (ks >= per) + (ks >= 2 * per) + (ks >= 3 * per), k0 = (ks - seg * per) * 64;
                            const CUtensorMap *am = seg < 2 ? (seg ? &maps.du : &maps.dg) : seg == 2 ? &maps.dgl : &maps.dul;
                            for (int j = 0; j < 2; ++j) tma_load_2d_pair(a + j * 8192, am, bar, k0, arow + j * 64);
                            for (int j = 0; j < BN / 128; ++j)
                                tma_load_2d_pair(b + j * 8192, seg & 1 ? &maps.wu : &maps.wg, bar, bcol + j * 64, k0);
                        } else {
                            // K: the tokens, and with two halves the same tokens' rests.
                            const int per = (p.n + 63) / 64, low = kb >= per, k0 = (kb - low * per) * 64;
                            const CUtensorMap *am = low ? (t.kind == 1 ? &maps.dgl : &maps.dul)
                                                        : t.kind == 1 ? &maps.dg : &maps.du;
                            for (int j = 0; j < 2; ++j) tma_load_2d_pair(a + j * 8192, am, bar, arow + j * 64, k0);
                            for (int j = 0; j < BN / 128; ++j)
                                tma_load_2d_pair(b + j * 8192, &maps.x, bar, bcol + j * 64, k0);
                        }
                    }
                }
            }
            // Drain: the MMAs have released the last loads' stages, so no arrival at
            // this CTA's barriers is still on its way when the cluster ends; and
            // (whatever happened) the loads themselves have landed: the even
            // CTA's barriers cover the odd one's too.
            const int last = it > C::STAGES ? it - C::STAGES : 0;
            for (int j = last; ok && j < it; ++j) ok = wait_bar(&empty[j % C::STAGES], (j / C::STAGES) & 1, abort);
            if (rank == 0)
                for (int j = last; j < it; ++j) wait_bar(&full[j % C::STAGES], (j / C::STAGES) & 1, nullptr);
        }
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer
        if (rank == 0 && lane == 0) {
            constexpr uint32_t FMT = sizeof(T) == 2 && !std::is_same<T, __half>::value ? (1u << 7) | (1u << 10) : 0u;
            constexpr uint32_t BASE = (1u << 4) | FMT | (uint32_t(BN >> 3) << 17) | (uint32_t(C::BM >> 4) << 24);
            int it = 0, ti = 0;
            bool ok = true;
            for (int i = first; ok && i < end; i += step, ++ti) {
                const GluTile t = glu_tile<MODE, BN>(p, i);
                const int buf = ti & 1;
                const bool a_mn = MODE == GLU_PRODUCTS && t.kind != 0;
                constexpr bool b_mn = MODE == GLU_PRODUCTS;
                const uint32_t idesc = BASE | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u);
                if (!wait_bar(&accempty[buf], ((ti >> 1) & 1) ^ 1, abort)) break;
                tc_fence_after();
                for (int kb = 0; kb < t.steps; ++kb, ++it) {
                    const int s = it % C::STAGES;
                    if (!wait_bar(&full[s], (it / C::STAGES) & 1, abort)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t a = smem_u32(a_tile(s)), b = smem_u32(b_tile(s));
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) {
                        const uint64_t ad = a_mn ? desc_mn_sw128(a + kk * 2048, 8192) : desc_sw128(a + kk * 32);
                        const uint64_t bd = b_mn ? desc_mn_sw128(b + kk * 2048, 8192) : desc_sw128(b + kk * 32);
                        mma_f16_pair(tmem + uint32_t(buf * BN), ad, bd, idesc, kb > 0 || kk > 0 ? 1u : 0u);
                    }
                    tc_commit_pair(&empty[s]);
                }
                if (ok) tc_commit_pair(&accfull[buf]);
            }
            // Drain: every MMA issued above has completed before tensor memory is freed.
            asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                             smem_u32(mdone))
                         : "memory");
            wait_bar(mdone, 0, nullptr);
        }
        __syncwarp();
    } else if (warp >= 4) {
        // ------------------------------------------------------------ epilogue
        // A thread has one row of the accumulator; memory wants whole rows of a
        // tile from neighbouring lanes.  Between the two each warp turns its rows
        // in its own piece of shared memory, in 16-byte chunks whose places are
        // permuted by row so that both ways are free of bank conflicts.
        const int quad = warp & 3, part = (warp - 4) >> 2;
        const uint32_t lanes = tmem + (uint32_t(quad * 32) << 16);
        uint8_t *mine = staging + (warp - 4) * C::STAGING;
        auto chunk = [&](int r, int c) {
            return reinterpret_cast<uint4 *>(mine + r * C::ROW + ((c ^ (r * C::ROW / 128)) & (C::CHUNKS - 1)) * 16);
        };
        // Lane's chunk of the i-th group of rows that one access covers.
        const int crow = lane / C::CHUNKS, ccol = lane % C::CHUNKS;
        constexpr int PER = 32 / C::CHUNKS;
        int ti = 0;
        for (int i = first; i < end; i += step, ++ti) {
            const GluTile t = glu_tile<MODE, BN>(p, i);
            const int buf = ti & 1, row0 = t.row0 + rank * 128 + quad * 32;
            const uint32_t acc = lanes + uint32_t(buf * BN);
            uint4 dh[MODE == GLU_DGRAD ? C::CHUNKS : 1];
            if constexpr (MODE == GLU_DGRAD) {  // dout's rows while the products are still running
                const int col = t.col0 + part * (BN / 4) + ccol * 8;
#pragma unroll
                for (int c = 0; c < C::CHUNKS; ++c) {
                    const int r = row0 + c * PER + crow;
                    dh[c] = make_uint4(0, 0, 0, 0);
                    if (r < p.n && col < p.m)
                        dh[c] = *reinterpret_cast<const uint4 *>(static_cast<const T *>(p.dout) + r * p.dout_stride + col);
                }
            }
            // The one wait for a whole tile's products: 2 us a step on top of the usual
            // limit, about six times what a step takes, since K may be 2^25 steps long.
            const uint64_t limit = WAIT_NS + uint64_t(t.steps) * 2000;
            if (!__all_sync(0xffffffffu, wait_bar(&accfull[buf], (ti >> 1) & 1, abort, limit))) break;
            tc_fence_after();
            // The accumulator is free for the tile after next once both CTAs' warps have read it.
            auto release = [&] {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive_cluster(cluster_addr(0, &accempty[buf]));
            };
            if constexpr (MODE == GLU_PRODUCTS) {
                const bool dw = t.kind != 0, f32 = dw ? p.dw_f32 : p.splits > 1;
                const int rows = dw ? p.m : p.n, each = f32 ? 32 : 64;  // columns in 128 bytes
                const long long pitch = !dw && f32 ? p.k : p.out_stride[t.kind];
                void *dst = !dw && f32 ? static_cast<void *>(p.parts + (long long)t.part * p.n * p.k) : p.out[t.kind];
                const int last = (part + 1) * (BN / 2);
                for (int c0 = part * (BN / 2); c0 < last; c0 += each) {
                    if (t.col0 + c0 >= p.k) break;
                    uint32_t r[32];
                    tmem_ld32(acc + uint32_t(c0), r);
                    tmem_wait_ld();
                    reg_fence(r);
                    if (f32) {
#pragma unroll
                        for (int c = 0; c < 8; ++c)
                            *chunk(lane, c) = make_uint4(r[4 * c], r[4 * c + 1], r[4 * c + 2], r[4 * c + 3]);
                    } else {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            if (h) {
                                tmem_ld32(acc + uint32_t(c0 + 32), r);
                                tmem_wait_ld();
                                reg_fence(r);
                            }
#pragma unroll
                            for (int c = 0; c < 4; ++c) {
                                uint32_t w[4];
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    w[e] = pack2<T>(__uint_as_float(r[8 * c + 2 * e]),
                                                    __uint_as_float(r[8 * c + 2 * e + 1]));
                                *chunk(lane, 4 * h + c) = make_uint4(w[0], w[1], w[2], w[3]);
                            }
                        }
                    }
                    __syncwarp();
                    const int col = t.col0 + c0 + ccol * (f32 ? 4 : 8);
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        const int rr = row0 + c * PER + crow;
                        if (rr >= rows || col >= p.k) continue;
                        uint4 v = *chunk(c * PER + crow, ccol);
                        uint8_t *to = static_cast<uint8_t *>(dst) + (rr * pitch + col) * (f32 ? 4 : 2);
                        if (dw && p.dw_accumulate) {
                            const float4 o = *reinterpret_cast<const float4 *>(to);
                            v = make_uint4(__float_as_uint(__uint_as_float(v.x) + o.x),
                                           __float_as_uint(__uint_as_float(v.y) + o.y),
                                           __float_as_uint(__uint_as_float(v.z) + o.z),
                                           __float_as_uint(__uint_as_float(v.w) + o.w));
                        }
                        *reinterpret_cast<uint4 *>(to) = v;
                    }
                    __syncwarp();
                }
                release();
            } else {
                // Gate columns 0 .. BN/2 - 1 of the accumulator, up columns BN/2 ..; this warp's half of each.
                if constexpr (MODE == GLU_DGRAD) {
#pragma unroll
                    for (int c = 0; c < C::CHUNKS; ++c) *chunk(c * PER + crow, ccol) = dh[c];
                    __syncwarp();
                }
                constexpr int STEP = BN / 4 < 32 ? BN / 4 : 32;
                constexpr int DU = 32 * C::ROW / 16;  // chunks from dG's tile to dU's
                for (int c0 = 0; c0 < BN / 4; c0 += STEP) {
                    uint32_t g[STEP], u[STEP];
                    const uint32_t at = acc + uint32_t(part * (BN / 4) + c0);
                    if constexpr (STEP == 32) {
                        tmem_ld32(at, g);
                        tmem_ld32(at + BN / 2, u);
                    } else {
                        tmem_ld16(at, g);
                        tmem_ld16(at + BN / 2, u);
                    }
                    tmem_wait_ld();
                    reg_fence(g), reg_fence(u);
                    if (c0 + STEP == BN / 4) release();
#pragma unroll
                    for (int j = 0; j < STEP / 8; ++j) {
                        uint4 *place = chunk(lane, c0 / 8 + j);
                        uint32_t w[4];
                        if constexpr (MODE == GLU_FORWARD) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int z = 8 * j + 2 * e;
                                w[e] = pack2<T>(glu_act<ACT>(__uint_as_float(g[z])) * __uint_as_float(u[z]),
                                                glu_act<ACT>(__uint_as_float(g[z + 1])) * __uint_as_float(u[z + 1]));
                            }
                        } else {
                            float2 d[4];
                            unpack2(*place, d, T());
                            uint32_t v[4], wl[4], vl[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int z = 8 * j + 2 * e;
                                float a0, a1;
                                const float d0 = glu_act_grad<ACT>(__uint_as_float(g[z]), &a0);
                                const float d1 = glu_act_grad<ACT>(__uint_as_float(g[z + 1]), &a1);
                                const float2 dg = make_float2(d[e].x * __uint_as_float(u[z]) * d0,
                                                              d[e].y * __uint_as_float(u[z + 1]) * d1);
                                const float2 du = make_float2(d[e].x * a0, d[e].y * a1);
                                w[e] = pack2<T>(dg.x, dg.y), v[e] = pack2<T>(du.x, du.y);
                                if (BN < 256) wl[e] = rest2<T>(dg, w[e]), vl[e] = rest2<T>(du, v[e]);
                            }
                            place[DU] = make_uint4(v[0], v[1], v[2], v[3]);
                            if (BN < 256 && p.low[0]) {  // a few KB in all: straight from the rows' threads
                                const int r = row0 + lane, col = t.col0 + part * (BN / 4) + c0 + 8 * j;
                                if (r < p.n && col < p.m) {
                                    const long long at = (long long)r * p.m + col;
                                    *reinterpret_cast<uint4 *>(static_cast<T *>(p.low[0]) + at) = make_uint4(wl[0], wl[1], wl[2], wl[3]);
                                    *reinterpret_cast<uint4 *>(static_cast<T *>(p.low[1]) + at) = make_uint4(vl[0], vl[1], vl[2], vl[3]);
                                }
                            }
                        }
                        *place = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
                __syncwarp();
                const int col = t.col0 + part * (BN / 4) + ccol * 8;
#pragma unroll
                for (int c = 0; c < C::CHUNKS; ++c) {
                    const int r = row0 + c * PER + crow;
                    if (r >= p.n || col >= p.m) continue;
                    const uint4 *place = chunk(c * PER + crow, ccol);
                    const long long at = r * p.out_stride[0] + col;
                    *reinterpret_cast<uint4 *>(static_cast<T *>(p.out[0]) + at) = *place;
                    if (MODE == GLU_DGRAD) *reinterpret_cast<uint4 *>(static_cast<T *>(p.out[1]) + at) = place[DU];
                }
                __syncwarp();
            }
        }
    }
    // Both CTAs' barriers and shared memory stay until neither uses the other's.
    tc_fence_before();
    __syncwarp();
    cluster_sync_all();
    tc_fence_after();
    if (warp == 1) tmem_dealloc_pair(tmem, 512);
    __syncwarp();
    cluster_sync_all();
}

// dx from its parts, added in order and rounded once.
template <typename T>
__global__ void __launch_bounds__(256) glu_add_kernel(T *__restrict__ dx, long long stride, const float *__restrict__ parts,
                                                      int splits, int n, int k) {
    pdl_wait();
    pdl_trigger();
    const int per_row = k / 8;
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= (long long)n * per_row) return;
    const int row = int(i / per_row), col = int(i - (long long)row * per_row) * 8;
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = 0.0f;
    for (int s = 0; s < splits; ++s) {
        Pack<float, 8> x;
        float g[8];
        x.load(parts + ((long long)s * n + row) * k + col);
        x.get(g);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] += g[e];
    }
    Pack<T, 8> y;
    y.set(f);
    y.store(dx + row * stride + col);
}

// A few rows (single tokens in serving): the weights' bytes are what there is to
// move, and the tensor cores' 256-row tiles would be empty.  A warp takes COLS
// output columns: their weight rows stream through registers once, against NT
// rows of x, each of whose vectors serves all COLS columns.
template <typename T, int ACT, int NT, int COLS>
__global__ void __launch_bounds__(256) glu_rows_kernel(T *__restrict__ out, long long out_stride,
                                                       const T *__restrict__ x, long long x_stride,
                                                       const T *__restrict__ wg, long long wg_stride,
                                                       const T *__restrict__ wu, long long wu_stride, int k, int m) {
    pdl_wait();
    pdl_trigger();
    const int col = (blockIdx.x * 8 + (threadIdx.x >> 5)) * COLS, lane = threadIdx.x & 31;
    if (col >= m) return;  // m is a multiple of COLS
    float2 g[NT][COLS], u[NT][COLS];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int c = 0; c < COLS; ++c) g[t][c] = u[t][c] = make_float2(0.0f, 0.0f);
#pragma unroll 2
    for (int i = lane * 8; i < k; i += 256) {
        uint4 a[COLS], b[COLS], y[NT];
#pragma unroll
        for (int c = 0; c < COLS; ++c) {
            a[c] = *reinterpret_cast<const uint4 *>(wg + (col + c) * wg_stride + i);
            b[c] = *reinterpret_cast<const uint4 *>(wu + (col + c) * wu_stride + i);
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) y[t] = *reinterpret_cast<const uint4 *>(x + t * x_stride + i);
#pragma unroll
        for (int c = 0; c < COLS; ++c) {
            float2 fa[4], fb[4];
            unpack2(a[c], fa, T()), unpack2(b[c], fb, T());
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                float2 fx[4];
                unpack2(y[t], fx, T());
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    g[t][c] = fma2(fx[e], fa[e], g[t][c]);
                    u[t][c] = fma2(fx[e], fb[e], u[t][c]);
                }
            }
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int c = 0; c < COLS; ++c) {
            const float gs = warp_sum_f(g[t][c].x + g[t][c].y), us = warp_sum_f(u[t][c].x + u[t][c].y);
            if (lane == 0) out[t * out_stride + col + c] = from_f32<T>(glu_act<ACT>(gs) * us);
        }
}

}  // namespace eg2
