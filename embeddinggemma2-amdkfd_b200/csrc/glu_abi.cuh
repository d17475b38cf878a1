// Launchers and C entry points (include/eg2_ops.h, part 3) of the gated
// feed-forward projection.  Included once, at the end of kernels.cu.
#pragma once
#include "glu.cuh"
#include "glu_plan.h"

namespace eg2 {

// Up to this many rows run on the CUDA cores.  Weights from memory, us on the CUDA
// cores for 1, 2, 3, 4, 5 and 8 rows against the tensor cores' (the same for all):
// 512 x 2048 2.5, 3.4, 4.2, 3.4, 4.1, 5.2 against 7.3; 2048 x 8192 15.1, 19.1, 23.4,
// 17.6, 31.4, 38.7 against 21.2.
constexpr unsigned GLU_FEW_ROWS = 4;

// [rows][width] of a 16-bit type, boxes of 64 elements x box_rows, 128-byte swizzle.
static bool glu_tmap(CUtensorMap *map, unsigned type, const void *base, int64_t stride, unsigned width, unsigned rows,
                     unsigned box_rows) {
    return encode_tmap_2d(map, type == EG_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                          base, width, rows, uint64_t(stride) * 2, 64, box_rows, true);
}
// A [rows][width] matrix of `size`-byte elements that a tensor map or 16-byte accesses can take.
static bool glu_matrix_ok(const void *p, int64_t *stride, unsigned width, unsigned rows, int size) {
    if (rows < 2) *stride = width;
    return p && aligned16(p) && *stride >= int64_t(width) && *stride * size % 16 == 0 && *stride < (1ll << 36);
}

// f(type tag, activation) for the kernels' template arguments.
template <typename F>
static cudaError_t glu_dispatch(unsigned type, unsigned act, F f) {
    if (act > 1) return cudaErrorInvalidValue;
    if (type == EG_F16) return act ? f(Tag<__half>{}, Int<1>{}) : f(Tag<__half>{}, Int<0>{});
    if (type == EG_BF16) return act ? f(Tag<__nv_bfloat16>{}, Int<1>{}) : f(Tag<__nv_bfloat16>{}, Int<0>{});
    return cudaErrorInvalidValue;
}
template <int MODE, int BN, typename T, int ACT>
static cudaError_t glu_go(const GluMaps &maps, const GluParams &p, int clusters, cudaStream_t s) {
    static AllowSmem allow;
    if (cudaError_t e = allow(glu_kernel<MODE, BN, T, ACT>, int(GluCfg<MODE, BN>::SMEM))) return e;
    return launch_pdl(glu_kernel<MODE, BN, T, ACT>, dim3(2 * clusters), dim3(GluCfg<MODE, BN>::THREADS), GluCfg<MODE, BN>::SMEM, s,
                      maps, p);
}
// Pairs of SMs on the current device: one cluster each.
static int glu_pairs() { return sm_count() < 2 ? 1 : sm_count() / 2; }

static cudaError_t glu_check(unsigned n, unsigned k, unsigned m, unsigned type, unsigned act) {
    if ((type != EG_F16 && type != EG_BF16) || act > 1 || !k || !m || k % 8 || m % 8 || n > 0x7fffff00u ||
        k > (1u << 24) || m > (1u << 24))
        return cudaErrorInvalidValue;
    return cudaSuccess;
}

template <int MODE>
static cudaError_t glu_project(const void *x, int64_t xs, const void *wg, int64_t wgs, const void *wu, int64_t wus,
                               unsigned type, unsigned act, GluParams &p, cudaStream_t s) {
    GluMaps maps{};
    // The width whose slowest cluster is done first; the wider one where they tie.
    const int pairs = glu_pairs(), steps = ceil_div(p.k, 64);
    int bn = 256;
    long long best = LLONG_MAX;
    for (int i = MODE == GLU_DGRAD && p.low[0] ? 1 : 2; i >= 0; --i) {  // 256 columns have no room for the rests
        const long long c = glu_cost(glu_tiles(unsigned(p.n), unsigned(p.m), 32 << i), steps, i, pairs);
        if (c < best) best = c, bn = 64 << i;
    }
    const unsigned wrows = bn == 64 ? 32 : 64;
    if (!glu_tmap(&maps.x, type, x, xs, unsigned(p.k), unsigned(p.n), 64) ||
        !glu_tmap(&maps.wg, type, wg, wgs, unsigned(p.k), unsigned(p.m), wrows) ||
        !glu_tmap(&maps.wu, type, wu, wus, unsigned(p.k), unsigned(p.m), wrows))
        return cudaErrorInvalidValue;
    p.tiles = glu_tiles(unsigned(p.n), unsigned(p.m), bn / 2);
    // 16411 x 2048 x 8192: 738 us, 751 with 8 (the weights are read half as often), 732
    // with 32; 8192 x 4096 x 4096 353, 360 and 375; 4096 x 2048 x 16384 362, 371 and 365.
    p.group = 16;
    const int clusters = p.tiles < pairs ? p.tiles : pairs;
    return glu_dispatch(type, act, [&](auto t, auto a) {
        using T = typename decltype(t)::type;
        constexpr int ACT = decltype(a)::value;
        if (bn == 256) return glu_go<MODE, 256, T, ACT>(maps, p, clusters, s);
        if (bn == 128) return glu_go<MODE, 128, T, ACT>(maps, p, clusters, s);
        return glu_go<MODE, 64, T, ACT>(maps, p, clusters, s);
    });
}

static cudaError_t glu(const EgGlu &a, cudaStream_t s) {
    if (cudaError_t e = glu_check(a.n, a.k, a.m, a.type, a.act)) return e;
    if (!a.n) return cudaSuccess;
    int64_t xs = a.x_stride, gs = a.w_gate_stride, us = a.w_up_stride, os = a.out_stride;
    if (!glu_matrix_ok(a.x, &xs, a.k, a.n, 2) || !glu_matrix_ok(a.w_gate, &gs, a.k, a.m, 2) ||
        !glu_matrix_ok(a.w_up, &us, a.k, a.m, 2) || !glu_matrix_ok(a.out, &os, a.m, a.n, 2))
        return cudaErrorInvalidValue;
    if (a.n <= GLU_FEW_ROWS)
        return glu_dispatch(a.type, a.act, [&](auto t, auto act) {
            using T = typename decltype(t)::type;
            constexpr int ACT = decltype(act)::value;
            auto go = [&](auto kernel, int cols) {
                return launch_pdl(kernel, dim3(ceil_div(a.m, 8 * cols)), dim3(256), 0, s, static_cast<T *>(a.out),
                                  (long long)os, static_cast<const T *>(a.x), (long long)xs,
                                  static_cast<const T *>(a.w_gate), (long long)gs, static_cast<const T *>(a.w_up),
                                  (long long)us, int(a.k), int(a.m));
            };
            switch (a.n) {
                case 1: return go(glu_rows_kernel<T, ACT, 1, 1>, 1);
                case 2: return go(glu_rows_kernel<T, ACT, 2, 2>, 2);
                case 3: return go(glu_rows_kernel<T, ACT, 3, 2>, 2);
                default: return go(glu_rows_kernel<T, ACT, 4, 2>, 2);
            }
        });
    GluParams p{};
    p.n = int(a.n), p.k = int(a.k), p.m = int(a.m);
    p.out[0] = a.out, p.out_stride[0] = os;
    return glu_project<GLU_FORWARD>(a.x, xs, a.w_gate, gs, a.w_up, us, a.type, a.act, p, s);
}

static cudaError_t glu_grad(const EgGluGrad &a, cudaStream_t s) {
    if (cudaError_t e = glu_check(a.n, a.k, a.m, a.type, a.act)) return e;
    if ((a.dw_type != EG_F32 && a.dw_type != a.type) || (a.accumulate && a.dw_type != EG_F32))
        return cudaErrorInvalidValue;
    const int dws = type_size(a.dw_type);
    int64_t xs = a.x_stride, gs = a.w_gate_stride, us = a.w_up_stride, os = a.dout_stride, dxs = a.dx_stride;
    int64_t dgs = a.dw_gate_stride, dus = a.dw_up_stride;
    if ((a.dw_gate && !glu_matrix_ok(a.dw_gate, &dgs, a.k, a.m, dws)) ||
        (a.dw_up && !glu_matrix_ok(a.dw_up, &dus, a.k, a.m, dws)))
        return cudaErrorInvalidValue;
    if (!a.n) {  // no tokens: the weights' gradients are zero
        if (a.accumulate) return cudaSuccess;
        for (int i = 0; i < 2; ++i) {
            void *w = i ? a.dw_up : a.dw_gate;
            if (!w) continue;
            if (cudaError_t e = cudaMemset2DAsync(w, size_t(i ? dus : dgs) * dws, 0, size_t(a.k) * dws, a.m, s))
                return e;
        }
        return cudaSuccess;
    }
    const bool one_row = a.dout_stride == 0;  // a broadcast gradient; dout is read by plain loads, not through a map
    if (!glu_matrix_ok(a.x, &xs, a.k, a.n, 2) || !glu_matrix_ok(a.w_gate, &gs, a.k, a.m, 2) ||
        !glu_matrix_ok(a.w_up, &us, a.k, a.m, 2) || !glu_matrix_ok(a.dout, &os, a.m, one_row ? 1 : a.n, 2) ||
        (a.dx && !glu_matrix_ok(a.dx, &dxs, a.k, a.n, 2)))
        return cudaErrorInvalidValue;
    if (one_row) os = 0;
    if (!a.dx && !a.dw_gate && !a.dw_up) return cudaSuccess;
    const int most = glu_most_splits(a.n, a.k, a.m);
    if (!a.workspace || (reinterpret_cast<uintptr_t>(a.workspace) & 255) ||
        a.workspace_bytes < glu_grad_bytes(a.n, a.k, a.m, most))
        return cudaErrorInvalidValue;
    uint8_t *dg = static_cast<uint8_t *>(a.workspace), *du = dg + glu_half(a.n, a.m);
    GluParams p{};
    p.n = int(a.n), p.k = int(a.k), p.m = int(a.m);
    p.dout = a.dout, p.dout_stride = os;
    p.out[0] = dg, p.out[1] = du, p.out_stride[0] = p.out_stride[1] = a.m;
    p.halves = glu_halves(a.n, a.k, a.m);
    if (p.halves == 2) p.low[0] = du + glu_half(a.n, a.m), p.low[1] = du + 2 * glu_half(a.n, a.m);
    if (cudaError_t e = glu_project<GLU_DGRAD>(a.x, xs, a.w_gate, gs, a.w_up, us, a.type, a.act, p, s)) return e;

    GluMaps maps{};
    if (!glu_tmap(&maps.x, a.type, a.x, xs, a.k, a.n, 64) || !glu_tmap(&maps.wg, a.type, a.w_gate, gs, a.k, a.m, 64) ||
        !glu_tmap(&maps.wu, a.type, a.w_up, us, a.k, a.m, 64) || !glu_tmap(&maps.dg, a.type, dg, a.m, a.m, a.n, 64) ||
        !glu_tmap(&maps.du, a.type, du, a.m, a.m, a.n, 64) ||
        (p.halves == 2 && (!glu_tmap(&maps.dgl, a.type, p.low[0], a.m, a.m, a.n, 64) ||
                           !glu_tmap(&maps.dul, a.type, p.low[1], a.m, a.m, a.n, 64))))
        return cudaErrorInvalidValue;
    p.out[0] = a.dx, p.out[1] = a.dw_gate, p.out[2] = a.dw_up;
    p.out_stride[0] = dxs, p.out_stride[1] = dgs, p.out_stride[2] = dus;
    p.dw_f32 = a.dw_type == EG_F32, p.dw_accumulate = a.accumulate != 0;
    const int weights = (a.dw_gate != nullptr) + (a.dw_up != nullptr);
    const int pairs = glu_pairs() < GLU_PAIRS ? glu_pairs() : GLU_PAIRS;
    const GluPlan plan = glu_plan(a.n, a.k, a.m, a.dx != nullptr, weights, pairs, most);
    const int w_tiles = weights * glu_tiles(a.m, a.k, 256);
    p.splits = plan.splits, p.parts = reinterpret_cast<float *>(dg + glu_parts_at(a.n, a.k, a.m));
    p.dx_tiles = a.dx ? glu_tiles(a.n, a.k, 256) * plan.splits : 0;
    p.tiles = p.dx_tiles + w_tiles;
    p.dx_clusters = plan.dxc < p.dx_tiles ? plan.dxc : p.dx_tiles;
    const int w_clusters = pairs - (plan.dxc < 0 ? 0 : plan.dxc);
    const int clusters = plan.dxc < 0 ? pairs : p.dx_clusters + (w_tiles < w_clusters ? w_tiles : w_clusters);
    // Whole rows of tiles where those are few: 8203 x 2048 x 8192 (8 tiles a row) takes
    // 1206 us with 1, 1235 with 8, 1250 with 16, 4096 x 2304 x 4096 (9) 344 and 363 with 1
    // and 8.  Bands of 8 where they are many: 8192 x 4096 x 8192 (16 tiles) 2.71 and 2.49
    // ms, 2048 x 8192 x 8192 (32) 1.40 and 1.25 ms.  In between neither is ahead by more
    // than runs differ (4096 rows, m = 4096: 10 tiles 401 and 432 us, 16 tiles 615 and 614).
    p.group = ceil_div(a.k, 256) <= 9 ? 1 : 8;
    return glu_dispatch(a.type, 0, [&](auto t, auto) {
        using T = typename decltype(t)::type;
        if (cudaError_t e = glu_go<GLU_PRODUCTS, 256, T, 0>(maps, p, clusters, s)) return e;
        if (!a.dx || p.splits < 2) return cudaSuccess;
        return launch_pdl(glu_add_kernel<T>, dim3(ceil_div((long long)a.n * (a.k / 8), 256)), dim3(256), 0, s,
                          static_cast<T *>(a.dx), (long long)dxs, static_cast<const float *>(p.parts), p.splits,
                          p.n, p.k);
    });
}

}  // namespace eg2

extern "C" {
int eg2_launch_glu(const EgGlu *p, void *s) { return rc(glu(*p, S(s))); }
uint64_t eg2_glu_grad_workspace(unsigned n, unsigned k, unsigned m) {
    return n && k && m ? glu_grad_bytes(n, k, m, glu_most_splits(n, k, m)) : 0;
}
int eg2_launch_glu_grad(const EgGluGrad *p, void *s) { return rc(glu_grad(*p, S(s))); }
}
