// Per-head RMS norm of queries, keys and values with the position rotation, and
// its gradient, for rows of d <= 512 elements in fp32, fp16 or bf16.
//
//   r = 1 / sqrt(mean(x^2) + eps), y = x r w
//   queries and keys: (out_i, out_{i+h}) = (y_i c_i - y_{i+h} s_i, y_{i+h} c_i + y_i s_i), h = d / 2,
//                     c, s = the tables' rows at the token's position
//   values:           out = x r
// Gradient, from x and g = dL/dout:
//   dy = the inverse rotation of g, dw = sum over rows of dy x r, u = dy w,
//   dx = r (u - x r^2 mean(u x))
// A token whose position is outside the tables is padding: its outputs and dx
// are zero, it adds nothing to dw, and its rows are not read.
//
// Sums, statistics and products are in fp32; each output is rounded once.  Both
// directions are bound by memory: every row is read once and written once.
//
// A row is held by G lanes, each with NV vectors of V elements of the lower
// half and the matching ones of the upper half, so that a rotated pair is in
// one lane and the row's sums are log2(G) shuffles.  A group of lanes takes HB
// heads of one token at a time: their loads are all in flight together, and the
// token's cosines and sines and the weights are fetched once for them.
#pragma once
#include "typed.cuh"

namespace eg2 {

struct QkvPart {  // queries, keys or values
    const void *x, *g, *w;  // input; gradient of the output (backward); weight or null
    void *out;              // output, or gradient of the input
    long long x_tok, x_head, g_tok, g_head, out_tok, out_head;
    int heads, blocks;  // blocks = ceil(heads / HB)
};
struct QkvNormParams {
    QkvPart part[3];
    const float *rope_cos, *rope_sin;
    const int *pos;
    float *dw;  // backward: [gridDim.x][2][d] partial weight gradients, or null
    int n, d, positions, weight_f32;
    float eps;
};

template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int o = G / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
template <typename T, int V>
__device__ __forceinline__ void load_weight(float (&w)[V], const void *p, int i, int f32) {
    if (f32) {
        Pack<float, V> x;
        x.load(static_cast<const float *>(p) + i);
        x.get(w);
    } else {
        Pack<T, V> x;
        x.load(static_cast<const T *>(p) + i);
        x.get(w);
    }
}

template <typename T, int V, int G, int NV, int HB>
__global__ void __launch_bounds__(256) qkv_norm_kernel(const __grid_constant__ QkvNormParams p) {
    pdl_wait();
    pdl_trigger();
    const int gl = threadIdx.x % G, half = p.d / 2;
    const int blocks = p.part[0].blocks + p.part[1].blocks + p.part[2].blocks;
    const long long item = ((long long)blockIdx.x * blockDim.x + threadIdx.x) / G;
    const bool live = item < (long long)p.n * blocks;
    const int t = live ? int(item / blocks) : 0;
    int b = live ? int(item % blocks) : 0, kind = 0;
    while (b >= p.part[kind].blocks) b -= p.part[kind++].blocks;
    const QkvPart &q = p.part[kind];
    const int pos = live ? p.pos[t] : -1;
    const bool keep = unsigned(pos) < unsigned(p.positions);
    const T *x = static_cast<const T *>(q.x) + t * q.x_tok + (long long)b * HB * q.x_head;
    T *out = static_cast<T *>(q.out) + t * q.out_tok + (long long)b * HB * q.out_head;
    const int heads = live ? min(HB, q.heads - b * HB) : 0;

    Pack<T, V> lo[HB][NV], hi[HB][NV];
#pragma unroll
    for (int h = 0; h < HB; ++h) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int i = (v * G + gl) * V;
            if (keep && h < heads && i < half) {
                lo[h][v].load(x + h * q.x_head + i);
                hi[h][v].load(x + h * q.x_head + half + i);
            } else {
                lo[h][v].zero(), hi[h][v].zero();
            }
        }
    }
    float c[NV][V], s[NV][V], wl[NV][V], wh[NV][V];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int i = (v * G + gl) * V;
#pragma unroll
        for (int e = 0; e < V; ++e) c[v][e] = 1.0f, s[v][e] = 0.0f, wl[v][e] = wh[v][e] = 1.0f;
        if (kind < 2 && keep && i < half) {
            Pack<float, V> a;
            a.load(p.rope_cos + (long long)pos * half + i);
            a.get(c[v]);
            a.load(p.rope_sin + (long long)pos * half + i);
            a.get(s[v]);
        }
        if (q.w && i < half) {
            load_weight<T, V>(wl[v], q.w, i, p.weight_f32);
            load_weight<T, V>(wh[v], q.w, half + i, p.weight_f32);
        }
    }
#pragma unroll
    for (int h = 0; h < HB; ++h) {
        float ss = 0.0f;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            float a[V], e[V];
            lo[h][v].get(a), hi[h][v].get(e);
#pragma unroll
            for (int i = 0; i < V; ++i) ss = fmaf(a[i], a[i], fmaf(e[i], e[i], ss));
        }
        const float r = keep ? __frsqrt_rn(group_sum<G>(ss) / float(p.d) + p.eps) : 0.0f;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int i0 = (v * G + gl) * V;
            float a[V], e[V];
            lo[h][v].get(a), hi[h][v].get(e);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float ya = a[i] * r * wl[v][i], yb = e[i] * r * wh[v][i];
                a[i] = keep ? ya * c[v][i] - yb * s[v][i] : 0.0f;
                e[i] = keep ? yb * c[v][i] + ya * s[v][i] : 0.0f;
            }
            if (h < heads && i0 < half) {
                Pack<T, V> y;
                y.set(a);
                y.store(out + h * q.out_head + i0);
                y.set(e);
                y.store(out + h * q.out_head + half + i0);
            }
        }
    }
}

// The gradient.  A group walks over items with the grid's stride and keeps its
// columns' share of both weight gradients in registers; the CTA's groups are
// then added in order through shared memory into one partial row per CTA, and
// qkv_dw_kernel adds those in order: no atomics, the same bits on every run.
template <typename T, int V, int G, int NV, int HB>
__global__ void __launch_bounds__(256) qkv_norm_grad_kernel(const __grid_constant__ QkvNormParams p) {
    extern __shared__ float dw_groups[];  // [256 / G][2][d]
    pdl_wait();
    pdl_trigger();
    const int gl = threadIdx.x % G, half = p.d / 2;
    const int blocks = p.part[0].blocks + p.part[1].blocks + p.part[2].blocks;
    const long long items = (long long)p.n * blocks, step = (long long)gridDim.x * (256 / G);
    const float inv_d = 1.0f / float(p.d);
    float dw[2][NV][2][V];
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int e = 0; e < V; ++e) dw[k][v][0][e] = dw[k][v][1][e] = 0.0f;
    // Every group of a warp makes the same number of rounds (the sums shuffle
    // over the whole warp); one past the items is dead.
    const long long first = (long long)blockIdx.x * (256 / G);
    for (long long base = first; base < items; base += step) {
        const long long item = base + threadIdx.x / G;
        const bool live = item < items;
        const int t = live ? int(item / blocks) : 0;
        int b = live ? int(item % blocks) : 0, kind = 0;
        while (b >= p.part[kind].blocks) b -= p.part[kind++].blocks;
        const QkvPart &q = p.part[kind];
        const int pos = live ? p.pos[t] : -1;
        const bool keep = unsigned(pos) < unsigned(p.positions);
        const T *x = static_cast<const T *>(q.x) + t * q.x_tok + (long long)b * HB * q.x_head;
        const T *g = static_cast<const T *>(q.g) + t * q.g_tok + (long long)b * HB * q.g_head;
        T *out = static_cast<T *>(q.out) + t * q.out_tok + (long long)b * HB * q.out_head;
        const int heads = live ? min(HB, q.heads - b * HB) : 0;
        Pack<T, V> xl[HB][NV], xh[HB][NV], ol[HB][NV], oh[HB][NV];
#pragma unroll
        for (int h = 0; h < HB; ++h) {
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int i = (v * G + gl) * V;
                if (keep && h < heads && i < half) {
                    xl[h][v].load(x + h * q.x_head + i);
                    xh[h][v].load(x + h * q.x_head + half + i);
                    ol[h][v].load(g + h * q.g_head + i);
                    oh[h][v].load(g + h * q.g_head + half + i);
                } else {
                    xl[h][v].zero(), xh[h][v].zero(), ol[h][v].zero(), oh[h][v].zero();
                }
            }
        }
        float c[NV][V], s[NV][V], wl[NV][V], wh[NV][V];
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int i = (v * G + gl) * V;
#pragma unroll
            for (int e = 0; e < V; ++e) c[v][e] = 1.0f, s[v][e] = 0.0f, wl[v][e] = wh[v][e] = 1.0f;
            if (kind < 2 && keep && i < half) {
                Pack<float, V> a;
                a.load(p.rope_cos + (long long)pos * half + i);
                a.get(c[v]);
                a.load(p.rope_sin + (long long)pos * half + i);
                a.get(s[v]);
            }
            if (q.w && i < half) {
                load_weight<T, V>(wl[v], q.w, i, p.weight_f32);
                load_weight<T, V>(wh[v], q.w, half + i, p.weight_f32);
            }
        }
#pragma unroll
        for (int h = 0; h < HB; ++h) {
            float ss = 0.0f, ux = 0.0f;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                float a[V], e[V], ga[V], ge[V];
                xl[h][v].get(a), xh[h][v].get(e), ol[h][v].get(ga), oh[h][v].get(ge);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float da = ga[i] * c[v][i] + ge[i] * s[v][i], de = ge[i] * c[v][i] - ga[i] * s[v][i];
                    ss = fmaf(a[i], a[i], fmaf(e[i], e[i], ss));
                    ux = fmaf(da * wl[v][i], a[i], fmaf(de * wh[v][i], e[i], ux));
                }
            }
            ss = group_sum<G>(ss), ux = group_sum<G>(ux);
            const float r = keep ? __frsqrt_rn(ss * inv_d + p.eps) : 0.0f;
            const float m = r * r * (ux * inv_d);
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int i0 = (v * G + gl) * V;
                float a[V], e[V], ga[V], ge[V];
                xl[h][v].get(a), xh[h][v].get(e), ol[h][v].get(ga), oh[h][v].get(ge);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float da = ga[i] * c[v][i] + ge[i] * s[v][i], de = ge[i] * c[v][i] - ga[i] * s[v][i];
                    const float wa = da * (a[i] * r), we = de * (e[i] * r);
                    if (kind == 0) dw[0][v][0][i] += wa, dw[0][v][1][i] += we;
                    if (kind == 1) dw[1][v][0][i] += wa, dw[1][v][1][i] += we;
                    a[i] = keep ? r * (da * wl[v][i] - a[i] * m) : 0.0f;
                    e[i] = keep ? r * (de * wh[v][i] - e[i] * m) : 0.0f;
                }
                if (h < heads && i0 < half) {
                    Pack<T, V> y;
                    y.set(a);
                    y.store(out + h * q.out_head + i0);
                    y.set(e);
                    y.store(out + h * q.out_head + half + i0);
                }
            }
        }
    }
    if (!p.dw) return;
    const int grp = threadIdx.x / G;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int i0 = (v * G + gl) * V;
            if (i0 < half) {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    dw_groups[(grp * 2 + k) * p.d + i0 + e] = dw[k][v][0][e];
                    dw_groups[(grp * 2 + k) * p.d + half + i0 + e] = dw[k][v][1][e];
                }
            }
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * p.d; i += 256) {
        float sum = 0.0f;
        for (int r = 0; r < 256 / G; ++r) sum += dw_groups[r * 2 * p.d + i];
        p.dw[(size_t)blockIdx.x * 2 * p.d + i] = sum;
    }
}

struct QkvDwParams {
    void *dw[2];       // queries', keys'; null: not wanted
    const float *part;  // [parts][2][d]
    int parts, d, f32, accumulate;
};
// Column sums of the partial rows: 32 columns per CTA, each warp every eighth
// row, the warps' sums in order.
template <typename T>
__global__ void __launch_bounds__(256) qkv_dw_kernel(const QkvDwParams p) {
    __shared__ float sums[8][33];
    pdl_wait();
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, col = blockIdx.x * 32 + lane;
    float s = 0.0f;
    if (col < 2 * p.d) {
#pragma unroll 8
        for (int r = warp; r < p.parts; r += 8) s += p.part[(size_t)r * 2 * p.d + col];
    }
    sums[warp][lane] = s;
    __syncthreads();
    if (warp || col >= 2 * p.d) return;
#pragma unroll
    for (int w = 1; w < 8; ++w) s += sums[w][lane];
    const int k = col >= p.d, i = col - k * p.d;
    if (!p.dw[k]) return;
    if (p.f32) {
        float *o = static_cast<float *>(p.dw[k]) + i;
        *o = p.accumulate ? *o + s : s;
    } else {
        T *o = static_cast<T *>(p.dw[k]) + i;
        *o = from_f32<T>(p.accumulate ? to_f32(*o) + s : s);
    }
}

}  // namespace eg2
