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
// A row is held by G lanes, each with NV vectors of V elements of the lower half
// and the matching ones of the upper half, so that a rotated pair is in one lane
// and the row's sums are log2(G) shuffles.
#pragma once
#include "typed.cuh"

namespace eg2 {

struct QkvPart {  // queries, keys or values
    const void *x, *g, *w;  // input; gradient of the output (backward); weight or null
    void *out;              // output, or gradient of the input
    long long x_tok, x_head, g_tok, g_head, out_tok, out_head;
    int heads, blocks;  // blocks of HB heads (streaming form)
};
struct QkvNormParams {
    QkvPart part[3];
    const float *rope_cos, *rope_sin;
    const int *pos;
    int cta_end[3];  // CTAs of queries, keys, values end here (0 .. cta_end[0] - 1 are queries')
    float *dw;       // gradient: partial weight gradients, one row of d per CTA, or null
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

// The direct form: one head per group of lanes, straight from global memory.  It
// takes the rows that are not whole 16-byte vectors, and the calls of a few
// tokens, where all rows are in flight at once anyway.
template <typename T, int V, int G, int NV>
__global__ void __launch_bounds__(256) qkv_norm_kernel(const __grid_constant__ QkvNormParams p) {
    pdl_wait();
    pdl_trigger();
    const int gl = threadIdx.x % G, half = p.d / 2;
    const int heads = p.part[0].heads + p.part[1].heads + p.part[2].heads;
    const long long item = ((long long)blockIdx.x * blockDim.x + threadIdx.x) / G;
    const bool live = item < (long long)p.n * heads;
    const int t = live ? int(item / heads) : 0;
    int h = live ? int(item - (long long)t * heads) : 0, kind = 0;
    while (h >= p.part[kind].heads) h -= p.part[kind++].heads;
    const QkvPart &q = p.part[kind];
    const int pos = live ? p.pos[t] : -1;
    const bool keep = unsigned(pos) < unsigned(p.positions);
    const T *x = static_cast<const T *>(q.x) + t * q.x_tok + h * q.x_head;
    T *out = static_cast<T *>(q.out) + t * q.out_tok + h * q.out_head;
    float a[NV][V], b[NV][V], c[NV][V], s[NV][V], wl[NV][V], wh[NV][V], ss = 0.0f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int i = (v * G + gl) * V;
        Pack<T, V> lo, hi;
        lo.zero(), hi.zero();
        if (keep && i < half) lo.load(x + i), hi.load(x + half + i);
        lo.get(a[v]), hi.get(b[v]);
#pragma unroll
        for (int e = 0; e < V; ++e) c[v][e] = 1.0f, s[v][e] = 0.0f, wl[v][e] = wh[v][e] = 1.0f;
        if (kind < 2 && keep && i < half) {
            Pack<float, V> f;
            f.load(p.rope_cos + (long long)pos * half + i);
            f.get(c[v]);
            f.load(p.rope_sin + (long long)pos * half + i);
            f.get(s[v]);
        }
        if (q.w && i < half) {
            load_weight<T, V>(wl[v], q.w, i, p.weight_f32);
            load_weight<T, V>(wh[v], q.w, half + i, p.weight_f32);
        }
#pragma unroll
        for (int e = 0; e < V; ++e) ss = fmaf(a[v][e], a[v][e], fmaf(b[v][e], b[v][e], ss));
    }
    const float r = keep ? __frsqrt_rn(group_sum<G>(ss) / float(p.d) + p.eps) : 0.0f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int i = (v * G + gl) * V;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float ya = a[v][e] * r * wl[v][e], yb = b[v][e] * r * wh[v][e];
            a[v][e] = keep ? ya * c[v][e] - yb * s[v][e] : 0.0f;
            b[v][e] = keep ? yb * c[v][e] + ya * s[v][e] : 0.0f;
        }
        if (live && i < half) {
            Pack<T, V> y;
            y.set(a[v]);
            y.store(out + i);
            y.set(b[v]);
            y.store(out + half + i);
        }
    }
}

// The streaming form of both directions, for rows of whole 16-byte vectors.  The
// grid is two resident CTAs per SM, shared out among queries, keys and values by
// their rows, so that a group keeps one weight (and, in the gradient, one weight
// gradient) in registers.  A group takes the same HB heads of every `down`th
// token, neighbouring groups the neighbouring heads (which share the token's
// cosines and sines in one access), and fetches the next token's rows before it
// works on this one's, so that loads are in flight all the time.
//
// Measured on B200, bf16: forward 32771 tokens x 12 heads x 128 in 37 us (202 MB,
// 5.5 TB/s; 62 us with direct loads that only other warps covered, 60 with all of
// a group's operands through shared memory), gradient 16411 x 20 x 128 in 44 us
// (253 MB, 5.8 TB/s; 112 us direct, 54 with the next rows in registers).  What
// bounds both now is memory; they issue on half of the cycles.
template <typename T, int G, int NV, int HB, bool GRAD, bool EXACT>
__global__ void __launch_bounds__(256, 2) qkv_stream_kernel(const __grid_constant__ QkvNormParams p) {
    constexpr int V = 16 / int(sizeof(T)), P = V / 2;
    extern __shared__ __align__(16) float sums[];  // gradient: the ring, then [256 / G][d]
    pdl_wait();
    pdl_trigger();
    // EXACT: the G * NV vectors are the whole half, whose length is then known here.
    const int gl = threadIdx.x % G, half = EXACT ? G * NV * V : p.d / 2;
    int kind = 0;
    while (int(blockIdx.x) >= p.cta_end[kind]) ++kind;
    const QkvPart &q = p.part[kind];
    const int cta0 = kind ? p.cta_end[kind - 1] : 0;
    // The kind's groups as a grid: `across` blocks of HB heads side by side by
    // `down` tokens.  (Only with more blocks than groups is across < blocks.)
    const int groups = (p.cta_end[kind] - cta0) * (256 / G), g0 = (int(blockIdx.x) - cta0) * (256 / G);
    const int across = min(q.blocks, groups), down = groups / across;
    const int mine = g0 + int(threadIdx.x) / G, t0 = mine / across;
    // Rounds are the same for the whole CTA: the sums shuffle over whole warps.
    const int tfirst = g0 / across, rounds = tfirst < p.n ? (p.n - tfirst + down - 1) / down : 0;
    const float inv_d = 1.0f / float(p.d);
    const bool rope = kind < 2;

    // Weights, and the sums of their gradients, of this lane's columns.
    float2 wl[NV][P], wh[NV][P], dl[GRAD ? NV : 1][P], dh[GRAD ? NV : 1][P];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int i = (v * G + gl) * V;
        float a[V], b[V];
#pragma unroll
        for (int e = 0; e < V; ++e) a[e] = b[e] = 1.0f;
        if (q.w && (EXACT || i < half)) {
            load_weight<T, V>(a, q.w, i, p.weight_f32);
            load_weight<T, V>(b, q.w, half + i, p.weight_f32);
        }
#pragma unroll
        for (int e = 0; e < P; ++e) {
            wl[v][e] = make_float2(a[2 * e], a[2 * e + 1]), wh[v][e] = make_float2(b[2 * e], b[2 * e + 1]);
            if (GRAD) dl[v][e] = dh[v][e] = make_float2(0.0f, 0.0f);
        }
    }
    // The next item's rows: in registers, as they lie in memory (forward), or
    // copied to this thread's slots of shared memory, [stage][slot][thread], while
    // the other stage is worked on (gradient, which has no registers to spare).
    constexpr int SLOTS = HB * NV * 4;
    uint4 next[GRAD ? 1 : HB][NV][2];
    uint4 *ring = reinterpret_cast<uint4 *>(sums) + threadIdx.x;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    for (int b0 = 0; b0 < q.blocks; b0 += across) {
        const int h0 = (b0 + mine % across) * HB, heads = t0 < down ? q.heads - h0 : 0;
        const int tend = heads > 0 ? p.n : 0;
        auto position = [&](int t) -> int { return t < tend ? p.pos[t] : -1; };
        // Addresses of the next item to fetch and of the one to store, this lane's columns.
        const T *x = static_cast<const T *>(q.x) + t0 * q.x_tok + h0 * q.x_head + gl * V;
        const T *g = static_cast<const T *>(q.g) + (GRAD ? t0 * q.g_tok + h0 * q.g_head + gl * V : 0);
        T *out = static_cast<T *>(q.out) + t0 * q.out_tok + h0 * q.out_head + gl * V;
        auto fetch = [&](int stage, int pos) {
            const bool on = unsigned(pos) < unsigned(p.positions);
#pragma unroll
            for (int h = 0; h < HB; ++h) {
#pragma unroll
                for (int v = 0; v < NV; ++v) {
                    const bool row = on && h < heads && (EXACT || (v * G + gl) * V < half);
                    const T *src = x + h * q.x_head + v * G * V;
                    if constexpr (GRAD) {
                        const T *grd = g + h * q.g_head + v * G * V;
                        uint4 *at = ring + (stage * SLOTS + (h * NV + v) * 4) * 256;
                        copy16(at, src, row), copy16(at + 256, src + half, row);
                        copy16(at + 512, grd, row), copy16(at + 768, grd + half, row);
                    } else {
                        next[h][v][0] = next[h][v][1] = zero;
                        if (row) {
                            next[h][v][0] = *reinterpret_cast<const uint4 *>(src);
                            next[h][v][1] = *reinterpret_cast<const uint4 *>(src + half);
                        }
                    }
                }
            }
            if (GRAD) copies_commit();
            x += down * q.x_tok;
            if (GRAD) g += down * q.g_tok;
        };
        int t = t0, now = position(t0), ahead = position(t0 + down);
        fetch(0, now);
        for (int round = 0; round < rounds; ++round, t += down) {
            const int pos = now, stage = round & 1;
            const bool keep = unsigned(pos) < unsigned(p.positions);
            const int live = t < tend ? heads : 0;
            uint4 cur[GRAD ? 1 : HB][NV][2];
            if constexpr (!GRAD) memcpy(cur, next, sizeof(cur));
            float2 c[NV][P], s[NV][P];
            if (rope) {
#pragma unroll
                for (int v = 0; v < NV; ++v) {
                    const int i = (v * G + gl) * V;
#pragma unroll
                    for (int k = 0; k < V / 4; ++k) {
                        uint4 w[2] = {zero, zero};
                        if (keep && (EXACT || i < half)) {
                            w[0] = *reinterpret_cast<const uint4 *>(p.rope_cos + (long long)pos * half + i + 4 * k);
                            w[1] = *reinterpret_cast<const uint4 *>(p.rope_sin + (long long)pos * half + i + 4 * k);
                        }
                        float2 f[2];
                        unpack2(w[0], f, 0.0f);
                        c[v][2 * k] = f[0], c[v][2 * k + 1] = f[1];
                        unpack2(w[1], f, 0.0f);
                        s[v][2 * k] = f[0], s[v][2 * k + 1] = f[1];
                    }
                }
            }
            now = ahead;
            ahead = position(t + 2 * down);
            fetch(stage ^ 1, now);
            if (GRAD) copies_wait<1>();
            const float2 minus = make_float2(-1.0f, -1.0f);
            // JOIN rows at a time: their sums first, so that the shuffles run side by side.
            constexpr int JOIN = GRAD ? 1 : HB;
#pragma unroll
            for (int h1 = 0; h1 < HB; h1 += JOIN) {
                float2 a[JOIN][NV][P], b[JOIN][NV][P], ga[GRAD ? JOIN : 1][NV][P], gb[GRAD ? JOIN : 1][NV][P];
                float ss[JOIN], ux[JOIN];
#pragma unroll
                for (int h = 0; h < JOIN; ++h) {
                    float2 ss2 = make_float2(0.0f, 0.0f), ux2 = make_float2(0.0f, 0.0f);
#pragma unroll
                    for (int v = 0; v < NV; ++v) {
                        const uint4 *at = ring + (stage * SLOTS + ((h1 + h) * NV + v) * 4) * 256;
                        unpack2(GRAD ? at[0] : cur[h][v][0], a[h][v], T());
                        unpack2(GRAD ? at[256] : cur[h][v][1], b[h][v], T());
#pragma unroll
                        for (int e = 0; e < P; ++e)
                            ss2 = fma2(a[h][v][e], a[h][v][e], fma2(b[h][v][e], b[h][v][e], ss2));
                        if constexpr (GRAD) {
                            unpack2(at[512], ga[h][v], T());
                            unpack2(at[768], gb[h][v], T());
#pragma unroll
                            for (int e = 0; e < P; ++e) {
                                float2 &da = ga[h][v][e], &db = gb[h][v][e];
                                if (rope) {
                                    const float2 turned = fma2(db, s[v][e], mul2(da, c[v][e]));
                                    db = fma2(mul2(da, s[v][e]), minus, mul2(db, c[v][e]));
                                    da = turned;
                                }
                                ux2 = fma2(mul2(da, wl[v][e]), a[h][v][e], ux2);
                                ux2 = fma2(mul2(db, wh[v][e]), b[h][v][e], ux2);
                            }
                        }
                    }
                    ss[h] = ss2.x + ss2.y, ux[h] = ux2.x + ux2.y;
                }
#pragma unroll
                for (int o = G / 2; o; o >>= 1) {
#pragma unroll
                    for (int h = 0; h < JOIN; ++h) {
                        ss[h] += __shfl_xor_sync(0xffffffffu, ss[h], o);
                        if (GRAD) ux[h] += __shfl_xor_sync(0xffffffffu, ux[h], o);
                    }
                }
#pragma unroll
                for (int h = 0; h < JOIN; ++h) {
                    // rsqrtf (two units of fp32) and 1 / d rounded once: below every 16-bit
                    // type's rounding; an fp32 gradient is 1.5e-7 off, a plain form's 1.4e-7.
                    // A block's missing heads are rows of zeros: r = 0 there, for without
                    // eps it would be infinite, and 0 * r would enter the weights' gradients.
                    const float r = keep && h1 + h < live ? rsqrtf(ss[h] * inv_d + p.eps) : 0.0f;
                    const float m = GRAD ? -r * (r * r * (ux[h] * inv_d)) : 0.0f;
                    const float2 r2 = make_float2(r, r), m2 = make_float2(m, m);
#pragma unroll
                    for (int v = 0; v < NV; ++v) {
                        float2 oa[P], ob[P];
#pragma unroll
                        for (int e = 0; e < P; ++e) {
                            if constexpr (GRAD) {
                                dl[v][e] = fma2(ga[h][v][e], mul2(a[h][v][e], r2), dl[v][e]);
                                dh[v][e] = fma2(gb[h][v][e], mul2(b[h][v][e], r2), dh[v][e]);
                                oa[e] = fma2(a[h][v][e], m2, mul2(mul2(ga[h][v][e], wl[v][e]), r2));
                                ob[e] = fma2(b[h][v][e], m2, mul2(mul2(gb[h][v][e], wh[v][e]), r2));
                            } else {
                                const float2 ya = mul2(mul2(a[h][v][e], r2), wl[v][e]);
                                const float2 yb = mul2(mul2(b[h][v][e], r2), wh[v][e]);
                                oa[e] = ya, ob[e] = yb;
                                if (rope) {
                                    oa[e] = fma2(mul2(yb, s[v][e]), minus, mul2(ya, c[v][e]));
                                    ob[e] = fma2(ya, s[v][e], mul2(yb, c[v][e]));
                                }
                            }
                        }
                        if (h1 + h < live && (EXACT || (v * G + gl) * V < half)) {
                            uint4 lo = packed(oa, T()), hi = packed(ob, T());
                            if (!keep) lo = hi = zero;
                            T *dst = out + (h1 + h) * q.out_head + v * G * V;
                            *reinterpret_cast<uint4 *>(dst) = lo;
                            *reinterpret_cast<uint4 *>(dst + half) = hi;
                        }
                    }
                }
            }
            out += down * q.out_tok;
        }
        if (GRAD) copies_wait<0>();  // what was fetched behind the last item
    }
    if constexpr (GRAD) {
        // The CTA's groups in order, into one partial row of d per CTA.
        if (!p.dw || kind == 2) return;
        __syncthreads();
        const int grp = threadIdx.x / G;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int i = (v * G + gl) * V;
            if (EXACT || i < half) {
#pragma unroll
                for (int e = 0; e < P; ++e) {
                    *reinterpret_cast<float2 *>(sums + grp * p.d + i + 2 * e) = dl[v][e];
                    *reinterpret_cast<float2 *>(sums + grp * p.d + half + i + 2 * e) = dh[v][e];
                }
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < p.d; i += 256) {
            float sum = 0.0f;
            for (int r = 0; r < 256 / G; ++r) sum += sums[r * p.d + i];
            p.dw[(size_t)blockIdx.x * p.d + i] = sum;
        }
    }
}

// The gradient for rows that are not whole 16-byte vectors: a warp per row, one
// element of each half per lane at a time, the CTAs shared out as above.
template <typename T>
__global__ void __launch_bounds__(256) qkv_norm_grad_kernel(const __grid_constant__ QkvNormParams p) {
    constexpr int NV = 8;
    __shared__ float sums[8][512];
    pdl_wait();
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = p.d / 2;
    int kind = 0;
    while (int(blockIdx.x) >= p.cta_end[kind]) ++kind;
    const QkvPart &q = p.part[kind];
    const int cta0 = kind ? p.cta_end[kind - 1] : 0;
    const long long items = (long long)p.n * q.heads, step = (long long)(p.cta_end[kind] - cta0) * 8;
    float dl[NV], dh[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) dl[v] = dh[v] = 0.0f;
    for (long long item = (long long)(blockIdx.x - cta0) * 8 + warp; item < items; item += step) {
        const int t = int(item / q.heads), h = int(item - (long long)t * q.heads), pos = p.pos[t];
        const bool keep = unsigned(pos) < unsigned(p.positions);
        const T *x = static_cast<const T *>(q.x) + t * q.x_tok + h * q.x_head;
        const T *g = static_cast<const T *>(q.g) + t * q.g_tok + h * q.g_head;
        T *out = static_cast<T *>(q.out) + t * q.out_tok + h * q.out_head;
        float a[NV], b[NV], ga[NV], gb[NV], ss = 0.0f, ux = 0.0f;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int i = v * 32 + lane;
            a[v] = b[v] = ga[v] = gb[v] = 0.0f;
            if (!keep || i >= half) continue;
            a[v] = to_f32(x[i]), b[v] = to_f32(x[half + i]);
            const float oa = to_f32(g[i]), ob = to_f32(g[half + i]);
            const float c = kind < 2 ? p.rope_cos[(long long)pos * half + i] : 1.0f;
            const float s = kind < 2 ? p.rope_sin[(long long)pos * half + i] : 0.0f;
            ga[v] = oa * c + ob * s, gb[v] = ob * c - oa * s;
            float wl[1] = {1.0f}, wh[1] = {1.0f};
            if (q.w) load_weight<T, 1>(wl, q.w, i, p.weight_f32), load_weight<T, 1>(wh, q.w, half + i, p.weight_f32);
            ss = fmaf(a[v], a[v], fmaf(b[v], b[v], ss));
            ux = fmaf(ga[v] * wl[0], a[v], fmaf(gb[v] * wh[0], b[v], ux));
        }
        ss = group_sum<32>(ss), ux = group_sum<32>(ux);
        const float r = keep ? __frsqrt_rn(ss / float(p.d) + p.eps) : 0.0f;
        const float m = r * r * (ux / float(p.d));
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int i = v * 32 + lane;
            if (i >= half) continue;
            dl[v] += ga[v] * (a[v] * r), dh[v] += gb[v] * (b[v] * r);
            float wl[1] = {1.0f}, wh[1] = {1.0f};
            if (q.w) load_weight<T, 1>(wl, q.w, i, p.weight_f32), load_weight<T, 1>(wh, q.w, half + i, p.weight_f32);
            out[i] = from_f32<T>(keep ? r * (ga[v] * wl[0] - a[v] * m) : 0.0f);
            out[half + i] = from_f32<T>(keep ? r * (gb[v] * wh[0] - b[v] * m) : 0.0f);
        }
    }
    if (!p.dw || kind == 2) return;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int i = v * 32 + lane;
        if (i < half) sums[warp][i] = dl[v], sums[warp][half + i] = dh[v];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < p.d; i += 256) {
        float sum = 0.0f;
        for (int w = 0; w < 8; ++w) sum += sums[w][i];
        p.dw[(size_t)blockIdx.x * p.d + i] = sum;
    }
}

struct QkvDwParams {
    void *dw[2];       // queries', keys'; null: not wanted
    const float *part;  // [rows][d]: queries' rows end at row_end[0], keys' at row_end[1]
    int row_end[2], d, f32, accumulate;
};
// Column sums of the partial rows: 32 columns of one weight per CTA, each of its 32
// warps every 32nd row (all its loads in flight), then the warps' sums in order.
template <typename T>
__global__ void __launch_bounds__(1024) qkv_dw_kernel(const QkvDwParams p) {
    __shared__ float sums[32][33];
    pdl_wait();
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, k = blockIdx.y, col = blockIdx.x * 32 + lane;
    if (!p.dw[k]) return;
    float s = 0.0f;
    if (col < p.d) {
#pragma unroll 8
        for (int r = (k ? p.row_end[0] : 0) + warp; r < p.row_end[k]; r += 32) s += p.part[(size_t)r * p.d + col];
    }
    sums[warp][lane] = s;
    __syncthreads();
    if (warp || col >= p.d) return;
#pragma unroll
    for (int w = 1; w < 32; ++w) s += sums[w][lane];
    if (p.f32) {
        float *o = static_cast<float *>(p.dw[k]) + col;
        *o = p.accumulate ? *o + s : s;
    } else {
        T *o = static_cast<T *>(p.dw[k]) + col;
        *o = from_f32<T>(p.accumulate ? to_f32(*o) + s : s);
    }
}

}  // namespace eg2
