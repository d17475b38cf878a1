// Launchers and C entry points (include/eg2_ops.h, part 3) of the typed row
// operators: argument checks, the choice of a kernel by type, width and
// alignment, and workspace layout.  Included once, at the end of kernels.cu.
#pragma once
#include "embedrows.cuh"
#include "qkvnorm.cuh"

namespace eg2 {

static inline int type_size(unsigned t) { return t == EG_F32 ? 4 : t == EG_F16 || t == EG_BF16 ? 2 : 0; }
static inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
static inline int ceil_div(long long a, long long b) { return int((a + b - 1) / b); }

template <int I>
struct Int {
    static constexpr int value = I;
};
// f(type tag) for an element type; cudaErrorInvalidValue for any other number.
template <typename T>
struct Tag {
    using type = T;
};
template <typename F>
static cudaError_t by_type(unsigned t, F f) {
    switch (t) {
        case EG_F32: return f(Tag<float>{});
        case EG_F16: return f(Tag<__half>{});
        case EG_BF16: return f(Tag<__nv_bfloat16>{});
        default: return cudaErrorInvalidValue;
    }
}

// Opts one kernel into its dynamic shared memory, once per device.
struct AllowSmem {
    std::mutex mu;
    bool done[64] = {};
    template <typename K>
    cudaError_t operator()(K kernel, int bytes) {
        int dev = 0;
        if (cudaError_t e = cudaGetDevice(&dev)) return e;
        std::lock_guard<std::mutex> g(mu);
        if (dev < 64 && done[dev]) return cudaSuccess;
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (!e && dev < 64) done[dev] = true;
        return e;
    }
};

// Whether vectors of `bytes` bytes (of `size`-byte elements) fit every one of `rows` rows at p.
static bool rows_fit(const void *p, long long stride, unsigned rows, int bytes, int size) {
    const int w = bytes < 16 ? bytes : 16;
    return reinterpret_cast<uintptr_t>(p) % w == 0 && (rows < 2 || stride * size % w == 0);
}

// ---------------------------------------------------------------- embed_rows
static cudaError_t embed_rows(const EgEmbedRows &a, cudaStream_t s) {
    const int so = type_size(a.out_type), st = type_size(a.table_type);
    if (!so || !st || !a.d || a.d > (1u << 20) || a.n > 0x7fffffffu || a.vocab > 0x7ffffffeu)
        return cudaErrorInvalidValue;
    if (!a.n) return cudaSuccess;
    if (!a.out || !a.ids || (a.vocab && !a.table) || (a.n > 1 && a.out_stride < (int64_t)a.d) ||
        (a.vocab > 1 && a.table_stride < (int64_t)a.d))
        return cudaErrorInvalidValue;
    const EmbedRowsParams p{a.out, a.table, a.ids, a.out_stride, a.table_stride, int(a.n), int(a.vocab), int(a.d),
                            a.scale};
    return by_type(a.table_type, [&](auto ti) {
        return by_type(a.out_type, [&](auto to) {
            using TI = typename decltype(ti)::type;
            using TO = typename decltype(to)::type;
            const auto fit = [&](int v) {
                return a.d % v == 0 && rows_fit(a.out, a.out_stride, a.n, v * so, so) &&
                       rows_fit(a.table, a.table_stride, a.vocab, v * st, st);
            };
            const dim3 grid(ceil_div(a.n, 8));
            if (fit(8)) return launch_pdl(embed_rows_kernel<TI, TO, 8>, grid, dim3(256), 0, s, p);
            if (fit(2)) return launch_pdl(embed_rows_kernel<TI, TO, 2>, grid, dim3(256), 0, s, p);
            return launch_pdl(embed_rows_kernel<TI, TO, 1>, grid, dim3(256), 0, s, p);
        });
    });
}

// Workspace: two arrays of (key, token), the digit histogram, the touched rows' flags,
// and the head and tail parts of every chunk.
struct EmbedGradLayout {
    int tiles, subtiles, chunk, chunks;
    size_t items[2], hist, touched, head, tail, total;
};
static EmbedGradLayout embed_grad_layout(unsigned n, unsigned d) {
    EmbedGradLayout L{};
    // About 8 warps on each of 148 SMs, a warp for 256 columns of a chunk; 8 items at
    // least, and no more than there are (a share passes 2^31 for many wide rows).
    const long long warps = 8 * 148, share = ((long long)n * ceil_div(d, 256) + warps - 1) / warps;
    L.chunk = int(((share < 8 ? 8 : share > n ? n : share) + 7) / 8 * 8);
    L.chunks = ceil_div(n, L.chunk);
    L.subtiles = ceil_div(n, (long long)EmbedSort::SUB * EmbedSort::MAX_TILES);
    if (L.subtiles < 1) L.subtiles = 1;
    L.tiles = ceil_div(n, (long long)EmbedSort::SUB * L.subtiles);
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    for (int i = 0; i < 2; ++i) L.items[i] = take(size_t(n) * 8);
    L.hist = take(size_t(L.tiles) * EmbedSort::MAX_BINS * 4);
    L.touched = take(EmbedSort::MAX_TOUCHED);
    L.head = take(size_t(L.chunks) * d * 4);
    L.tail = take(size_t(L.chunks) * d * 4);
    L.total = at;
    return L;
}

static cudaError_t embed_rows_grad(const EgEmbedRowsGrad &a, cudaStream_t s) {
    const int sw = type_size(a.dtable_type), sg = type_size(a.dout_type);
    if (!sw || !sg || !a.d || a.d > (1u << 20) || a.n > (1u << 30) || a.vocab > 0x7ffffffeu)
        return cudaErrorInvalidValue;
    if (!a.vocab || (!a.n && a.accumulate)) return cudaSuccess;
    if (!a.dtable || (a.vocab > 1 && a.dtable_stride < (int64_t)a.d)) return cudaErrorInvalidValue;
    const long long stride = a.vocab > 1 ? a.dtable_stride : a.d;
    if (!a.n)
        return cudaMemset2DAsync(a.dtable, size_t(stride) * sw, 0, size_t(a.d) * sw, a.vocab, s);
    const EmbedGradLayout L = embed_grad_layout(a.n, a.d);
    if (!a.dout || !a.ids || !a.workspace || a.workspace_bytes < L.total ||
        (reinterpret_cast<uintptr_t>(a.workspace) & 255) || a.dout_stride < 0)
        return cudaErrorInvalidValue;
    uint8_t *ws = static_cast<uint8_t *>(a.workspace);
    uint2 *items[2] = {reinterpret_cast<uint2 *>(ws + L.items[0]), reinterpret_cast<uint2 *>(ws + L.items[1])};

    // Keys are 0 .. vocab (padding last); equal digits over as few passes as cover them.
    int key_bits = 1;
    while (key_bits < 31 && (a.vocab >> key_bits)) ++key_bits;
    const int passes = ceil_div(key_bits, EmbedSort::MAX_BITS), bits = ceil_div(key_bits, passes);
    EmbedSortParams q{};
    q.hist = reinterpret_cast<unsigned *>(ws + L.hist);
    q.n = int(a.n), q.vocab = int(a.vocab), q.tiles = L.tiles, q.subtiles = L.subtiles, q.bits = bits;
    // The table's untouched rows are cleared beside the other work: beside the sort
    // about what can be written in the time that it takes anyway, the rest beside the
    // sums.  262144 x 512 bf16, uniform ids: 96 MB beside the small sort 49 us at 1999
    // tokens and 52 at 4096, with 48 MB 50 and 58, with none 58 and 65; 64 MB a scatter
    // 59 us at 5000 tokens and 71 at 40000, with none 65 and 75, at 100003 95 either
    // way, at 300000 167 against 157, where the sums have the time.  (Natural ids at
    // 100003: 93 us, 95 with 32 or 134 MB, 96 also beside the histograms.)  A larger
    // vocabulary than there are flags for is cleared whole before the sums.
    const bool flags_fit = a.vocab <= EmbedSort::MAX_TOUCHED;
    uint8_t *touched = a.accumulate || !flags_fit ? nullptr : ws + L.touched;
    const long long block_bytes = 8ll * a.d * sw;
    long long left = ceil_div(a.vocab, 8);  // blocks of 8 rows, handed out from the end
    auto share = [&](long long bytes, int warps, bool skip) {
        EmbedFill f{};
        if (a.accumulate) return f;
        long long count = bytes < 0 ? left : bytes / block_bytes;
        if (count > left) count = left;
        f.table = static_cast<unsigned char *>(a.dtable), f.touched = skip ? touched : nullptr;
        f.stride = stride * sw, f.width = int(a.d) * sw, f.rows = int(a.vocab);
        // Short CTAs, about 16 KB a warp, but enough of them for every SM.
        const long long per_warp = block_bytes >= 16384 ? 1 : 16384 / block_bytes;
        long long ctas = (count + warps * per_warp - 1) / (warps * per_warp);
        if (ctas < sm_count()) ctas = count < sm_count() ? count : sm_count();
        f.each = int(ctas ? (count + ctas - 1) / ctas : 0);
        f.ctas = f.each ? ceil_div(count, f.each) : 0;
        left -= count;
        f.block0 = left, f.blocks = count;
        return f;
    };
    int sorted = passes & 1;  // which pair of arrays ends up holding the items in order
    if (a.n <= EmbedSmall::CAP) {
        using S = EmbedSmall;
        EmbedSmallParams c{};
        sorted = 0;
        c.ids = a.ids, c.out = items[0], c.touched = touched;
        c.n = q.n, c.vocab = q.vocab, c.bits = bits, c.passes = passes, c.per = ceil_div(a.n, S::THREADS);
        c.fill = share(flags_fit ? 96 << 20 : -1, S::WARPS, false);
        static AllowSmem allow;
        if (cudaError_t e = allow(embed_sort_kernel, S::SMEM)) return e;
        if (cudaError_t e = launch_pdl(embed_sort_kernel, dim3(1 + c.fill.ctas), dim3(S::THREADS), S::SMEM, s, c))
            return e;
    } else {
        for (int pass = 0; pass < passes; ++pass) {
            q.ids = pass ? nullptr : a.ids;
            q.in = items[pass & 1], q.out = items[(pass + 1) & 1];
            q.shift = pass * bits;
            for (int half = 0; half < 2; ++half) {
                const bool last = pass == passes - 1 && half;
                q.touched = pass == passes - 1 ? touched : nullptr;
                q.fill = share(last && !flags_fit ? -1 : half ? 64 << 20 : 0, EmbedSort::WARPS, false);
                if (cudaError_t e = launch_pdl(half ? embed_scatter_kernel : embed_hist_kernel,
                                               dim3(L.tiles + q.fill.ctas), dim3(EmbedSort::THREADS), 0, s, q))
                    return e;
            }
        }
    }
    EmbedSumParams u{};
    u.dtable = a.dtable, u.dout = a.dout, u.items = items[sorted];
    u.head = reinterpret_cast<float *>(ws + L.head), u.tail = reinterpret_cast<float *>(ws + L.tail);
    u.dtable_stride = stride, u.dout_stride = a.dout_stride;
    u.n = int(a.n), u.vocab = int(a.vocab), u.d = int(a.d), u.chunk = L.chunk, u.chunks = L.chunks;
    u.scale = a.scale, u.accumulate = a.accumulate != 0;
    u.fill = share(-1, EmbedSum::WARPS, true);
    // 16 bytes of dout per lane and row where all rows allow it, else pairs, else single elements.
    const auto fit = [&](int v) {
        return a.d % v == 0 && rows_fit(a.dout, a.dout_stride, a.n, v * sg, sg) &&
               rows_fit(a.dtable, stride, a.vocab, v * sw, sw);
    };
    return by_type(a.dout_type, [&](auto tg) {
        return by_type(a.dtable_type, [&](auto tw) {
            using TG = typename decltype(tg)::type;
            using TW = typename decltype(tw)::type;
            const auto go = [&](auto vec) -> cudaError_t {
                constexpr int V = decltype(vec)::value;
                u.col_blocks = ceil_div(a.d, 32 * V);
                u.sum_ctas = ceil_div((long long)L.chunks * u.col_blocks, EmbedSum::WARPS);
                const size_t ring = V * sizeof(TG) == 16 ? EmbedSum::RING : 0;  // 48 KB: no opt-in needed
                if (cudaError_t e = launch_pdl(embed_sum_kernel<TG, TW, V>, dim3(u.sum_ctas + u.fill.ctas),
                                               dim3(EmbedSum::THREADS), ring, s, u))
                    return e;
                if (L.chunks < 2) return cudaSuccess;
                return launch_pdl(embed_join_kernel<TW, V>, dim3(ceil_div(L.chunks, 32), u.col_blocks), dim3(256), 0, s, u);
            };
            constexpr int WIDE = 16 / int(sizeof(TG));
            return fit(WIDE) ? go(Int<WIDE>{}) : fit(2) ? go(Int<2>{}) : go(Int<1>{});
        });
    });
}

// ---------------------------------------------------------------- qkv_norm_rope
constexpr int QKV_MAX_PARTS = 1024;  // at least the gradient's CTAs (two per SM), one partial row each

// Checks one tensor's strides (elements) and says whether whole 16-byte vectors fit it.
static bool qkv_tensor_ok(const void *p, int64_t tok, int64_t head, unsigned n, unsigned heads, unsigned d, int size,
                          bool written, bool *wide) {
    if (!p || tok < 0 || head < 0) return false;
    // Rows that are written must not overlap: in one order of the two strides each has room for the other.
    if (written) {
        const int64_t span = heads > 1 ? head * (heads - 1) + d : d, tspan = n > 1 ? tok * (int64_t(n) - 1) + d : d;
        const bool by_tok = (heads < 2 || head >= d) && (n < 2 || tok >= span);
        const bool by_head = (n < 2 || tok >= d) && (heads < 2 || head >= tspan);
        if (!by_tok && !by_head) return false;
    }
    if (!aligned16(p) || (n > 1 && tok * size % 16) || (heads > 1 && head * size % 16)) *wide = false;
    return true;
}

// f(V, G, NV) as integral constants for a row of half = d / 2 elements of T.
template <typename T, typename F>
static cudaError_t qkv_shape(int half, bool wide, F f) {
    constexpr int V = 16 / int(sizeof(T));
    if (!wide || half % V) return f(Int<1>{}, Int<32>{}, Int<8>{});
    const int vecs = half / V;
    if (vecs <= 4) return f(Int<V>{}, Int<4>{}, Int<1>{});
    if (vecs <= 8) return f(Int<V>{}, Int<8>{}, Int<1>{});
    if (vecs <= 16) return f(Int<V>{}, Int<16>{}, Int<1>{});
    if (vecs <= 32) return f(Int<V>{}, Int<32>{}, Int<1>{});
    if constexpr (sizeof(T) == 4) return f(Int<V>{}, Int<32>{}, Int<2>{});
    return cudaErrorInvalidValue;
}

static cudaError_t qkv_common(QkvNormParams *p, bool *wide, unsigned n, const unsigned heads[3], unsigned d,
                              unsigned type, unsigned weight_type, unsigned positions, const void *const x[3],
                              const int64_t xs[3][2], void *const out[3], const int64_t outs[3][2],
                              const void *const weight[2], const float *rc, const float *rs, const int *pos,
                              float eps) {
    const int size = type_size(type);
    if (!size || !d || d > 512 || d % 2 || n > (1u << 30) || positions > 0x7fffffffu ||
        (weight_type != EG_F32 && weight_type != type))
        return cudaErrorInvalidValue;
    *wide = true;
    *p = QkvNormParams{};
    for (int i = 0; i < 3; ++i) {
        QkvPart &q = p->part[i];
        if (heads[i] > 65536) return cudaErrorInvalidValue;
        q.heads = int(heads[i]);
        if (!heads[i] || !n) continue;
        if (!qkv_tensor_ok(x[i], xs[i][0], xs[i][1], n, heads[i], d, size, false, wide) ||
            !qkv_tensor_ok(out[i], outs[i][0], outs[i][1], n, heads[i], d, size, true, wide))
            return cudaErrorInvalidValue;
        q.x = x[i], q.out = out[i], q.w = i < 2 ? weight[i] : nullptr;
        q.x_tok = xs[i][0], q.x_head = xs[i][1], q.out_tok = outs[i][0], q.out_head = outs[i][1];
        if (q.w && !aligned16(q.w)) *wide = false;
        if (i < 2) {
            if (positions && (!rc || !rs)) return cudaErrorInvalidValue;  // no rows: never read
            if (!aligned16(rc) || !aligned16(rs)) *wide = false;
        }
    }
    if (n && !pos) return cudaErrorInvalidValue;
    // At least 8 rows a CTA in both directions: fewer than 2^31 CTAs, or items of them.
    if (((long long)n * (p->part[0].heads + p->part[1].heads + p->part[2].heads)) >> 33) return cudaErrorInvalidValue;
    p->rope_cos = rc, p->rope_sin = rs, p->pos = pos;
    p->n = int(n), p->d = int(d), p->positions = int(positions), p->weight_f32 = weight_type == EG_F32, p->eps = eps;
    return cudaSuccess;
}
// Shares a grid of at most `most` CTAs, each taking `per` items at a time, out
// among the kinds by their work: an item's rows, and about half a row for the item itself.
static int qkv_share(QkvNormParams *p, int hb, int per, int most) {
    long long work[3], total = 0;
    int need[3], cta[3], want = 0, big = 0;
    for (int i = 0; i < 3; ++i) {
        QkvPart &q = p->part[i];
        q.blocks = ceil_div(q.heads, hb);
        work[i] = 2 * q.heads + q.blocks;
        total += work[i];
        need[i] = q.heads ? ceil_div((long long)p->n * q.blocks, per) : 0;
        if (work[i] > work[big]) big = i;
    }
    for (int i = 0; i < 3; ++i) {
        const long long share = work[i] * most / total;
        cta[i] = int(share < need[i] ? share : need[i]);
        if (!cta[i] && need[i]) cta[i] = 1;
        want += cta[i];
    }
    const int left = need[big] - cta[big] < most - want ? need[big] - cta[big] : most - want;
    if (left > 0) cta[big] += left;
    for (int i = 0, end = 0; i < 3; ++i) p->cta_end[i] = end += cta[i];
    return p->cta_end[2];
}
template <typename T, int G, int NV, bool GRAD>
static cudaError_t qkv_stream(QkvNormParams &p, cudaStream_t s) {
    constexpr int V = 16 / int(sizeof(T)), HB = 2 / NV;
    const int ctas = qkv_share(&p, HB, 256 / G, 2 * sm_count());
    constexpr size_t smem = GRAD ? 2 * 8 * 256 * 16 : 0;  // two stages of 8 vectors per thread
    const auto go = [&](auto kernel, AllowSmem &allow) -> cudaError_t {
        if (GRAD)
            if (cudaError_t e = allow(kernel, int(smem))) return e;
        return launch_pdl(kernel, dim3(ctas), dim3(256), smem, s, p);
    };
    static AllowSmem exact, other;
    return p.d / 2 == G * NV * V ? go(qkv_stream_kernel<T, G, NV, HB, GRAD, true>, exact)
                                 : go(qkv_stream_kernel<T, G, NV, HB, GRAD, false>, other);
}

static cudaError_t qkv_norm_rope(const EgQkvNormRope &a, cudaStream_t s) {
    QkvNormParams p;
    bool wide;
    const unsigned heads[3] = {a.q_heads, a.k_heads, a.v_heads};
    if (cudaError_t e = qkv_common(&p, &wide, a.n, heads, a.d, a.type, a.weight_type, a.positions, a.x, a.x_stride,
                                   a.out, a.out_stride, a.weight, a.rope_cos, a.rope_sin, a.pos, a.eps))
        return e;
    const long long rows = (long long)p.n * (p.part[0].heads + p.part[1].heads + p.part[2].heads);
    if (!rows) return cudaSuccess;
    return by_type(a.type, [&](auto t) {
        using T = typename decltype(t)::type;
        return qkv_shape<T>(p.d / 2, wide, [&](auto v, auto g, auto nv) {
            constexpr int V = decltype(v)::value, G = decltype(g)::value, NV = decltype(nv)::value;
            // Rows enough to go round the streaming form's grid more than once, else direct.
            if constexpr (V > 1)
                if (rows * G > 2ll * sm_count() * 256 * 4) return qkv_stream<T, G, NV, false>(p, s);
            return launch_pdl(qkv_norm_kernel<T, V, G, NV>, dim3(ceil_div(rows, 256 / G)), dim3(256), 0, s, p);
        });
    });
}

static cudaError_t qkv_norm_rope_grad(const EgQkvNormRopeGrad &a, cudaStream_t s) {
    QkvNormParams p;
    bool wide;
    const unsigned heads[3] = {a.q_heads, a.k_heads, a.v_heads};
    if (cudaError_t e = qkv_common(&p, &wide, a.n, heads, a.d, a.type, a.weight_type, a.positions, a.x, a.x_stride,
                                   a.dx, a.dx_stride, a.weight, a.rope_cos, a.rope_sin, a.pos, a.eps))
        return e;
    for (int i = 0; i < 3; ++i) {
        if (!heads[i] || !a.n) continue;
        QkvPart &q = p.part[i];
        if (!qkv_tensor_ok(a.dout[i], a.dout_stride[i][0], a.dout_stride[i][1], a.n, heads[i], a.d,
                           type_size(a.type), false, &wide))
            return cudaErrorInvalidValue;
        q.g = a.dout[i], q.g_tok = a.dout_stride[i][0], q.g_head = a.dout_stride[i][1];
    }
    const bool want_dw = a.dweight[0] || a.dweight[1];
    const bool any = p.n && (a.q_heads + a.k_heads + a.v_heads);
    if (!any && (!want_dw || a.accumulate)) return cudaSuccess;
    const uint64_t need = eg2_qkv_norm_rope_grad_workspace(
        a.n, a.q_heads, a.k_heads > a.v_heads ? a.k_heads : a.v_heads, a.d);
    if (want_dw && any && (!a.workspace || a.workspace_bytes < need || (reinterpret_cast<uintptr_t>(a.workspace) & 255)))
        return cudaErrorInvalidValue;
    p.dw = want_dw ? static_cast<float *>(a.workspace) : nullptr;
    return by_type(a.type, [&](auto t) {
        using T = typename decltype(t)::type;
        if (any) {
            const cudaError_t e = qkv_shape<T>(p.d / 2, wide, [&](auto v, auto g, auto nv) {
                constexpr int V = decltype(v)::value, G = decltype(g)::value, NV = decltype(nv)::value;
                if constexpr (V > 1) return qkv_stream<T, G, NV, true>(p, s);
                const int ctas = qkv_share(&p, 1, 8, 2 * sm_count());
                return launch_pdl(qkv_norm_grad_kernel<T>, dim3(ctas), dim3(256), 0, s, p);
            });
            if (e || !want_dw) return e;
        }
        const QkvDwParams w{{a.dweight[0], a.dweight[1]}, p.dw, {p.cta_end[0], p.cta_end[1]}, p.d, p.weight_f32,
                            int(a.accumulate != 0)};
        return launch_pdl(qkv_dw_kernel<T>, dim3(ceil_div(p.d, 32), 2), dim3(1024), 0, s, w);
    });
}

}  // namespace eg2

extern "C" {
int eg2_launch_embed_rows(const EgEmbedRows *p, void *s) { return rc(embed_rows(*p, S(s))); }
uint64_t eg2_embed_rows_grad_workspace(unsigned n, unsigned d) { return n && d ? embed_grad_layout(n, d).total : 0; }
int eg2_launch_embed_rows_grad(const EgEmbedRowsGrad *p, void *s) { return rc(embed_rows_grad(*p, S(s))); }
int eg2_launch_qkv_norm_rope(const EgQkvNormRope *p, void *s) { return rc(qkv_norm_rope(*p, S(s))); }
uint64_t eg2_qkv_norm_rope_grad_workspace(unsigned n, unsigned q_heads, unsigned kv_heads, unsigned d) {
    // A CTA, and so a partial row, holds at least one head of one token.
    const uint64_t rows = uint64_t(n) * (uint64_t(q_heads) + 2 * uint64_t(kv_heads));
    return (rows < QKV_MAX_PARTS ? rows : QKV_MAX_PARTS) * d * 4;
}
int eg2_launch_qkv_norm_rope_grad(const EgQkvNormRopeGrad *p, void *s) { return rc(qkv_norm_rope_grad(*p, S(s))); }
}
