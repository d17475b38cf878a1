// Embedding lookup with scaling, and its gradient.
//
//   out[t] = scale * table[ids[t]]                       (embed_rows_kernel)
//   dtable[v] (+)= scale * sum over ids[t] = v of dout[t]  (the kernels below it)
//
// An id outside [0, vocab) marks padding: its output row is zero and its
// gradient row is not read.
//
// The gradient sorts the (id, token) pairs by id, stably, so that each id's rows
// are summed in token order whatever else is in the batch, with no atomics on
// values: the result is the same bits on every run.  All of it is bound by
// memory: ids and dout are read once, each touched row is written once.
#pragma once
#include "typed.cuh"

namespace eg2 {

struct EmbedRowsParams {
    void *out;
    const void *table;
    const int *ids;
    long long out_stride, table_stride;
    int n, vocab, d;
    float scale;
};

// A warp takes ROWS tokens and walks their columns 32 vectors at a time, so that
// ROWS independent row reads are in flight per lane.
template <typename TIn, typename TOut, int V, int ROWS>
__global__ void __launch_bounds__(256) embed_rows_kernel(const EmbedRowsParams p) {
    pdl_wait();
    pdl_trigger();
    const int warp = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    const long long t0 = (long long)warp * ROWS;
    const TIn *src[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        const int id = t0 + r < p.n ? p.ids[t0 + r] : -1;
        src[r] = unsigned(id) < unsigned(p.vocab) ? static_cast<const TIn *>(p.table) + id * p.table_stride : nullptr;
    }
    for (int c = lane * V; c < p.d; c += 32 * V) {
        Pack<TIn, V> x[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            if (src[r]) x[r].load(src[r] + c);
            else x[r].zero();
        }
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            if (t0 + r >= p.n) break;
            float f[V];
            x[r].get(f);
#pragma unroll
            for (int i = 0; i < V; ++i) f[i] = src[r] ? f[i] * p.scale : 0.0f;
            Pack<TOut, V> y;
            y.set(f);
            y.store(static_cast<TOut *>(p.out) + (t0 + r) * p.out_stride + c);
        }
    }
}

// ---------------------------------------------------------------- the gradient's sort
// Least-significant-digit radix sort of (id, token) by id: `passes` passes of
// `bits` bits (at most 10), each a histogram launch and a scatter launch.  The
// tokens are cut into tiles of SUB * subtiles consecutive items, one CTA each.
// Padding gets the key `vocab`, behind every id.
struct EmbedSort {
    static constexpr int THREADS = 256, WARPS = 8, PER = 8, SUB = THREADS * PER, MAX_BITS = 10,
                         MAX_BINS = 1 << MAX_BITS, MAX_TILES = 128;
};
struct EmbedSortParams {
    const int *ids;             // the first pass reads these, with the token index implied
    const unsigned *key_in;     // later passes
    const int *tok_in;
    unsigned *key_out;
    int *tok_out;
    unsigned *hist;             // [tiles][bins] of this pass
    int n, vocab, tiles, subtiles, shift, bits;
    // A share of the table to clear meanwhile (none when fill_rows is 0): CTAs
    // behind the tiles write zeros over rows [fill_row0, fill_row0 + fill_rows).
    unsigned char *fill;
    long long fill_row0, fill_rows, fill_stride_bytes;
    int fill_width_bytes, fill_ctas;
};
__device__ __forceinline__ unsigned embed_sort_key(const EmbedSortParams &p, int i) {
    if (!p.ids) return p.key_in[i];
    const unsigned id = unsigned(p.ids[i]);
    return id < unsigned(p.vocab) ? id : unsigned(p.vocab);
}
// Zeros over this launch's share of the rows, by `fill_ctas` CTAs.  A share
// without gaps between its rows is one flat range; otherwise a CTA takes whole rows.
__device__ __forceinline__ void embed_fill(const EmbedSortParams &p, int cta) {
    unsigned char *base = p.fill + p.fill_row0 * p.fill_stride_bytes;
    const bool flat = p.fill_stride_bytes == p.fill_width_bytes && (reinterpret_cast<uintptr_t>(base) & 15) == 0;
    const uint4 z = make_uint4(0, 0, 0, 0);
    if (flat) {
        const long long bytes = p.fill_rows * p.fill_stride_bytes, vecs = bytes / 16;
        const long long step = (long long)p.fill_ctas * blockDim.x;
        for (long long i = (long long)cta * blockDim.x + threadIdx.x; i < vecs; i += step)
            reinterpret_cast<uint4 *>(base)[i] = z;
        if (cta == 0)
            for (long long i = vecs * 16 + threadIdx.x * 2; i < bytes; i += blockDim.x * 2)
                *reinterpret_cast<uint16_t *>(base + i) = 0;
        return;
    }
    for (long long r = cta; r < p.fill_rows; r += p.fill_ctas) {
        unsigned char *row = base + r * p.fill_stride_bytes;
        if (((reinterpret_cast<uintptr_t>(row) | unsigned(p.fill_width_bytes)) & 15) == 0)
            for (int i = threadIdx.x * 16; i < p.fill_width_bytes; i += blockDim.x * 16)
                *reinterpret_cast<uint4 *>(row + i) = z;
        else
            for (int i = threadIdx.x * 2; i < p.fill_width_bytes; i += blockDim.x * 2)
                *reinterpret_cast<uint16_t *>(row + i) = 0;
    }
}
__global__ void __launch_bounds__(EmbedSort::THREADS) embed_hist_kernel(const EmbedSortParams p) {
    pdl_wait();
    pdl_trigger();
    if (int(blockIdx.x) >= p.tiles) {
        embed_fill(p, blockIdx.x - p.tiles);
        return;
    }
    __shared__ unsigned count[EmbedSort::MAX_BINS];
    const int bins = 1 << p.bits;
    for (int b = threadIdx.x; b < bins; b += blockDim.x) count[b] = 0;
    __syncthreads();
    const long long i0 = (long long)blockIdx.x * p.subtiles * EmbedSort::SUB;
    const long long i1 = min((long long)p.n, i0 + (long long)p.subtiles * EmbedSort::SUB);
    for (long long i = i0 + threadIdx.x; i < i1; i += blockDim.x)
        atomicAdd(&count[(embed_sort_key(p, int(i)) >> p.shift) & (bins - 1)], 1u);
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += blockDim.x) p.hist[(size_t)blockIdx.x * bins + b] = count[b];
}
// An item's place: items of smaller digits in all tiles, of its digit in earlier
// tiles, in earlier warps of its tile, and earlier in its warp.  A warp holds 32
// * PER consecutive items and ranks 32 at a time with match.any.
__global__ void __launch_bounds__(EmbedSort::THREADS) embed_scatter_kernel(const EmbedSortParams p) {
    using S = EmbedSort;
    pdl_wait();
    pdl_trigger();
    if (int(blockIdx.x) >= p.tiles) {
        embed_fill(p, blockIdx.x - p.tiles);
        return;
    }
    __shared__ unsigned base[S::MAX_BINS];            // next place of each digit for this tile
    __shared__ unsigned count[S::WARPS][S::MAX_BINS];  // per warp: counts, then places
    __shared__ unsigned warp_total[S::WARPS];
    const int bins = 1 << p.bits, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // Each thread owns `own` consecutive digits: totals and earlier tiles' counts.
    const int own = (bins + S::THREADS - 1) / S::THREADS;  // 1..4
    unsigned total[4] = {0, 0, 0, 0}, before[4] = {0, 0, 0, 0}, sum = 0;
    for (int k = 0; k < own; ++k) {
        const int b = tid * own + k;
        if (b < bins) {
#pragma unroll 8
            for (int t = 0; t < p.tiles; ++t) {
                const unsigned c = p.hist[(size_t)t * bins + b];
                total[k] += c;
                if (t < int(blockIdx.x)) before[k] += c;
            }
        }
        sum += total[k];
    }
    unsigned incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
    }
    if (lane == 31) warp_total[warp] = incl;
    __syncthreads();
    unsigned start = incl - sum;
    for (int w = 0; w < warp; ++w) start += warp_total[w];
    for (int k = 0; k < own; ++k) {
        const int b = tid * own + k;
        if (b < bins) base[b] = start + before[k];
        start += total[k];
    }
    for (int s = 0; s < p.subtiles; ++s) {
        const long long i0 = ((long long)blockIdx.x * p.subtiles + s) * S::SUB;
        if (i0 >= p.n) break;
        __syncthreads();
        for (int b = lane; b < bins; b += 32) count[warp][b] = 0;
        __syncwarp();
        unsigned key[S::PER], rank[S::PER];
#pragma unroll
        for (int j = 0; j < S::PER; ++j) {
            const long long i = i0 + warp * (32 * S::PER) + j * 32 + lane;
            key[j] = i < p.n ? embed_sort_key(p, int(i)) : 0xffffffffu;
        }
#pragma unroll
        for (int j = 0; j < S::PER; ++j) {
            const long long i = i0 + warp * (32 * S::PER) + j * 32 + lane;
            const bool live = i < p.n;
            const unsigned digit = (key[j] >> p.shift) & (bins - 1);
            const unsigned peers = __match_any_sync(0xffffffffu, live ? digit : 0x80000000u);
            rank[j] = __popc(peers & ((1u << lane) - 1u));
            unsigned prior = 0;
            if (live) prior = count[warp][digit];
            __syncwarp();
            if (live && rank[j] == 0) count[warp][digit] = prior + __popc(peers);
            __syncwarp();
            rank[j] += prior;
        }
        __syncthreads();
        for (int b = tid; b < bins; b += S::THREADS) {
            unsigned at = base[b];
#pragma unroll
            for (int w = 0; w < S::WARPS; ++w) {
                const unsigned c = count[w][b];
                count[w][b] = at;
                at += c;
            }
            base[b] = at;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < S::PER; ++j) {
            const long long i = i0 + warp * (32 * S::PER) + j * 32 + lane;
            if (i < p.n) {
                const unsigned at = count[warp][(key[j] >> p.shift) & (bins - 1)] + rank[j];
                p.key_out[at] = key[j];
                p.tok_out[at] = p.ids ? int(i) : p.tok_in[i];
            }
        }
    }
}

// ---------------------------------------------------------------- the gradient's sums
// The sorted items are cut into chunks of `chunk` (at most 32).  A warp sums the
// runs of equal ids in one chunk over 32 * V columns, in order, in fp32.  A run
// that lies in the chunk is written; one that began in an earlier chunk goes to
// head[chunk], one that goes on behind it to tail[chunk], and embed_join_kernel
// adds those up.
struct EmbedSumParams {
    void *dtable;
    const void *dout;
    const unsigned *key;
    const int *tok;
    float *head, *tail;  // [chunks][d]
    long long dtable_stride, dout_stride;
    int n, vocab, d, chunk, chunks;
    float scale;
    int accumulate;
};
template <typename TW, int V>
__device__ __forceinline__ void embed_write_row(const EmbedSumParams &p, unsigned id, int c, const float (&acc)[V]) {
    TW *dst = static_cast<TW *>(p.dtable) + (long long)id * p.dtable_stride + c;
    float f[V];
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = acc[i] * p.scale;
    Pack<TW, V> y;
    if (p.accumulate) {
        float old[V];
        y.load(dst);
        y.get(old);
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] += old[i];
    }
    y.set(f);
    y.store(dst);
}
template <typename TG, typename TW, int V>
__global__ void __launch_bounds__(256) embed_sum_kernel(const EmbedSumParams p) {
    constexpr int AHEAD = 8;  // rows in flight per warp
    pdl_wait();
    pdl_trigger();
    const int ch = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int c = (blockIdx.y * 32 + lane) * V;
    if (ch >= p.chunks) return;
    const int i0 = ch * p.chunk, m = min(p.chunk, p.n - i0);
    const unsigned none = unsigned(p.vocab);  // padding's key
    const unsigned mykey = lane < m ? p.key[i0 + lane] : none;
    const int mytok = lane < m ? p.tok[i0 + lane] : 0;
    const unsigned prev = i0 > 0 ? p.key[i0 - 1] : 0xffffffffu;
    const unsigned next = i0 + m < p.n ? p.key[i0 + m] : 0xffffffffu;
    const bool mine = c < p.d;
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.0f;
    bool from_before = __shfl_sync(0xffffffffu, mykey, 0) == prev;
    for (int r0 = 0; r0 < m; r0 += AHEAD) {
        Pack<TG, V> x[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            const unsigned id = __shfl_sync(0xffffffffu, mykey, (r0 + j) & 31);
            const int t = __shfl_sync(0xffffffffu, mytok, (r0 + j) & 31);
            if (mine && r0 + j < m && id != none)
                x[j].load(static_cast<const TG *>(p.dout) + (long long)t * p.dout_stride + c);
            else
                x[j].zero();
        }
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            const int r = r0 + j;
            const unsigned id = __shfl_sync(0xffffffffu, mykey, r & 31);
            const unsigned after = __shfl_sync(0xffffffffu, mykey, (r + 1) & 31);
            if (r >= m || id == none) continue;
            float f[V];
            x[j].get(f);
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] += f[i];
            const bool last = r == m - 1;
            const bool goes_on = last && id == next;
            if (!goes_on && !last && after == id) continue;
            if (mine) {  // the run ends here, or the chunk does
                Pack<float, V> sum;
                sum.set(acc);
                if (from_before) sum.store(p.head + (size_t)ch * p.d + c);
                else if (goes_on) sum.store(p.tail + (size_t)ch * p.d + c);
                else embed_write_row<TW, V>(p, id, c, acc);
            }
            from_before = false;
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] = 0.0f;
        }
    }
}
// Runs over more than one chunk: the CTA of the chunk where one begins adds its
// parts, each warp a contiguous share of the chunks, then the warps' sums in order.
template <typename TW, int V>
__global__ void __launch_bounds__(256) embed_join_kernel(const EmbedSumParams p) {
    __shared__ float part[8][32 * V];
    pdl_wait();
    pdl_trigger();
    const int ch = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int i0 = ch * p.chunk, i1 = i0 + p.chunk;
    if (i1 >= p.n) return;  // nothing goes on behind the last chunk
    const unsigned id = p.key[i1];
    if (id == unsigned(p.vocab) || p.key[i1 - 1] != id) return;
    if (i0 > 0 && p.key[i0] == id && p.key[i0 - 1] == id) return;  // began in an earlier chunk
    // First chunk behind ch whose first item is not of this run.
    int lo = ch + 1, hi = p.chunks;
    while (lo < hi) {
        const int mid = lo + (hi - lo) / 2;
        if (p.key[(long long)mid * p.chunk] == id) lo = mid + 1;
        else hi = mid;
    }
    const int count = lo - (ch + 1), each = (count + 7) / 8;
    const int c = (blockIdx.y * 32 + lane) * V;
    const bool mine = c < p.d;
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.0f;
    if (mine) {
        Pack<float, V> x;
        if (warp == 0) {
            x.load(p.tail + (size_t)ch * p.d + c);
            x.get(acc);
        }
        const int a = ch + 1 + warp * each, b = min(lo, a + each);
#pragma unroll 4
        for (int k = a; k < b; ++k) {
            float f[V];
            x.load(p.head + (size_t)k * p.d + c);
            x.get(f);
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] += f[i];
        }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) part[warp][lane * V + i] = acc[i];
    __syncthreads();
    if (warp == 0 && mine) {
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = 0.0f;
        for (int w = 0; w < 8; ++w) {
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] += part[w][lane * V + i];
        }
        embed_write_row<TW, V>(p, id, c, acc);
    }
}

}  // namespace eg2
