// Embedding lookup with scaling, and its gradient.
//
//   out[t] = scale * table[ids[t]]                       (embed_rows_kernel)
//   dtable[v] (+)= scale * sum over ids[t] = v of dout[t]  (the kernels below it)
//
// An id outside [0, vocab) marks padding: its output row is zero and its
// gradient row is not read.
//
// The gradient sorts the (id, token) pairs by id, stably, and sums each id's rows in
// that order, with no atomics on values: the same n, d and ids give the same bits.
// The sorted list is cut at fixed places, and a run over more than one piece is
// added piece by piece (over many, by eight warps' shares), so how an id's fp32
// additions associate depends on where its run lies, and so on the other ids of
// the batch.  All of it is bound by memory: ids and dout are read once, each
// touched row is written once.
//
// Measured on B200, tables of 262144 x 512: lookup of 61447 bf16 rows 15.9 us
// (85 MB, 5.3 TB/s); gradient of 1999 fp32 rows 83 us (541 MB, the rate of a plain
// copy), of 100003 bf16 rows 93 us (366 MB; the sort before the sums is 35 us of it).
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

// A warp takes a token and walks its columns DEEP * 32 vectors at a time.  What
// keeps memory busy here is many warps with little in each: at 61447 x 512 bf16
// one row a warp takes 15 us, as two do; four rows, each DEEP = 2, took 18.
template <typename TIn, typename TOut, int V>
__global__ void __launch_bounds__(256) embed_rows_kernel(const EmbedRowsParams p) {
    constexpr int DEEP = 2;
    pdl_wait();
    pdl_trigger();
    const int t = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (t >= p.n) return;
    const int id = p.ids[t];
    const bool live = unsigned(id) < unsigned(p.vocab);
    const TIn *src = static_cast<const TIn *>(p.table) + (live ? id * p.table_stride : 0);
    TOut *dst = static_cast<TOut *>(p.out) + t * p.out_stride;
    for (int c0 = lane * V; c0 < p.d; c0 += DEEP * 32 * V) {
        Pack<TIn, V> x[DEEP];
#pragma unroll
        for (int k = 0; k < DEEP; ++k) {
            x[k].zero();
            if (live && c0 + k * 32 * V < p.d) x[k].load(src + c0 + k * 32 * V);
        }
#pragma unroll
        for (int k = 0; k < DEEP; ++k) {
            if (c0 + k * 32 * V >= p.d) break;
            float f[V];
            x[k].get(f);
#pragma unroll
            for (int i = 0; i < V; ++i) f[i] = live ? f[i] * p.scale : 0.0f;
            Pack<TOut, V> y;
            y.set(f);
            y.store(dst + c0 + k * 32 * V);
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
                         MAX_BINS = 1 << MAX_BITS, MAX_TILES = 128,
                         MAX_TOUCHED = 1 << 20;  // rows whose flags the workspace holds
};
// The rows of the table that no token touches are zero.  That is most of the
// gradient's bytes, so CTAs beside each launch's own write a share of them
// meanwhile, a warp a block of 8 rows at a time.  The sort's launches clear the
// touched rows of their share too (from the table's end, where a vocabulary
// sorted by frequency has few); the sums' launch knows them and leaves them out.
struct EmbedFill {
    unsigned char *table;
    const unsigned char *touched;  // null: all rows of the share
    long long stride, block0, blocks;
    int width, rows;               // bytes of a row; rows of the table
    int ctas, each;                // a CTA clears `each` consecutive blocks, a warp one at a time
};
__device__ __forceinline__ void embed_fill(const EmbedFill &f, int cta) {
    const uint4 z = make_uint4(0, 0, 0, 0);
    const int lane = threadIdx.x & 31;
    const bool wide = ((reinterpret_cast<uintptr_t>(f.table) | uintptr_t(f.stride) | unsigned(f.width)) & 15) == 0;
    const long long end = min(f.blocks, (cta + 1ll) * f.each);
    for (long long i = (long long)cta * f.each + (threadIdx.x >> 5); i < end; i += blockDim.x >> 5) {
        const long long row0 = (f.block0 + i) * 8;
        const int rows = int(min(8ll, f.rows - row0));
        const unsigned skip =
            __ballot_sync(0xffffffffu, f.touched && lane < rows && f.touched[row0 + lane]);
        unsigned char *base = f.table + row0 * f.stride;
        if (wide && !skip && f.stride == f.width) {
            const int vecs = int(rows * f.stride / 16);
#pragma unroll 4
            for (int k = lane; k < vecs; k += 32) reinterpret_cast<uint4 *>(base)[k] = z;
            continue;
        }
        for (int r = 0; r < rows; ++r, base += f.stride) {
            if (skip >> r & 1) continue;
            if (wide)
                for (int k = lane * 16; k < f.width; k += 512) *reinterpret_cast<uint4 *>(base + k) = z;
            else
                for (int k = lane * 2; k < f.width; k += 64) *reinterpret_cast<uint16_t *>(base + k) = 0;
        }
    }
}

struct EmbedSortParams {
    const int *ids;             // the first pass reads these, with the token index implied
    const uint2 *in;            // later passes: (key, token)
    uint2 *out;
    unsigned *hist;             // [tiles][bins] of this pass
    int n, vocab, tiles, subtiles, shift, bits;
    unsigned char *touched;     // one flag per table row: set in the last pass (null: not in this one)
    EmbedFill fill;
};
__device__ __forceinline__ unsigned embed_sort_key(const EmbedSortParams &p, int i) {
    if (!p.ids) return p.in[i].x;
    const unsigned id = unsigned(p.ids[i]);
    return id < unsigned(p.vocab) ? id : unsigned(p.vocab);
}
__global__ void __launch_bounds__(EmbedSort::THREADS) embed_hist_kernel(const EmbedSortParams p) {
    pdl_wait();
    if (p.touched)  // before the scatter that marks them
        for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < (p.vocab + 15) / 16; i += gridDim.x * blockDim.x)
            reinterpret_cast<uint4 *>(p.touched)[i] = make_uint4(0, 0, 0, 0);
    if (int(blockIdx.x) >= p.tiles) {
        embed_fill(p.fill, blockIdx.x - p.tiles);
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
// * PER consecutive items and ranks 32 at a time by votes.
__global__ void __launch_bounds__(EmbedSort::THREADS) embed_scatter_kernel(const EmbedSortParams p) {
    using S = EmbedSort;
    pdl_wait();
    if (int(blockIdx.x) >= p.tiles) {
        embed_fill(p.fill, blockIdx.x - p.tiles);
        return;
    }
    __shared__ unsigned base[S::MAX_BINS];            // next place of each digit for this tile
    __shared__ unsigned count[S::WARPS][S::MAX_BINS];  // per warp: counts, then places
    __shared__ unsigned warp_total[S::WARPS];
    const int bins = 1 << p.bits, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // Each thread owns `own` consecutive digits (a power of two): totals and earlier tiles' counts.
    const int own = bins <= S::THREADS ? 1 : bins / S::THREADS;
    unsigned total[4] = {0, 0, 0, 0}, before[4] = {0, 0, 0, 0}, sum = 0;
    if (tid * own < bins) {
        const unsigned *h = p.hist + tid * own;
        auto add = [&](int t, int k, unsigned c) {
            total[k] += c;
            if (t < int(blockIdx.x)) before[k] += c;
        };
        if (own == 1) {
#pragma unroll 16
            for (int t = 0; t < p.tiles; ++t) add(t, 0, h[(size_t)t * bins]);
        } else if (own == 2) {
#pragma unroll 16
            for (int t = 0; t < p.tiles; ++t) {
                const uint2 c = *reinterpret_cast<const uint2 *>(h + (size_t)t * bins);
                add(t, 0, c.x), add(t, 1, c.y);
            }
        } else {
#pragma unroll 8
            for (int t = 0; t < p.tiles; ++t) {
                const uint4 c = *reinterpret_cast<const uint4 *>(h + (size_t)t * bins);
                add(t, 0, c.x), add(t, 1, c.y), add(t, 2, c.z), add(t, 3, c.w);
            }
        }
        sum = (total[0] + total[1]) + (total[2] + total[3]);
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
        int tok[S::PER];
#pragma unroll
        for (int j = 0; j < S::PER; ++j) {
            const long long i = i0 + warp * (32 * S::PER) + j * 32 + lane;
            key[j] = 0xffffffffu, tok[j] = int(i);
            if (i >= p.n) continue;
            if (p.ids) {
                key[j] = embed_sort_key(p, int(i));
            } else {
                const uint2 item = p.in[i];
                key[j] = item.x, tok[j] = int(item.y);
            }
        }
        if (p.touched) {  // the last pass: plain stores of one value, neighbours of one id store once
#pragma unroll
            for (int j = 0; j < S::PER; ++j) {
                const unsigned left = __shfl_up_sync(0xffffffffu, key[j], 1);
                if (key[j] < unsigned(p.vocab) && (lane == 0 || left != key[j])) p.touched[key[j]] = 1;
            }
        }
#pragma unroll
        for (int j = 0; j < S::PER; ++j) {
            const long long i = i0 + warp * (32 * S::PER) + j * 32 + lane;
            const bool live = i < p.n;
            const unsigned digit = (key[j] >> p.shift) & (bins - 1);
            // The live lanes with this lane's digit, one vote per bit.
            unsigned peers = __ballot_sync(0xffffffffu, live);
            for (int bit = 0; bit < p.bits; ++bit) {
                const bool set = digit >> bit & 1;
                const unsigned vote = __ballot_sync(0xffffffffu, set);
                peers &= set ? vote : ~vote;
            }
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
                p.out[at] = make_uint2(key[j], unsigned(tok[j]));
            }
        }
    }
}

// The same sort of up to 4096 items by one CTA in one launch: the items stay in
// registers, up to 4 a thread, and change places through shared memory; the last
// pass writes to memory.  The other CTAs clear the table meanwhile.  (Clusters of 8
// and 16 CTAs that sort up to 131072 items this way, through distributed shared
// memory, took longer than the launches above: 65 and 41 us against 36 at 100003.)
struct EmbedSmall {
    static constexpr int THREADS = 1024, WARPS = 32, MAX_PER = 4, CAP = THREADS * MAX_PER;
    static constexpr int BINS = EmbedSort::MAX_BINS;
    static constexpr int SMEM = CAP * 8 + WARPS * BINS * 2 + BINS * 4 + WARPS * 4;
};
struct EmbedSmallParams {
    const int *ids;
    uint2 *out;
    unsigned char *touched;
    int n, vocab, bits, passes, per;  // per: items of a thread
    EmbedFill fill;
};
__global__ void __launch_bounds__(EmbedSmall::THREADS, 1) embed_sort_kernel(const EmbedSmallParams p) {
    using S = EmbedSmall;
    extern __shared__ __align__(16) uint8_t embed_smem[];
    uint2 *buf = reinterpret_cast<uint2 *>(embed_smem);                               // [CAP] (key, token)
    uint16_t(*count)[S::BINS] = reinterpret_cast<uint16_t(*)[S::BINS]>(buf + S::CAP);  // per warp
    unsigned *base = reinterpret_cast<unsigned *>(count + S::WARPS), *warp_total = base + S::BINS;
    pdl_wait();
    if (blockIdx.x) {
        embed_fill(p.fill, blockIdx.x - 1);
        return;
    }
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, bins = 1 << p.bits;
    const int i0 = warp * 32 * p.per + lane;  // this thread's items: i0 + 32 j
    // Token in the low 13 bits, the item's rank among its warp's equal digits above it.
    unsigned key[S::MAX_PER], tok[S::MAX_PER];
#pragma unroll
    for (int j = 0; j < S::MAX_PER; ++j) {
        const int i = i0 + 32 * j;
        key[j] = 0xffffffffu, tok[j] = 0;
        if (j < p.per && i < p.n) {
            const unsigned id = unsigned(p.ids[i]);
            key[j] = id < unsigned(p.vocab) ? id : unsigned(p.vocab);
            tok[j] = unsigned(i);
        }
    }
    if (p.touched) {
        for (int i = tid; i < (p.vocab + 15) / 16; i += S::THREADS)
            reinterpret_cast<uint4 *>(p.touched)[i] = make_uint4(0, 0, 0, 0);
    }
    for (int pass = 0; pass < p.passes; ++pass) {
        const int shift = pass * p.bits;
        const bool final = pass == p.passes - 1;
        for (int b = lane; b < bins / 2; b += 32) reinterpret_cast<unsigned *>(count[warp])[b] = 0;
        __syncwarp();
#pragma unroll
        for (int j = 0; j < S::MAX_PER; ++j) {
            if (j >= p.per) break;
            const bool live = i0 + 32 * j < p.n;
            const unsigned digit = (key[j] >> shift) & (bins - 1);
            unsigned peers = __ballot_sync(0xffffffffu, live);
            for (int bit = 0; bit < p.bits; ++bit) {
                const bool set = digit >> bit & 1;
                const unsigned vote = __ballot_sync(0xffffffffu, set);
                peers &= set ? vote : ~vote;
            }
            const unsigned place = __popc(peers & ((1u << lane) - 1u));
            unsigned prior = 0;
            if (live) prior = count[warp][digit];
            __syncwarp();
            if (live && place == 0) count[warp][digit] = uint16_t(prior + __popc(peers));
            __syncwarp();
            tok[j] = (tok[j] & 0x1fffu) | (prior + place) << 13;
        }
        __syncthreads();
        // Thread b: digit b's counts become each warp's first place; then the digits' starts.
        unsigned total = 0;
        if (tid < bins) {
            unsigned c[S::WARPS];
#pragma unroll
            for (int w = 0; w < S::WARPS; ++w) c[w] = count[w][tid];
#pragma unroll
            for (int w = 0; w < S::WARPS; ++w) {
                count[w][tid] = uint16_t(total);
                total += c[w];
            }
        }
        unsigned incl = total;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        if (lane == 31) warp_total[warp] = incl;
        __syncthreads();
        const unsigned of_lane = lane < warp ? warp_total[lane] : 0;
        const unsigned start = __reduce_add_sync(0xffffffffu, of_lane) + incl - total;
        if (tid < bins) base[tid] = start;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < S::MAX_PER; ++j) {
            if (j >= p.per) break;
            const bool live = i0 + 32 * j < p.n;
            const unsigned digit = (key[j] >> shift) & (bins - 1), t = tok[j] & 0x1fffu;
            if (final && p.touched) {  // plain stores of one value, neighbours of one id store once
                const unsigned neighbour = __shfl_up_sync(0xffffffffu, key[j], 1);
                if (key[j] < unsigned(p.vocab) && (lane == 0 || neighbour != key[j])) p.touched[key[j]] = 1;
            }
            if (!live) continue;
            const unsigned at = base[digit] + count[warp][digit] + (tok[j] >> 13);
            (final ? p.out : buf)[at] = make_uint2(key[j], t);
        }
        if (final) break;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < S::MAX_PER; ++j) {
            if (j >= p.per) break;
            const int i = i0 + 32 * j;
            if (i < p.n) key[j] = buf[i].x, tok[j] = buf[i].y;
        }
    }
}

// ---------------------------------------------------------------- the gradient's sums
// The sorted items are cut into chunks.  A warp sums the runs of equal ids in one
// chunk over 32 * V columns, in order, in fp32.  A run that lies in the chunk is
// written; one that began in an earlier chunk goes to head[chunk], one that goes
// on behind it to tail[chunk], and embed_join_kernel adds those up.
struct EmbedSumParams {
    void *dtable;
    const void *dout;
    const uint2 *items;  // (key, token), sorted by key, tokens ascending
    float *head, *tail;  // [chunks][d]
    long long dtable_stride, dout_stride;
    int n, vocab, d, chunk, chunks, col_blocks, sum_ctas;
    float scale;
    int accumulate;
    EmbedFill fill;
};
template <typename TW, int V>
__device__ __forceinline__ TW *embed_row(const EmbedSumParams &p, unsigned id, int c) {
    return static_cast<TW *>(p.dtable) + (long long)id * p.dtable_stride + c;
}
// scale * acc, added to what the row held (read before) when accumulating, rounded once.
template <typename TW, int V>
__device__ __forceinline__ void embed_write_row(const EmbedSumParams &p, unsigned id, int c, const float (&acc)[V],
                                                const Pack<TW, V> &held) {
    float f[V], old[V];
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = acc[i] * p.scale;
    if (p.accumulate) {
        held.get(old);
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] += old[i];
    }
    Pack<TW, V> y;
    y.set(f);
    y.store(embed_row<TW, V>(p, id, c));
}
// Rows of whole 16-byte vectors (V of them a lane) come through a ring in shared
// memory, by cp.async, two units of 8 rows ahead of the one being added; each lane
// copies and reads only its own vectors, so there is nothing to synchronise.
// Other rows (V = 1 or 2 elements a lane) are read a unit at a time into registers.
struct EmbedSum {
    static constexpr int THREADS = 128, WARPS = 4, UNIT = 8, STAGES = 3;
    static constexpr int RING = STAGES * UNIT * THREADS * 16;
};
template <typename TG, typename TW, int V>
__global__ void __launch_bounds__(EmbedSum::THREADS) embed_sum_kernel(const __grid_constant__ EmbedSumParams p) {
    using E = EmbedSum;
    constexpr bool STREAM = V * sizeof(TG) == 16;
    extern __shared__ uint4 embed_ring[];
    pdl_wait();
    pdl_trigger();
    // The summing CTAs first, for they run long; the clearing ones are short and
    // take the places that are left.
    if (int(blockIdx.x) >= p.sum_ctas) {
        embed_fill(p.fill, blockIdx.x - p.sum_ctas);
        return;
    }
    const long long w = (long long)blockIdx.x * E::WARPS + (threadIdx.x >> 5);
    const int ch = int(w / p.col_blocks), lane = threadIdx.x & 31;
    const int c = (int(w - (long long)ch * p.col_blocks) * 32 + lane) * V;
    if (ch >= p.chunks) return;
    const int i0 = ch * p.chunk, i1 = min(i0 + p.chunk, p.n), units = (i1 - i0 + E::UNIT - 1) / E::UNIT;
    const unsigned none = unsigned(p.vocab);  // padding's key
    const bool mine = c < p.d;
    // Keys and tokens 32 items at a time, one per lane: this block's and the next one's.
    auto items = [&](int i) -> uint2 { return i + lane < i1 ? p.items[i + lane] : make_uint2(none, 0); };
    uint2 now = items(i0), then = items(i0 + 32);
    const unsigned next = i1 < p.n ? p.items[i1].x : 0xffffffffu;
    bool from_before = i0 > 0 && p.items[i0 - 1].x == __shfl_sync(0xffffffffu, now.x, 0);
    auto row = [&](const uint2 &s, int r, bool *on) {
        const unsigned id = __shfl_sync(0xffffffffu, s.x, r);
        const int t = int(__shfl_sync(0xffffffffu, s.y, r));
        *on = mine && id != none;
        return static_cast<const TG *>(p.dout) + (long long)t * p.dout_stride + c;
    };
    auto slot = [&](int stage, int r) { return embed_ring + (stage * E::UNIT + r) * E::THREADS + threadIdx.x; };
    auto fetch = [&](int stage, const uint2 &s, int r0) {
#pragma unroll
        for (int r = 0; r < E::UNIT; ++r) {
            bool on;
            const TG *src = row(s, r0 + r, &on);
            copy16(slot(stage, r), src, on);
        }
    };
    if constexpr (STREAM) {
        fetch(0, now, 0);
        copies_commit();
        if (units > 1) fetch(1, now, 8);
        copies_commit();
    }
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.0f;
    int stage = 0;  // of the unit being added
    for (int u0 = 0; u0 < units; u0 += 4) {
        const int base = i0 + u0 * E::UNIT;
        const uint2 later = items(base + 64);
        // Items after which a run, or the chunk, ends.
        const unsigned down = __shfl_down_sync(0xffffffffu, now.x, 1);
        const unsigned first_then = __shfl_sync(0xffffffffu, then.x, 0);
        const unsigned after = lane == 31 ? first_then : down;
        const unsigned ends =
            __ballot_sync(0xffffffffu, now.x != none && (base + lane == i1 - 1 || now.x != after));
#pragma unroll 1  // once in the code: the row ends below are long
        for (int j = 0; j < 4; ++j) {
            if (u0 + j >= units) break;
            Pack<TG, V> x[E::UNIT];
            Pack<TW, V> held[E::UNIT];  // accumulating: the rows that end here, asked for together
#pragma unroll
            for (int r = 0; r < E::UNIT; ++r) {
                held[r].zero();
                if (!p.accumulate || !(ends >> (j * 8 + r) & 1)) continue;
                const unsigned id = __shfl_sync(0xffffffffu, now.x, j * 8 + r);
                if (mine) held[r].load(embed_row<TW, V>(p, id, c));
            }
            if constexpr (STREAM) {
                const int to = stage == 0 ? 2 : stage - 1;  // (stage + 2) % 3
                if (u0 + j + 2 < units) fetch(to, j < 2 ? now : then, ((j + 2) & 3) * 8);
                copies_commit();
                copies_wait<2>();
#pragma unroll
                for (int r = 0; r < E::UNIT; ++r) x[r].w[0] = *slot(stage, r);
                stage = stage == 2 ? 0 : stage + 1;
            } else {
#pragma unroll
                for (int r = 0; r < E::UNIT; ++r) {
                    bool on;
                    const TG *src = row(now, j * 8 + r, &on);
                    x[r].zero();
                    if (on) x[r].load(src);
                }
            }
#pragma unroll
            for (int r = 0; r < E::UNIT; ++r) {
                float f[V];
                x[r].get(f);
#pragma unroll
                for (int i = 0; i < V; ++i) acc[i] += f[i];
                if (!(ends >> (j * 8 + r) & 1)) continue;
                const unsigned id = __shfl_sync(0xffffffffu, now.x, j * 8 + r);
                if (mine) {
                    Pack<float, V> sum;
                    sum.set(acc);
                    if (from_before) sum.store(p.head + (size_t)ch * p.d + c);
                    else if (base + j * 8 + r == i1 - 1 && id == next) sum.store(p.tail + (size_t)ch * p.d + c);
                    else embed_write_row<TW, V>(p, id, c, acc, held[r]);
                }
                from_before = false;
#pragma unroll
                for (int i = 0; i < V; ++i) acc[i] = 0.0f;
            }
        }
        now = then, then = later;
    }
    if constexpr (STREAM) copies_wait<0>();
}
// Runs over more than one chunk: tail[first chunk] plus the heads of the chunks
// that follow.  A CTA looks through 32 chunks for those where such a run begins,
// a warp at a time; a run of few parts is added by the warp that found it, in
// order, a long one by the whole CTA: each warp a contiguous share of the parts,
// then the warps' sums in order.
template <typename TW, int V>
__global__ void __launch_bounds__(256) embed_join_kernel(const __grid_constant__ EmbedSumParams p) {
    constexpr int FEW = 16;
    __shared__ float part[8][32 * V];
    __shared__ int long_first[32], long_end[32], longs;
    pdl_wait();
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int c = (blockIdx.y * 32 + lane) * V;
    const bool mine = c < p.d;
    if (threadIdx.x == 0) longs = 0;
    __syncthreads();
    // Lanes 0..3: does a run begin in this chunk and go on behind it?
    const int ch = blockIdx.x * 32 + warp * 4 + lane;
    unsigned id = 0;
    bool begins = false;
    if (lane < 4 && ch < p.chunks - 1) {
        const long long i0 = (long long)ch * p.chunk, i1 = i0 + p.chunk;
        const unsigned first = p.items[i0].x, last = p.items[i1 - 1].x;
        const unsigned prev = i0 > 0 ? p.items[i0 - 1].x : 0xffffffffu;
        id = p.items[i1].x;
        begins = id != unsigned(p.vocab) && last == id && !(first == id && prev == id);
    }
    unsigned found = __ballot_sync(0xffffffffu, begins);
    while (found) {
        const int src = __ffs(found) - 1;
        found &= found - 1;
        const int first = __shfl_sync(0xffffffffu, ch, src);
        const unsigned run = __shfl_sync(0xffffffffu, id, src);
        // stop: the first chunk behind first + 1 whose first item is not of the run, by
        // probing 32 chunks at once, `span` apart: wider while all are, then closer.
        int stop = first + 2;
        for (int span = 1; stop < p.chunks;) {
            const long long k = stop + (long long)(lane + 1) * span - 1;  // the last of this lane's span
            const bool in = k < p.chunks && p.items[k * p.chunk].x == run;
            const int whole = __ffs(~__ballot_sync(0xffffffffu, in)) - 1;  // spans that are all of the run; -1: 32
            stop += (whole < 0 ? 32 : whole) * span;
            if (whole < 0) span *= 32;
            else if (span == 1) break;
            else span /= 32;
        }
        if (stop - first > FEW) {
            if (lane == 0) {
                const int at = atomicAdd(&longs, 1);
                long_first[at] = first, long_end[at] = stop;
            }
        } else if (mine) {
            float acc[V];
            Pack<float, V> x;
            Pack<TW, V> held;
            held.zero();
            if (p.accumulate) held.load(embed_row<TW, V>(p, run, c));
            x.load(p.tail + (size_t)first * p.d + c);
            x.get(acc);
#pragma unroll 4
            for (int k = first + 1; k < stop; ++k) {
                float f[V];
                x.load(p.head + (size_t)k * p.d + c);
                x.get(f);
#pragma unroll
                for (int i = 0; i < V; ++i) acc[i] += f[i];
            }
            embed_write_row<TW, V>(p, run, c, acc, held);
        }
    }
    __syncthreads();
    for (int l = 0; l < longs; ++l) {
        const int first = long_first[l], stop = long_end[l], each = (stop - first - 1 + 7) / 8;
        float acc[V];
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = 0.0f;
        if (mine) {
            Pack<float, V> x;
            if (warp == 0) {
                x.load(p.tail + (size_t)first * p.d + c);
                x.get(acc);
            }
            const int a = first + 1 + warp * each, b = min(stop, a + each);
#pragma unroll 8
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
            const unsigned run = p.items[(long long)(first + 1) * p.chunk].x;
            Pack<TW, V> held;
            held.zero();
            if (p.accumulate) held.load(embed_row<TW, V>(p, run, c));
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] = 0.0f;
            for (int w = 0; w < 8; ++w) {
#pragma unroll
                for (int i = 0; i < V; ++i) acc[i] += part[w][lane * V + i];
            }
            embed_write_row<TW, V>(p, run, c, acc, held);
        }
        __syncthreads();
    }
}

}  // namespace eg2
