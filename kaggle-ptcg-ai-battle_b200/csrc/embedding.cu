// Embedding lookup with scaling, and its gradient by sorted ids.
//   forward    out[i, :] = scale * table[id_i, :]      (0 where id_i is the padding id)
//   gradient   dtable[v, :] (+)= scale * sum over the i with id_i = v of dout[i, :]
// The reference's embedding gradients are atomic adds from every token
// (k_tok_cat_bwd, native/model/ptcg_model2.cu:36-64).  Here the places are
// sorted by id first, so each table row is summed in an order that follows
// from the ids alone (not from scheduling) and written once, and an id that
// half of the batch holds costs no contention.  Sums are fp32; the only
// rounding to fewer bits is the forward's to its output type.
#include <algorithm>

#include "vec.cuh"

namespace {

// columns: what a launch's 65535 slices of 32 single ones cover
constexpr int MAX_WIDTH = 65535 * 32;

// -------------------------------------------------------------- forward
// Bound: HBM for ids and output, L2 for the table's rows after their first
// touch.  2 M rows of 128 from an fp32 table of 4096 to bf16: 117 us, 4.6 TB/s
// of output and 9.2 TB/s of table rows from L1 and L2; 32768 rows of 1024, bf16
// to bf16, 25 us (5.4 TB/s).  LX lanes take a row's V-element pieces, 256 / LX rows to a
// block pass, four rows (eight of single elements) in flight per thread and the
// next rows' ids ahead of them.
template <typename TT, typename TO, int V>
__global__ void __launch_bounds__(256, V == 4 ? 5 : 4) k_embed_fwd(
        TO* __restrict__ out, long ldo, const TT* __restrict__ table, long ldt,
        const int* __restrict__ ids, long n, int vocab, int pieces, int lx_log2, float scale,
        int pad_id, int has_pad) {
    const int tx = threadIdx.x & ((1 << lx_log2) - 1), ty = threadIdx.x >> lx_log2;
    const int ry = 256 >> lx_log2;
    constexpr int U = V == 1 ? 8 : 4;                      // rows in flight a thread
    const long step = (long)gridDim.x * ry * U;
    int next[U];
    auto fetch = [&](long r0) {
        #pragma unroll
        for (int u = 0; u < U; u++) {
            const long r = r0 + u * ry + ty;
            next[u] = r < n ? ids[r] : 0;
        }
    };
    fetch((long)blockIdx.x * ry * U);
    for (long r0 = (long)blockIdx.x * ry * U; r0 < n; r0 += step) {
        int id[U];
        #pragma unroll
        for (int u = 0; u < U; u++) id[u] = next[u];
        fetch(r0 + step);
        for (int c = tx; c < pieces; c += 1 << lx_log2) {
            float v[U][V];
            #pragma unroll
            for (int u = 0; u < U; u++) {
                const int row = min(max(id[u], 0), vocab - 1);
                VecIO<TT, V>::ld(v[u], table + (long)row * ldt + (long)c * V);
            }
            #pragma unroll
            for (int u = 0; u < U; u++) {
                const long r = r0 + u * ry + ty;
                if (r >= n) break;
                const bool pad = has_pad && id[u] == pad_id;
                #pragma unroll
                for (int e = 0; e < V; e++) v[u][e] = pad ? 0.f : v[u][e] * scale;
                VecIO<TO, V>::st(out + r * ldo + (long)c * V, v[u]);
            }
        }
    }
}

// ----------------------------------------------------------------- sort
// Stable least-digit-first radix sort of (id, place), up to 9 bits a pass, two
// launches a pass: the digit counts of each tile, then a scatter whose blocks
// derive their own bases from all tiles' counts (a block reads tiles x bins
// counters from L2, which is cheaper here than a third launch for the scan).
// Lanes with equal digits find each other by one ballot per digit bit; the
// match instruction took 166 us where this takes 20 (first count of 2 M places).
// Bound: latency; 16 bytes per place and pass (2 M places of 4096 ids, two
// passes: 67 us, 1 TB/s; 32768 places of 65537 ids 25 us).  The counters that a
// block reads grow with the tiles: from some 100 M places on they, not the
// places, would set the time.
constexpr int SORT_T = 1024, MAX_BITS = 9, MAX_BINS = 1 << MAX_BITS;

// the sort key of a place: its clamped id, or `vocab` for a padding place,
// which sorts behind every row
PTCG_DEV uint32_t key_of(int id, int vocab, int pad_id, int has_pad) {
    if (has_pad && id == pad_id) return (uint32_t)vocab;
    return (uint32_t)min(max(id, 0), vocab - 1);
}
// the lanes with the same digit among those with `in`
PTCG_DEV uint32_t same_digit(uint32_t d, bool in, int bits) {
    uint32_t m = __ballot_sync(0xffffffffu, in);
    for (int b = 0; b < bits; b++) {
        const bool one = (d >> b) & 1;
        const uint32_t v = __ballot_sync(0xffffffffu, one);
        m &= one ? v : ~v;
    }
    return m;
}

struct SortArgs {
    uint32_t *counts, *keys_out, *pos_out;
    const uint32_t *keys, *pos;
    const int* ids;
    long n;
    int shift, bits, vocab, pad_id, has_pad;
};

template <int ITEMS, bool FIRST>
__global__ void __launch_bounds__(SORT_T) k_sort_count(const __grid_constant__ SortArgs a) {
    __shared__ uint32_t hist[MAX_BINS];
    const int bins = 1 << a.bits, lane = threadIdx.x & 31;
    for (int i = threadIdx.x; i < bins; i += SORT_T) hist[i] = 0;
    __syncthreads();
    const long base = (long)blockIdx.x * SORT_T * ITEMS;
    uint32_t key[ITEMS];
    #pragma unroll
    for (int k = 0; k < ITEMS; k++) {
        const long i = base + k * SORT_T + threadIdx.x;
        key[k] = 0;
        if (i < a.n) key[k] = FIRST ? key_of(a.ids[i], a.vocab, a.pad_id, a.has_pad) : a.keys[i];
    }
    #pragma unroll
    for (int k = 0; k < ITEMS; k++) {
        const bool in = base + k * SORT_T + threadIdx.x < a.n;
        const uint32_t d = (key[k] >> a.shift) & (bins - 1);
        const uint32_t same = same_digit(d, in, a.bits);
        if (in && lane == __ffs(same) - 1) atomicAdd(&hist[d], __popc(same));
    }
    __syncthreads();
    for (int i = threadIdx.x; i < bins; i += SORT_T) a.counts[(long)blockIdx.x * bins + i] = hist[i];
}

// Shared memory of a tile's sort: per warp and digit the count, then the first
// place among the tile's places of that digit; the digits' first places.
struct TileSort {
    uint16_t wcnt[SORT_T / 32][MAX_BINS];
    uint32_t start[MAX_BINS], wsum[MAX_BINS / 32];
};
// Where each of this thread's ITEMS places goes in its tile sorted by the digit
// (stable: a warp holds 32 * ITEMS consecutive places, lane by lane).  t.start
// holds the digits' first places.  It is read, as t.wcnt is, after the last
// barrier in here: a caller synchronises before it writes t or calls again.
template <int ITEMS>
PTCG_DEV void tile_places(TileSort& t, uint32_t (&to)[ITEMS], const uint32_t (&key)[ITEMS], int n, int shift, int bits) {
    constexpr int NW = SORT_T / 32;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, bins = 1 << bits;
    const int base = warp * 32 * ITEMS;
    for (int i = tid; i < NW * MAX_BINS / 2; i += SORT_T) ((uint32_t*)t.wcnt)[i] = 0;
    __syncthreads();
    #pragma unroll
    for (int k = 0; k < ITEMS; k++) {
        const bool in = base + k * 32 + lane < n;
        const uint32_t d = (key[k] >> shift) & (bins - 1);
        const uint32_t same = same_digit(d, in, bits);
        uint32_t before = 0;
        if (in) before = t.wcnt[warp][d];
        __syncwarp();
        to[k] = before + __popc(same & ((1u << lane) - 1u));
        if (in && lane == __ffs(same) - 1) t.wcnt[warp][d] = (uint16_t)(before + __popc(same));
        __syncwarp();
    }
    __syncthreads();
    uint32_t all = 0, x = 0;
    if (tid < MAX_BINS) {
        if (tid < bins) {
            #pragma unroll 8
            for (int w = 0; w < NW; w++) {
                const uint32_t v = t.wcnt[w][tid];
                t.wcnt[w][tid] = (uint16_t)all;            // below the tile's 16384 places
                all += v;
            }
        }
        x = all;
        #pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31) t.wsum[warp] = x;
    }
    __syncthreads();
    if (tid < bins) {
        uint32_t s = x - all;
        for (int w = 0; w < warp; w++) s += t.wsum[w];
        t.start[tid] = s;
    }
    __syncthreads();
    #pragma unroll
    for (int k = 0; k < ITEMS; k++) {
        const uint32_t d = (key[k] >> shift) & (bins - 1);
        to[k] += t.start[d] + t.wcnt[warp][d];
    }
}

// A tile's places, brought into digit order in shared memory, so that they
// leave as runs of neighbours (scattered 4-byte writes took twice as long)
template <int ITEMS, bool FIRST>
__global__ void __launch_bounds__(SORT_T) k_sort_scatter(const __grid_constant__ SortArgs a) {
    constexpr int TILE = SORT_T * ITEMS;
    extern __shared__ uint32_t sorted[];                   // [TILE] keys, [TILE] places
    __shared__ TileSort t;
    __shared__ uint32_t tot[SORT_T], pre[SORT_T], base[MAX_BINS], wsum[MAX_BINS / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int bins = 1 << a.bits, tiles = gridDim.x, tile = blockIdx.x;
    const long first = (long)tile * TILE;
    const int n = (int)min((long)TILE, a.n - first);
    uint32_t key[ITEMS], ps[ITEMS], to[ITEMS];
    #pragma unroll
    for (int k = 0; k < ITEMS; k++) {
        const int i = warp * 32 * ITEMS + k * 32 + lane;
        key[k] = 0;
        ps[k] = (uint32_t)(first + i);
        if (i < n) {
            if (FIRST) {
                key[k] = key_of(a.ids[first + i], a.vocab, a.pad_id, a.has_pad);
            } else {
                key[k] = a.keys[first + i];
                ps[k] = a.pos[first + i];
            }
        }
    }
    {   // counts of each digit over all tiles, and over the tiles before this one
        const int d = tid & (bins - 1), part = tid >> a.bits, parts = SORT_T >> a.bits;
        uint32_t x = 0, p = 0;
        #pragma unroll 4
        for (int j = part; j < tiles; j += parts) {
            const uint32_t c = a.counts[(long)j * bins + d];
            x += c;
            p += j < tile ? c : 0u;
        }
        tot[tid] = x;
        pre[tid] = p;
    }
    tile_places<ITEMS>(t, to, key, n, a.shift, a.bits);
    #pragma unroll
    for (int k = 0; k < ITEMS; k++) {
        if (warp * 32 * ITEMS + k * 32 + lane < n) {
            sorted[to[k]] = key[k];
            sorted[TILE + to[k]] = ps[k];
        }
    }
    // the digits' first places for this tile, less their first places in it
    uint32_t all = 0, mine = 0, x = 0;
    if (tid < MAX_BINS) {
        if (tid < bins)
            for (int j = tid; j < SORT_T; j += bins) { all += tot[j]; mine += pre[j]; }
        x = all;
        #pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31) wsum[warp] = x;
    }
    __syncthreads();
    if (tid < bins) {
        mine += x - all;
        for (int w = 0; w < warp; w++) mine += wsum[w];
        base[tid] = mine - t.start[tid];
    }
    __syncthreads();
    for (int i = tid; i < n; i += SORT_T) {
        const uint32_t k = sorted[i], at = base[(k >> a.shift) & (bins - 1)] + i;
        a.keys_out[at] = k;
        a.pos_out[at] = sorted[TILE + i];
    }
}

// All passes of a batch that one block holds, in one launch: for small batches
// the launches would cost more than the sort (8000 places of 4096 ids 16 us,
// 20000 in five launches 22; with one place a thread, up to 1024, 5 us
// where eight a thread took 14)
constexpr int SMALL_N = SORT_T * 8;
template <int ITEMS>
__global__ void __launch_bounds__(SORT_T) k_sort_small(const __grid_constant__ SortArgs a, int passes) {
    extern __shared__ uint32_t sorted[];                   // [SORT_T * ITEMS] keys, as many places
    __shared__ TileSort t;
    const int n = (int)a.n, base = (threadIdx.x >> 5) * 32 * ITEMS + (threadIdx.x & 31);
    uint32_t key[ITEMS], ps[ITEMS], to[ITEMS];
    #pragma unroll
    for (int k = 0; k < ITEMS; k++) {
        const int i = base + k * 32;
        key[k] = i < n ? key_of(a.ids[i], a.vocab, a.pad_id, a.has_pad) : 0u;
        ps[k] = (uint32_t)i;
    }
    for (int p = 0; p < passes; p++) {
        tile_places<ITEMS>(t, to, key, n, p * a.bits, a.bits);
        #pragma unroll
        for (int k = 0; k < ITEMS; k++) {
            if (base + k * 32 < n) {
                sorted[to[k]] = key[k];
                sorted[SORT_T * ITEMS + to[k]] = ps[k];
            }
        }
        __syncthreads();
        #pragma unroll
        for (int k = 0; k < ITEMS; k++) {
            const int i = base + k * 32;
            if (i < n) {
                key[k] = sorted[i];
                ps[k] = sorted[SORT_T * ITEMS + i];
            }
        }
        __syncthreads();
    }
    #pragma unroll
    for (int k = 0; k < ITEMS; k++) {
        const int i = base + k * 32;
        if (i < n) {
            a.keys_out[i] = key[k];
            a.pos_out[i] = ps[k];
        }
    }
}

// ------------------------------------------------------------------ sums
// Segmented sum over the sorted places.  A block owns `chunk` consecutive
// sorted places and a slice of G * V columns; each of its 256 / G lane groups
// walks a run of them with the row sum in registers.  A segment (the places
// of one id) inside one run is written straight to its table row.  A run
// whose first segment began earlier, or whose last goes on, leaves that sum
// as a partial: the block joins its groups' partials in order through shared
// memory, and k_embed_join joins the blocks'.  Rows without a place are
// zeroed by extra blocks.  Bound: HBM, dout read once as gathered rows: 2 M
// bf16 rows of 128 into 4096 111 us (4.8 TB/s; 120 with three blocks a
// processor, which their registers would leave), as many fp32 rows 166 us (6.5
// TB/s), 32768 bf16 rows of 1024 into 65537 61 us (5.5 TB/s with the table's
// zeros).
constexpr int MAX_CHUNK = 2048;
enum { SEG_HEAD = 1, SEG_THROUGH = 2, SEG_TAIL = 4 };

struct SumArgs {
    const void* dout; long lddo;
    const uint32_t* keys; const uint32_t* pos;
    long n;
    float* dtab; long lddt;
    float* head; float* tail;        // [chunks][width] partials of each block
    uint32_t* flags; uint32_t* tail_id;
    int vocab, width, pieces, accumulate;
    int chunk, run, nchunks, zero_blocks;
    float scale;
};

template <int V>
PTCG_DEV void put_row(const SumArgs& a, uint32_t id, int piece, const float (&s)[V]) {
    float* p = a.dtab + (long)id * a.lddt + (long)piece * V;
    float v[V];
    #pragma unroll
    for (int e = 0; e < V; e++) v[e] = s[e] * a.scale;
    if (a.accumulate) {
        float o[V];
        VecIO<float, V>::ld(o, p);
        #pragma unroll
        for (int e = 0; e < V; e++) v[e] += o[e];
    }
    VecIO<float, V>::st(p, v);
}

template <typename T, int V, int G>
__global__ void __launch_bounds__(256, 4) k_embed_sum(const __grid_constant__ SumArgs a) {
    constexpr int NG = 256 / G, S = G * V, U = 8;
    __shared__ float s_head[NG][S], s_tail[NG][S];
    __shared__ uint32_t s_key[MAX_CHUNK + 2], s_pos[MAX_CHUNK];
    __shared__ uint32_t s_flag[NG], s_hid[NG], s_tid[NG];
    const int lane = threadIdx.x % G, grp = threadIdx.x / G;
    const int piece = blockIdx.y * G + lane;
    const bool col = piece < a.pieces;
    if (blockIdx.x >= (unsigned)a.nchunks) {               // rows nothing refers to
        // 256 rows at a time, a search in the sorted ids for each
        const float z[V] = {};
        for (long b = blockIdx.x - a.nchunks; b * 256 < a.vocab; b += a.zero_blocks) {
            const long row = b * 256 + threadIdx.x;
            long lo = 0, hi = a.n;                         // first place with a key >= row
            while (lo < hi) {
                const long mid = (lo + hi) >> 1;
                if (a.keys[mid] < (uint32_t)row) lo = mid + 1; else hi = mid;
            }
            __syncthreads();
            s_key[threadIdx.x] = row < a.vocab && !(lo < a.n && a.keys[lo] == (uint32_t)row);
            __syncthreads();
            for (int i = grp; i < 256; i += NG)
                if (col && s_key[i])
                    VecIO<float, V>::st(a.dtab + (b * 256 + i) * a.lddt + (long)piece * V, z);
        }
        return;
    }
    const uint32_t none = 0xffffffffu, vocab = (uint32_t)a.vocab;
    const long c0 = (long)blockIdx.x * a.chunk;
    const int len = (int)min((long)a.chunk, a.n - c0);
    // the chunk's keys with one neighbour on either side, and its places
    for (int i = threadIdx.x; i < len + 2; i += 256) {
        const long at = c0 - 1 + i;
        s_key[i] = at >= 0 && at < a.n ? a.keys[at] : none;
        if (i < len) s_pos[i] = a.pos[c0 + i];
    }
    __syncthreads();
    const uint32_t* key = s_key + 1;
    const T* dout = (const T*)a.dout + (long)piece * V;
    const int r0 = min(len, grp * a.run), r1 = min(len, r0 + a.run);
    uint32_t flag = 0, hid = none, tid = none;
    float acc[V];
    #pragma unroll
    for (int e = 0; e < V; e++) acc[e] = 0.f;
    if (r0 < r1) {
        uint32_t cur = key[r0];
        bool began = key[r0 - 1] == cur;                   // the open segment's start is earlier
        const uint32_t after = key[r1];
        for (int i = r0; i < r1; i += U) {
            Raw<T, V> raw[U];
            #pragma unroll
            for (int u = 0; u < U; u++) {
                // padding places (key vocab) carry no gradient: not read
                const bool take = i + u < r1 && key[min(i + u, r1 - 1)] < vocab && col;
                if (take) raw[u].ld(dout + (long)s_pos[i + u] * a.lddo);
                else raw[u].zero();
            }
            #pragma unroll
            for (int u = 0; u < U; u++) {
                if (i + u >= r1) break;
                const uint32_t k = key[i + u];
                if (k != cur) {
                    if (began) {
                        flag |= SEG_HEAD;
                        hid = cur;
                        #pragma unroll
                        for (int e = 0; e < V; e++) s_head[grp][lane * V + e] = acc[e];
                    } else if (cur < vocab && col) {
                        put_row<V>(a, cur, piece, acc);
                    }
                    began = false;
                    cur = k;
                    #pragma unroll
                    for (int e = 0; e < V; e++) acc[e] = 0.f;
                }
                float v[V];
                raw[u].get(v);
                #pragma unroll
                for (int e = 0; e < V; e++) acc[e] += v[e];
            }
        }
        const bool on = after == cur;
        if (began) {
            flag |= SEG_HEAD | (on ? SEG_THROUGH : 0);
            hid = cur;
            #pragma unroll
            for (int e = 0; e < V; e++) s_head[grp][lane * V + e] = acc[e];
        } else if (on) {
            flag |= SEG_TAIL;
            tid = cur;
            #pragma unroll
            for (int e = 0; e < V; e++) s_tail[grp][lane * V + e] = acc[e];
        } else if (cur < vocab && col) {
            put_row<V>(a, cur, piece, acc);
        }
    }
    if (lane == 0) { s_flag[grp] = flag; s_hid[grp] = hid; s_tid[grp] = tid; }
    __syncthreads();
    if (threadIdx.x >= G) return;
    // one group's lanes join the runs in order; `open`: a sum is being carried,
    // `early`: it began before this block
    uint32_t out = 0, out_id = none;
    bool open = false, early = false;
    uint32_t id = none;
    #pragma unroll
    for (int e = 0; e < V; e++) acc[e] = 0.f;
    for (int g = 0; g < NG; g++) {
        const uint32_t f = s_flag[g];
        if (f & SEG_HEAD) {
            if (!open) { open = true; early = true; id = s_hid[g]; }
            #pragma unroll
            for (int e = 0; e < V; e++) acc[e] += s_head[g][lane * V + e];
            if (!(f & SEG_THROUGH)) {
                if (early) {
                    out |= SEG_HEAD;
                    if (col) VecIO<float, V>::st(a.head + (long)blockIdx.x * a.width + (long)piece * V, acc);
                } else if (id < vocab && col) {
                    put_row<V>(a, id, piece, acc);
                }
                open = false;
            }
        }
        if (f & SEG_TAIL) {
            open = true;
            early = false;
            id = s_tid[g];
            #pragma unroll
            for (int e = 0; e < V; e++) acc[e] = s_tail[g][lane * V + e];
        }
        if (!open) {
            #pragma unroll
            for (int e = 0; e < V; e++) acc[e] = 0.f;
        }
    }
    if (open) {
        out |= early ? SEG_HEAD | SEG_THROUGH : SEG_TAIL;
        if (!early) out_id = id;
        float* p = (early ? a.head : a.tail) + (long)blockIdx.x * a.width + (long)piece * V;
        if (col) VecIO<float, V>::st(p, acc);
    }
    // every slice's block computes the same flags from the keys alone
    if (threadIdx.x == 0 && blockIdx.y == 0) {
        a.flags[blockIdx.x] = out;
        a.tail_id[blockIdx.x] = out_id;
    }
}

// Joins the segments that cross blocks: the block of chunk c whose tail goes
// on adds the heads of the chunks after it, up to and including the first
// that the segment does not pass through: a thread a column, or, for an id that
// many chunks hold, 8 threads over the partials of each, combined in order
// (7.5 us behind the 2 M places above, where a few ids hold most chunks; 3.6
// behind the 32768, 8.7 with 8 threads a column there as well).
__global__ void __launch_bounds__(256) k_embed_join(const __grid_constant__ SumArgs a) {
    const int c = blockIdx.x;
    if (!(a.flags[c] & SEG_TAIL)) return;
    const uint32_t id = a.tail_id[c];
    if (id >= (uint32_t)a.vocab) return;                    // the padding id's places
    __shared__ float part[8][32];
    __shared__ int s_end;
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    // chunks c + 1 .. end hold the rest
    if (threadIdx.x == 0) s_end = a.nchunks - 1;
    for (int j0 = c + 1; j0 < a.nchunks; j0 += 256) {
        __syncthreads();
        const int j = j0 + threadIdx.x;
        const bool stop = j < a.nchunks && !(a.flags[j] & SEG_THROUGH);
        if (stop) atomicMin(&s_end, j);
        if (__syncthreads_or(stop)) break;
    }
    __syncthreads();
    const int end = s_end, len = end - c;                   // partial rows: tail + len heads
    if (len <= 16) {                                        // a thread a column
        for (int x = blockIdx.y * 256 + threadIdx.x; x < a.width; x += gridDim.y * 256) {
            float s = a.tail[(long)c * a.width + x];
            #pragma unroll 4
            for (int j = 0; j < len; j++) s += a.head[(long)(c + 1 + j) * a.width + x];
            const float v[1] = {s};
            put_row<1>(a, id, x, v);
        }
        return;
    }
    const int per = (len + 7) / 8;
    for (int col = blockIdx.y * 32; col < a.width; col += gridDim.y * 32) {
        const int x = col + tx;
        float s = 0.f;
        if (x < a.width) {
            if (ty == 0) s = a.tail[(long)c * a.width + x];
            const int j1 = min(len, (ty + 1) * per);
            #pragma unroll 4
            for (int j = ty * per; j < j1; j++) s += a.head[(long)(c + 1 + j) * a.width + x];
        }
        part[ty][tx] = s;
        __syncthreads();
        if (ty == 0 && x < a.width) {
            #pragma unroll
            for (int k = 1; k < 8; k++) s += part[k][tx];
            const float v[1] = {s};
            put_row<1>(a, id, x, v);
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------ host side
struct Plan {
    int items, tiles, passes, bits;  // sort: bits of a digit
    int chunk, nchunks;              // sums (run and slices follow from the variant)
    long o_keys[2], o_pos[2], o_counts, o_head, o_tail, o_flags, o_tid, bytes;
};

long up256(long x) { return (x + 255) / 256 * 256; }

// Everything follows from n, vocab and width, so that the size can be asked
// for before the call; the alignment-dependent choices do not change it.
Plan plan(long n, int vocab, int width) {
    Plan p;
    int bits = 1;
    while (bits < 31 && (1L << bits) <= vocab) bits++;      // keys 0 .. vocab
    p.passes = (bits + MAX_BITS - 1) / MAX_BITS;
    p.bits = (bits + p.passes - 1) / p.passes;
    // 4 places a thread give four times the blocks of 16, but sixteen times the
    // counters that all blocks read, tiles^2 x bins: they are taken for one
    // block a processor, or two where the digits have at most 7 bits.  Whole
    // gradients of width 16 by 4 / 16 places, us: 4096 ids (7-bit digits) 600000
    // places 70 / 107, 1.2 M 108 / 123, 1.6 M 145 / 129, 4 M 387 / 277; 65537 ids (9-bit
    // digits) 600000 87 / 123, 620000 119 / 125, 1.2 M 156 / 139, 4 M 781 / 330
    p.items = n > 148L * SORT_T * 4 * (p.bits <= 7 ? 2 : 1) ? 16 : 4;
    p.tiles = (int)cdiv(n, (long)SORT_T * p.items);
    // about eight blocks a processor over all column slices, at least 8
    // places a lane group
    const int slices = (int)cdiv(width, 256);
    long want = (n * slices + 148 * 8 - 1) / (148 * 8);
    p.chunk = (int)(std::min(std::max(want, 64L), (long)MAX_CHUNK) + 31) / 32 * 32;
    p.nchunks = (int)cdiv(n, p.chunk);
    long o = 0;
    for (int i = 0; i < 2; i++) {
        p.o_keys[i] = o; o = up256(o + 4 * n);
        p.o_pos[i] = o; o = up256(o + 4 * n);
    }
    p.o_counts = o; o = up256(o + (4L << p.bits) * p.tiles);
    p.o_head = o; o = up256(o + 4L * width * p.nchunks);
    p.o_tail = o; o = up256(o + 4L * width * p.nchunks);
    p.o_flags = o; o = up256(o + 4L * p.nchunks);
    p.o_tid = o; o = up256(o + 4L * p.nchunks);
    p.bytes = o;
    return p;
}

template <typename TT, typename TO>
void embed_fwd(void* out, long ldo, const void* table, long ldt, const int* ids, long n,
               int vocab, int width, float scale, int pad_id, int V, cudaStream_t s) {
    const int pieces = width / V;
    // the lanes of a row that leave the fewest idle in its last step (100000 bf16
    // rows of 301: 40 us with 64 lanes and 8 rows in flight, 53 with 256 and 4)
    int lx = 0;
    while (lx < 8 && (1 << lx) < pieces) lx++;
    if (lx == 8)
        for (int l = 7; l >= 5; l--)
            if (cdiv(pieces, 1L << l) << l < cdiv(pieces, 1L << lx) << lx) lx = l;
    const long rows = (256 >> lx) * (V == 1 ? 8L : 4L);
    const long blocks = (n + rows - 1) / rows;
    const unsigned grid = (unsigned)(blocks < 148L * 32 ? blocks : 148L * 32);
    ++g_ptcg_launches;
    #define EF(V) k_embed_fwd<TT, TO, V><<<grid, 256, 0, s>>>((TO*)out, ldo, (const TT*)table, ldt, \
        ids, n, vocab, pieces, lx, scale, pad_id, pad_id >= 0)
    if constexpr (sizeof(TO) == 2)
        if (V == 8) { EF(8); return; }
    if (V == 4) EF(4); else EF(1);
    #undef EF
}

template <int ITEMS, bool FIRST>
cudaError_t sort_pass(const SortArgs& a, int tiles, cudaStream_t s) {
    constexpr int bytes = 8 * SORT_T * ITEMS;
    const cudaError_t e = cudaFuncSetAttribute(k_sort_scatter<ITEMS, FIRST>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return e;
    g_ptcg_launches += 2;
    k_sort_count<ITEMS, FIRST><<<tiles, SORT_T, 0, s>>>(a);
    k_sort_scatter<ITEMS, FIRST><<<tiles, SORT_T, bytes, s>>>(a);
    return cudaSuccess;
}
template <int ITEMS>
cudaError_t sort_small(const SortArgs& a, int passes, cudaStream_t s) {
    constexpr int bytes = 8 * SORT_T * ITEMS;
    const cudaError_t e = cudaFuncSetAttribute(k_sort_small<ITEMS>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return e;
    ++g_ptcg_launches, k_sort_small<ITEMS><<<1, SORT_T, bytes, s>>>(a, passes);
    return cudaSuccess;
}

template <typename T, int V, int G>
void embed_sum(SumArgs a, cudaStream_t s) {
    a.pieces = a.width / V;
    a.run = (int)cdiv(a.chunk, 256 / G);
    a.zero_blocks = a.accumulate ? 0 : (int)std::min<long>(148 * 4, cdiv(a.vocab, 256));
    const dim3 grid(a.nchunks + a.zero_blocks, cdiv(a.pieces, G));
    ++g_ptcg_launches, k_embed_sum<T, V, G><<<grid, 256, 0, s>>>(a);
}
template <typename T>
void embed_sum(const SumArgs& a, int V, cudaStream_t s) {
    // a lane group as wide as the row needs: 8, 16 or 32 lanes
    constexpr int VV = sizeof(T) == 2 ? 8 : 4;
    const int lanes = a.width / V;
    if (V == VV) {
        if (lanes <= 8) embed_sum<T, VV, 8>(a, s);
        else if (lanes <= 16) embed_sum<T, VV, 16>(a, s);
        else embed_sum<T, VV, 32>(a, s);
    } else {
        embed_sum<T, 1, 32>(a, s);
    }
}

}  // namespace

extern "C" {

int ptcg_embedding_fwd(const void* table, int table_dtype, long ldt, int vocab, int width,
                       const int* ids, long n, float scale, int pad_id, void* out, int out_dtype,
                       long ldo, void* stream) {
    OP_REQ(dt_ok(table_dtype) && dt_ok(out_dtype), PTCG_EINVAL, "embedding: unknown dtype");
    OP_REQ(vocab > 0 && width > 0 && n >= 0 && ldt >= width && ldo >= width, PTCG_EINVAL,
           "embedding: bad sizes (vocab %d, width %d, n %ld, ldt %ld, ldo %ld)", vocab, width, n,
           ldt, ldo);
    if (n == 0) return PTCG_OK;
    OP_REQ(table && ids && out, PTCG_EINVAL, "embedding: null pointer");
    OP_REQ(el_ok(table, table_dtype) && el_ok(out, out_dtype) && (uintptr_t)ids % 4 == 0,
           PTCG_EINVAL, "embedding: pointer not aligned to its element");
    cudaStream_t s = (cudaStream_t)stream;
    // pieces of 8 elements for bf16 outputs, else of 4 (2 M rows of 128: fp32 to
    // bf16 117 us in eights, 136 in fours, but bf16 to fp32, where an eight is two
    // stores of half sectors, 267 and 179; 100000 bf16 rows of 300: 27 us in
    // fours, 40 in ones)
    auto fits = [&](int v) { return width % v == 0 && vec_ok(table, table_dtype, ldt, v) && vec_ok(out, out_dtype, ldo, v); };
    const int V = out_dtype == PTCG_BF16 && fits(8) ? 8 : fits(4) ? 4 : 1;
    #define EF(TT, TO) embed_fwd<TT, TO>(out, ldo, table, ldt, ids, n, vocab, width, scale, pad_id, V, s)
    if (table_dtype == PTCG_BF16) { if (out_dtype == PTCG_BF16) EF(bf16, bf16); else EF(bf16, float); }
    else { if (out_dtype == PTCG_BF16) EF(float, bf16); else EF(float, float); }
    #undef EF
    OP_CKL();
    return PTCG_OK;
}

long ptcg_embedding_bwd_scratch(long n, int vocab, int width) {
    OP_REQ(n >= 0 && n <= 0x7fffffffL && vocab > 0 && width > 0 && width <= MAX_WIDTH, -1,
           "embedding gradient: bad sizes (n %ld, vocab %d, width %d)", n, vocab, width);
    return n == 0 ? 0 : plan(n, vocab, width).bytes;
}

int ptcg_embedding_bwd(const void* dout, int dout_dtype, long lddo, const int* ids, long n,
                       float scale, int pad_id, float* dtable, long lddt, int vocab, int width,
                       int accumulate, void* scratch, long scratch_bytes, void* stream) {
    OP_REQ(dt_ok(dout_dtype), PTCG_EINVAL, "embedding gradient: unknown dtype");
    OP_REQ(vocab > 0 && width > 0 && width <= MAX_WIDTH && n >= 0 && lddo >= width && lddt >= width && dtable,
           PTCG_EINVAL, "embedding gradient: bad arguments (vocab %d, width %d, n %ld, lddo %ld, lddt %ld)",
           vocab, width, n, lddo, lddt);
    OP_REQ(n <= 0x7fffffffL, PTCG_EINVAL, "embedding gradient: more than 2^31 - 1 places");
    OP_REQ((uintptr_t)dtable % 4 == 0, PTCG_EINVAL, "embedding gradient: dtable not aligned to its element");
    cudaStream_t s = (cudaStream_t)stream;
    if (n == 0) {
        if (!accumulate)
            OP_CK(cudaMemset2DAsync(dtable, lddt * 4, 0, (size_t)width * 4, vocab, s));
        return PTCG_OK;
    }
    OP_REQ(dout && ids && scratch, PTCG_EINVAL, "embedding gradient: null pointer");
    OP_REQ(el_ok(dout, dout_dtype) && (uintptr_t)ids % 4 == 0 && (uintptr_t)scratch % 16 == 0,
           PTCG_EINVAL, "embedding gradient: misaligned pointer (scratch: 16 bytes)");
    const Plan p = plan(n, vocab, width);
    OP_REQ(scratch_bytes >= p.bytes, PTCG_ERANGE, "embedding gradient: scratch of %ld bytes, %ld needed",
           scratch_bytes, p.bytes);
    uint8_t* base = (uint8_t*)scratch;
    uint32_t* keys[2] = {(uint32_t*)(base + p.o_keys[0]), (uint32_t*)(base + p.o_keys[1])};
    uint32_t* pos[2] = {(uint32_t*)(base + p.o_pos[0]), (uint32_t*)(base + p.o_pos[1])};
    const bool small = n <= SMALL_N;
    for (int i = 0; i < (small ? 1 : p.passes); i++) {
        const int to = i & 1;
        const SortArgs sa = {(uint32_t*)(base + p.o_counts), keys[to], pos[to], keys[to ^ 1], pos[to ^ 1],
                             ids, n, i * p.bits, p.bits, vocab, pad_id, pad_id >= 0};
        OP_CK(small ? (n <= SORT_T ? sort_small<1>(sa, p.passes, s) : sort_small<8>(sa, p.passes, s))
              : p.items == 16 ? (i == 0 ? sort_pass<16, true>(sa, p.tiles, s) : sort_pass<16, false>(sa, p.tiles, s))
                              : (i == 0 ? sort_pass<4, true>(sa, p.tiles, s) : sort_pass<4, false>(sa, p.tiles, s)));
    }
    const int last = small ? 0 : (p.passes - 1) & 1;
    SumArgs a;
    a.dout = dout; a.lddo = lddo;
    a.keys = keys[last]; a.pos = pos[last];
    a.n = n;
    a.dtab = dtable; a.lddt = lddt;
    a.head = (float*)(base + p.o_head); a.tail = (float*)(base + p.o_tail);
    a.flags = (uint32_t*)(base + p.o_flags); a.tail_id = (uint32_t*)(base + p.o_tid);
    a.vocab = vocab; a.width = width; a.pieces = 0; a.accumulate = accumulate != 0;
    a.chunk = p.chunk; a.run = 0; a.nchunks = p.nchunks; a.zero_blocks = 0;
    a.scale = scale;
    const int v = dout_dtype == PTCG_BF16 ? 8 : 4;
    const int V = width % v == 0 && vec_ok(dout, dout_dtype, lddo, v) && vec_ok(dtable, PTCG_FP32, lddt, v) ? v : 1;
    if (dout_dtype == PTCG_BF16) embed_sum<bf16>(a, V, s); else embed_sum<float>(a, V, s);
    if (p.nchunks > 1) {
        const int cols = (int)cdiv(width, 32);
        ++g_ptcg_launches, k_embed_join<<<dim3(p.nchunks, cols < 4 ? cols : 4), 256, 0, s>>>(a);
    }
    OP_CKL();
    return PTCG_OK;
}

}  // extern "C"
