// Cross attention: query rows over an encoder's states (or a cache) of
// another length, forward and backward, head width 32, 64 or 128.
//   S = scale q k^T over the kept keys, lse = log sum exp S, P = exp(S - lse),
//   out = P v;
//   delta = dout . out, dS = P o (dout v^T - delta),
//   dq = scale dS k, dk = scale dS^T q, dv = P^T dout.
// There is no order between queries and keys, so the lq rows of the query
// heads that share a key head are stacked into R = group * lq rows of one
// problem per (sequence, key head): grouped heads fill the same tiles as more
// queries would, and dk / dv sum over the group by themselves.
//
// Masked keys never reach a sum: their K and V rows become zeros in shared
// memory (not loaded, or cleared after a tile's TMA copy) and their
// probabilities are set to 0, so whatever they hold (NaN, infinities, rows
// never written) has no effect.  Their own gradients are written as zeros, not
// as the sums of zeros times dout, which may hold infinities.
#include <algorithm>

#include "cross.cuh"

namespace {

using namespace cross;

// ------------------------------------------------------- mma.sync pieces
PTCG_DEV void ldsm4(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}
PTCG_DEV void ldsm4t(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}
PTCG_DEV void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
                 "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// bf16 tiles of DH columns without padding: the 16-byte pieces of a row are
// permuted by the row so that the eight rows an ldmatrix phase touches fall
// into different banks (a 64-byte row shares its 128-byte line with its
// neighbour, hence row / 2 there)
template <int DH> PTCG_DEV uint32_t tile_off(int row, int piece) {
    const int x = DH == 32 ? (row >> 1) & 3 : row & 7;
    return (uint32_t)(row * DH * 2 + ((piece ^ x) << 4));
}
// This lane's part of an ldmatrix address: for A fragments of rows r0 .. +15 and
// for B fragments of B[k][n] = X[k][n] (rows k0 .. +15), or for B fragments of
// B[k][n] = X[n][k] (rows n0 .. +15).  Added to a tile's address (a multiple of
// 256 bytes), the 16-column step ks is an exclusive or of the piece bits and the
// row step a constant, so one address serves all fragments of a tile.
template <int DH> PTCG_DEV uint32_t lane_rows(int lane) {
    return tile_off<DH>(((lane >> 3) & 1) * 8 + (lane & 7), lane >> 4);
}
template <int DH> PTCG_DEV uint32_t lane_cols(int lane) {
    return tile_off<DH>((lane >> 4) * 8 + (lane & 7), (lane >> 3) & 1);
}
template <int DH> PTCG_DEV void frag(uint32_t (&f)[4], uint32_t at, int r0, int ks) {
    ldsm4(f, (at ^ (uint32_t)(ks * 32)) + r0 * DH * 2);
}
template <int DH> PTCG_DEV void frag_t(uint32_t (&f)[4], uint32_t at, int r0, int ks) {
    ldsm4t(f, (at ^ (uint32_t)(ks * 32)) + r0 * DH * 2);
}
// Staging: a thread takes piece tid % P of rows tid / P, + THREADS / P, ..; that
// step is a multiple of 8 rows, so the permutation, and with it the offset in
// the tile, moves by a constant.
template <int DH, int THREADS> struct Lanes {
    static constexpr int P = DH / 8, STEP = THREADS / P;
    static_assert(STEP % 8 == 0, "the tile's permutation repeats every 8 rows");
    int r, c;
    uint32_t off;
    PTCG_DEV Lanes() : r(threadIdx.x / P), c(threadIdx.x % P), off(tile_off<DH>(r, c)) {}
};
// stacked query rows r0 .. +N into a tile; rows past R are zeros
template <int DH, int N, int THREADS>
PTCG_DEV void stage_q(uint32_t dst, const bf16* src, const PtcgHeads& s, const CrossArgs& a,
                      int seq, int hk, int r0) {
    const Lanes<DH, THREADS> l;
    const bf16* base = src + seq * s.seq + (long)(hk * a.group) * s.head + l.c * 8;
    #pragma unroll
    for (int n = 0; n < N; n += l.STEP) {
        if (N % l.STEP && l.r + n >= N) break;
        const int r = r0 + l.r + n;
        const bool in = r < a.rows;
        const int g = a.by_lq.div(in ? r : 0), i = (in ? r : 0) - g * a.lq;
        cp16(dst + l.off + n * DH * 2, base + i * s.row + g * s.head, in);
    }
}
// key rows j0 .. +N into a tile; rows whose bit is clear are zeros and are not read
template <int DH, int N, int THREADS>
PTCG_DEV void stage_k(uint32_t dst, const bf16* src, const PtcgHeads& s, int seq, int hk, int j0,
                      const uint32_t* bits) {
    const Lanes<DH, THREADS> l;
    const bf16* base = src + krow(s, seq, hk, j0 + l.r) + l.c * 8;
    #pragma unroll
    for (int n = 0; n < N; n += l.STEP) {
        const int r = l.r + n;
        const bool in = (bits[r >> 5] >> (r & 31)) & 1;
        cp16(dst + l.off + n * DH * 2, in ? base + n * s.row : src, in);
    }
}
PTCG_DEV float quad_max(float v) {
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
    return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
PTCG_DEV float quad_sum(float v) {
    v += __shfl_xor_sync(0xffffffffu, v, 1);
    return v + __shfl_xor_sync(0xffffffffu, v, 2);
}
// ---------------------------------------------------------- bf16 forward
// A block owns 16 WM stacked rows and walks its keys 64 at a time through NST
// cp.async stages; the running maximum, sum and output rows stay in registers
// and P goes from the accumulators of S straight into the operand of P V
// (rounded to bf16: at most 2^-8 of each probability, the size of the output's
// own rounding).  WN = 4 is the form for at most 16 rows (single tokens): the
// four warps take 16 keys each of every tile and are joined at the end.
// Bound: HBM with few rows (single tokens, 16 heads on 4, width 128: 8 caches of
// 65536 keys 168 us, 6.4 TB/s; unequal ones of 436 MB 77 us, 5.7 TB/s), the launch
// for one decision (4.1 us), else issue slots around the products.
template <int DH, int WM, int WN, int NST>
__global__ void __launch_bounds__(WM * WN * 32, DH == 32 && WN == 1 ? 5 : 1) k_cross_fwd(const __grid_constant__ CrossArgs a) {
    constexpr int THREADS = WM * WN * 32, BM = WM * 16, BN = 64, KW = BN / WN, NT = KW / 8;
    constexpr int KS = DH / 16, TILE = BN * DH * 2;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = (uint8_t*)(((uintptr_t)smem_raw + 255) & ~(uintptr_t)255);
    __shared__ uint32_t bits[NST + 1][2];
    // 0 for a kept key, -inf for a masked one: where the scores start from
    __shared__ __align__(8) float bias[NST + 1][BN];
    const uint32_t sQ = s_addr(sm), sK = sQ + BM * DH * 2, sV = sK + NST * TILE;
    Where at = where(a);
    int kbeg, kend;
    if (WN == 4 && a.want) {
        if (!even_part(a, at, kbeg, kend)) return;
    }
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t fr = lane_rows<DH>(lane), fc = lane_cols<DH>(lane);
    const int wm = WN == 1 ? warp : 0, wn = WN == 1 ? 0 : warp;
    const int r0 = at.tile * BM, len = kept_len(a, at.seq);
    if (WN != 4 || !a.want) {
        kbeg = min(at.part * a.split, len);
        kend = min(len, kbeg + a.split);
    }
    const int nt = (kend - kbeg + BN - 1) / BN;
    const bf16 *K = (const bf16*)a.k, *V = (const bf16*)a.v;

    auto mask_byte = [&](int j) {           // this lane's key of tile j
        const int key = kbeg + j * BN + warp * 32 + lane;
        return warp < 2 && key < kend && kept(a, at.seq, key, len);
    };
    auto put_bits = [&](int j, bool b) {
        const uint32_t m = __ballot_sync(0xffffffffu, b);
        if (warp < 2) {
            bias[j % (NST + 1)][warp * 32 + lane] = b ? 0.f : -INFINITY;
            if (lane == 0) bits[j % (NST + 1)][warp] = m;
        }
    };
    auto load = [&](int j) {
        if (j < nt) {
            const uint32_t* b = bits[j % (NST + 1)];
            stage_k<DH, BN, THREADS>(sK + (j % NST) * TILE, K, a.sk, at.seq, at.hk, kbeg + j * BN, b);
            stage_k<DH, BN, THREADS>(sV + (j % NST) * TILE, V, a.sv, at.seq, at.hk, kbeg + j * BN, b);
        }
        cp_commit();
    };
    #pragma unroll
    for (int j = 0; j < NST; j++) put_bits(j, mask_byte(j));
    stage_q<DH, BM, THREADS>(sQ, (const bf16*)a.q, a.sq, a, at.seq, at.hk, r0);
    __syncthreads();
    #pragma unroll
    for (int j = 0; j < NST - 1; j++) load(j);

    float o[DH / 8][4], m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    #pragma unroll
    for (int i = 0; i < DH / 8; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    uint32_t qf[KS][4];
    const float sc = a.scale * LOG2E;
    const int t = lane & 3;
    const bool mine = r0 + wm * 16 < a.rows;        // this warp has rows
    for (int j = 0; j < nt; j++) {
        const bool next = mask_byte(j + NST);
        cp_wait<NST - 2>();
        __syncthreads();
        load(j + NST - 1);
        if (j == 0) {
            #pragma unroll
            for (int ks = 0; ks < KS; ks++) frag<DH>(qf[ks], sQ + fr, wm * 16, ks);
        }
        const uint32_t w0 = bits[j % (NST + 1)][0], w1 = bits[j % (NST + 1)][1];
        // this warp's keys: all 64, or its 16
        const uint32_t v0 = WN == 1 ? w0 : ((wn & 2 ? w1 : w0) >> ((wn & 1) * 16)) & 0xffffu;
        const uint32_t v1 = WN == 1 ? w1 : 0u;
        if ((v0 | v1) && mine) {
            const uint32_t kt = sK + (j % NST) * TILE, vt = sV + (j % NST) * TILE;
            // 16 keys at a time; groups that are masked whole are skipped
            const float* bj = bias[j % (NST + 1)] + wn * KW + 2 * t;
            auto group = [&](int i) { return ((i < 2 ? v0 : v1) >> ((i & 1) * 16)) & 0xffffu; };
            float s[NT][4];
            #pragma unroll
            for (int i = 0; i < NT / 2; i++) {
                #pragma unroll
                for (int n = 2 * i; n < 2 * i + 2; n++) {
                    const float2 b = *(const float2*)(bj + n * 8);
                    s[n][0] = s[n][2] = b.x;
                    s[n][1] = s[n][3] = b.y;
                }
                if (!group(i)) continue;
                #pragma unroll
                for (int ks = 0; ks < KS; ks++) {
                    uint32_t b[4];
                    frag<DH>(b, kt + fc, wn * KW + i * 16, ks);
                    mma(s[2 * i], qf[ks], b[0], b[1]);
                    mma(s[2 * i + 1], qf[ks], b[2], b[3]);
                }
            }
            float x0 = -INFINITY, x1 = -INFINITY;
            #pragma unroll
            for (int i = 0; i < NT; i++) {
                x0 = fmaxf(x0, fmaxf(s[i][0], s[i][1]));
                x1 = fmaxf(x1, fmaxf(s[i][2], s[i][3]));
            }
            const float n0 = fmaxf(m0, quad_max(x0) * sc), n1 = fmaxf(m1, quad_max(x1) * sc);
            // a row whose keys so far are all masked keeps a zero sum
            const float u0 = n0 == -INFINITY ? 0.f : n0, u1 = n1 == -INFINITY ? 0.f : n1;
            if (__any_sync(0xffffffffu, n0 != m0 || n1 != m1)) {
                const float c0 = ex2_approx(m0 - u0), c1 = ex2_approx(m1 - u1);
                l0 *= c0;
                l1 *= c1;
                #pragma unroll
                for (int i = 0; i < DH / 8; i++) { o[i][0] *= c0; o[i][1] *= c0; o[i][2] *= c1; o[i][3] *= c1; }
            }
            m0 = n0;
            m1 = n1;
            #pragma unroll
            for (int i = 0; i < NT / 2; i++) {
                if (!group(i)) continue;
                #pragma unroll
                for (int n = 2 * i; n < 2 * i + 2; n++) {
                    s[n][0] = ex2_approx(fmaf(s[n][0], sc, -u0));
                    s[n][1] = ex2_approx(fmaf(s[n][1], sc, -u0));
                    s[n][2] = ex2_approx(fmaf(s[n][2], sc, -u1));
                    s[n][3] = ex2_approx(fmaf(s[n][3], sc, -u1));
                    l0 += s[n][0] + s[n][1];
                    l1 += s[n][2] + s[n][3];
                }
                const uint32_t p[4] = {pack_bf2(s[2 * i][0], s[2 * i][1]), pack_bf2(s[2 * i][2], s[2 * i][3]),
                                       pack_bf2(s[2 * i + 1][0], s[2 * i + 1][1]),
                                       pack_bf2(s[2 * i + 1][2], s[2 * i + 1][3])};
                #pragma unroll
                for (int d = 0; d < KS; d++) {
                    uint32_t b[4];
                    frag_t<DH>(b, vt + fr, wn * KW + i * 16, d);
                    mma(o[2 * d], p, b[0], b[1]);
                    mma(o[2 * d + 1], p, b[2], b[3]);
                }
            }
        }
        put_bits(j + NST, next);
    }
    cp_wait<0>();
    l0 = quad_sum(l0);
    l1 = quad_sum(l1);
    const int g = lane >> 2;
    if (WN > 1) {
        // join the four warps' key shares: [WN][16] max and sum, [WN][16][DH] output
        __syncthreads();
        float* jm = (float*)sm;
        float* jl = jm + WN * 16;
        float* jo = jl + WN * 16;
        if (t == 0) {
            jm[wn * 16 + g] = m0; jm[wn * 16 + g + 8] = m1;
            jl[wn * 16 + g] = l0; jl[wn * 16 + g + 8] = l1;
        }
        #pragma unroll
        for (int i = 0; i < DH / 8; i++) {
            float* p = jo + (wn * 16 + g) * DH + i * 8 + 2 * t;
            *(float2*)p = make_float2(o[i][0], o[i][1]);
            *(float2*)(p + 8 * DH) = make_float2(o[i][2], o[i][3]);
        }
        __syncthreads();
        for (int i = threadIdx.x; i < 16 * DH / 2; i += THREADS) {
            const int r = i / (DH / 2), d = i % (DH / 2) * 2;
            if (r0 + r >= a.rows) continue;
            float m = -INFINITY, l = 0.f, y0 = 0.f, y1 = 0.f;
            #pragma unroll
            for (int k = 0; k < WN; k++) m = fmaxf(m, jm[k * 16 + r]);
            const float u = m == -INFINITY ? 0.f : m;
            #pragma unroll
            for (int k = 0; k < WN; k++) {
                const float c = ex2_approx(jm[k * 16 + r] - u);
                const float2 x = *(const float2*)(jo + (k * 16 + r) * DH + d);
                l = fmaf(jl[k * 16 + r], c, l);
                y0 = fmaf(x.x, c, y0);
                y1 = fmaf(x.y, c, y1);
            }
            const long row = ((long)at.seq * a.kv_heads + at.hk) * a.rows + r0 + r;
            if (a.nsplit > 1) {
                *(float2*)(a.part + (row * a.nsplit + at.part) * DH + d) = make_float2(y0, y1);
                if (d == 0) a.part_ml[row * a.nsplit + at.part] = make_float2(m, l);
            } else {
                const float inv = l == 0.f ? 0.f : 1.f / l;
                *(uint32_t*)((bf16*)a.out + qrow(a, a.so, at.seq, at.hk, r0 + r) + d) =
                    pack_bf2(y0 * inv, y1 * inv);
                if (d == 0 && a.lse) a.lse[row] = l == 0.f ? -INFINITY : (m + log2f(l)) * LN2;
            }
        }
        return;
    }
    const float i0 = l0 == 0.f ? 0.f : 1.f / l0, i1 = l1 == 0.f ? 0.f : 1.f / l1;
    #pragma unroll
    for (int half = 0; half < 2; half++) {
        const int r = r0 + wm * 16 + g + half * 8;
        if (r >= a.rows) continue;
        const long row = ((long)at.seq * a.kv_heads + at.hk) * a.rows + r;
        const float m = half ? m1 : m0, l = half ? l1 : l0, inv = half ? i1 : i0;
        if (a.nsplit > 1) {
            float* p = a.part + (row * a.nsplit + at.part) * DH;
            #pragma unroll
            for (int i = 0; i < DH / 8; i++)
                *(float2*)(p + i * 8 + 2 * t) = make_float2(o[i][2 * half], o[i][2 * half + 1]);
            if (t == 0) a.part_ml[row * a.nsplit + at.part] = make_float2(m, l);
        } else {
            bf16* p = (bf16*)a.out + qrow(a, a.so, at.seq, at.hk, r);
            #pragma unroll
            for (int i = 0; i < DH / 8; i++)
                *(uint32_t*)(p + i * 8 + 2 * t) = pack_bf2(o[i][2 * half] * inv, o[i][2 * half + 1] * inv);
            if (t == 0 && a.lse) a.lse[row] = l == 0.f ? -INFINITY : (m + log2f(l)) * LN2;
        }
    }
}

// The form for keys that fit a block's shared memory whole (a board's rows, a
// short context): nothing is pipelined, the masks are read once, and each warp
// walks the 16-key groups that have a kept key two at a time.  The tiled kernel
// spends some 390 instructions a warp on every 64 keys besides the groups' own
// 45 (staging, barriers, stages, masked groups' maxima); here that is paid once:
// 1024 x 8 problems of 64 rows on 129 keys, width 32, 58 us against 75, 8192 x 8
// of them 413 us (3.9 TB/s).  Bound: issue slots (69 % taken) and shared memory
// (42 % of its wavefronts).
constexpr int SHORT_KEYS = 256;

// mask words and score offsets of all keys (a multiple of 32 of them, up to
// SHORT_KEYS), by the block's four warps
PTCG_DEV void short_masks(const CrossArgs& a, int seq, int len, uint32_t* words, float* bias) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = (a.lk + 31) / 32;
    const uint8_t* keep = a.keep ? a.keep + (long)seq * a.lk : nullptr;
    #pragma unroll
    for (int i = 0; i < SHORT_KEYS / 128; i++) {
        const int w = warp + 4 * i, key = w * 32 + lane;
        if (w >= n) break;
        const bool in = key < len && (!keep || keep[key] != 0);
        const uint32_t m = __ballot_sync(0xffffffffu, in);
        bias[key] = in ? 0.f : -INFINITY;
        if (lane == 0) words[w] = m;
    }
}
// bit i: 16-key group i has a kept key
PTCG_DEV uint32_t short_groups(const CrossArgs& a, const uint32_t* words, int lane) {
    const bool in = lane * 16 < a.lk && ((words[lane >> 1] >> ((lane & 1) * 16)) & 0xffffu);
    return __ballot_sync(0xffffffffu, in);
}
// all kept rows of K and V (zeros for masked ones)
template <int DH>
PTCG_DEV void short_stage(const CrossArgs& a, const Where& at, uint32_t sK, uint32_t sV, int rows, const uint32_t* words) {
    const Lanes<DH, 128> l;
    const bf16* k = (const bf16*)a.k + krow(a.sk, at.seq, at.hk, l.r) + l.c * 8;
    const bf16* v = (const bf16*)a.v + krow(a.sv, at.seq, at.hk, l.r) + l.c * 8;
    const long dk = l.STEP * a.sk.row, dv = l.STEP * a.sv.row;
    uint32_t off = l.off;
    for (int r = l.r; r < rows; r += l.STEP) {
        const bool in = (words[r >> 5] >> (r & 31)) & 1;
        cp16(sK + off, in ? k : (const bf16*)a.k, in);
        cp16(sV + off, in ? v : (const bf16*)a.v, in);
        k += dk;
        v += dv;
        off += l.STEP * DH * 2;
    }
}

template <int DH>
__global__ void __launch_bounds__(128, DH == 32 ? 6 : DH == 64 ? 3 : 2) k_cross_fwd_short(const __grid_constant__ CrossArgs a) {
    constexpr int BM = 64, KS = DH / 16;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = (uint8_t*)(((uintptr_t)smem_raw + 255) & ~(uintptr_t)255);
    __shared__ uint32_t words[SHORT_KEYS / 32];
    __shared__ __align__(8) float bias[SHORT_KEYS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, keys = (a.lk + 15) & ~15;
    const uint32_t sQ = s_addr(sm), sK = sQ + BM * DH * 2, sV = sK + keys * DH * 2;
    const Where at = where(a);
    const int r0 = at.tile * BM, len = kept_len(a, at.seq);
    stage_q<DH, BM, 128>(sQ, (const bf16*)a.q, a.sq, a, at.seq, at.hk, r0);
    short_masks(a, at.seq, len, words, bias);
    __syncthreads();
    short_stage<DH>(a, at, sK, sV, keys, words);
    uint32_t rem = short_groups(a, words, lane);
    cp_commit();
    cp_wait<0>();
    __syncthreads();
    if (r0 + warp * 16 >= a.rows) return;
    const uint32_t fr = lane_rows<DH>(lane), kt = sK + lane_cols<DH>(lane), vt = sV + fr;
    uint32_t qf[KS][4];
    #pragma unroll
    for (int ks = 0; ks < KS; ks++) frag<DH>(qf[ks], sQ + fr, warp * 16, ks);
    float o[DH / 8][4], m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    #pragma unroll
    for (int i = 0; i < DH / 8; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    const float sc = a.scale * LOG2E;
    const int g = lane >> 2, t = lane & 3;
    while (rem) {
        const int ka = __ffs(rem) - 1;
        rem &= rem - 1;
        const bool two = rem != 0;
        const int kb = two ? __ffs(rem) - 1 : ka;
        rem &= rem - 1;                             // 0 stays 0
        float s[4][4];
        #pragma unroll
        for (int n = 0; n < 4; n++) {
            const float2 b = *(const float2*)(bias + (n < 2 ? ka : kb) * 16 + (n & 1) * 8 + 2 * t);
            s[n][0] = s[n][2] = n < 2 || two ? b.x : -INFINITY;
            s[n][1] = s[n][3] = n < 2 || two ? b.y : -INFINITY;
        }
        #pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            uint32_t b[4];
            frag<DH>(b, kt, ka * 16, ks);
            mma(s[0], qf[ks], b[0], b[1]);
            mma(s[1], qf[ks], b[2], b[3]);
        }
        if (two) {
            #pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                uint32_t b[4];
                frag<DH>(b, kt, kb * 16, ks);
                mma(s[2], qf[ks], b[0], b[1]);
                mma(s[3], qf[ks], b[2], b[3]);
            }
        }
        float x0 = fmaxf(s[0][0], s[0][1]), x1 = fmaxf(s[0][2], s[0][3]);
        #pragma unroll
        for (int n = 1; n < 4; n++) {
            x0 = fmaxf(x0, fmaxf(s[n][0], s[n][1]));
            x1 = fmaxf(x1, fmaxf(s[n][2], s[n][3]));
        }
        // a kept key among these: the maxima are finite unless the scores are not
        const float n0 = fmaxf(m0, quad_max(x0) * sc), n1 = fmaxf(m1, quad_max(x1) * sc);
        const float u0 = n0 == -INFINITY ? 0.f : n0, u1 = n1 == -INFINITY ? 0.f : n1;
        if (__any_sync(0xffffffffu, n0 != m0 || n1 != m1)) {
            const float c0 = ex2_approx(m0 - u0), c1 = ex2_approx(m1 - u1);
            l0 *= c0;
            l1 *= c1;
            #pragma unroll
            for (int i = 0; i < DH / 8; i++) { o[i][0] *= c0; o[i][1] *= c0; o[i][2] *= c1; o[i][3] *= c1; }
            m0 = n0;
            m1 = n1;
        }
        #pragma unroll
        for (int h = 0; h < 2; h++) {
            if (h == 1 && !two) break;
            #pragma unroll
            for (int n = 2 * h; n < 2 * h + 2; n++) {
                s[n][0] = ex2_approx(fmaf(s[n][0], sc, -u0));
                s[n][1] = ex2_approx(fmaf(s[n][1], sc, -u0));
                s[n][2] = ex2_approx(fmaf(s[n][2], sc, -u1));
                s[n][3] = ex2_approx(fmaf(s[n][3], sc, -u1));
                l0 += s[n][0] + s[n][1];
                l1 += s[n][2] + s[n][3];
            }
            const uint32_t p[4] = {pack_bf2(s[2 * h][0], s[2 * h][1]), pack_bf2(s[2 * h][2], s[2 * h][3]),
                                   pack_bf2(s[2 * h + 1][0], s[2 * h + 1][1]),
                                   pack_bf2(s[2 * h + 1][2], s[2 * h + 1][3])};
            #pragma unroll
            for (int d = 0; d < KS; d++) {
                uint32_t b[4];
                frag_t<DH>(b, vt, (h ? kb : ka) * 16, d);
                mma(o[2 * d], p, b[0], b[1]);
                mma(o[2 * d + 1], p, b[2], b[3]);
            }
        }
    }
    l0 = quad_sum(l0);
    l1 = quad_sum(l1);
    #pragma unroll
    for (int half = 0; half < 2; half++) {
        const int r = r0 + warp * 16 + g + half * 8;
        if (r >= a.rows) continue;
        const float m = half ? m1 : m0, l = half ? l1 : l0, inv = l == 0.f ? 0.f : 1.f / l;
        bf16* p = (bf16*)a.out + qrow(a, a.so, at.seq, at.hk, r) + 2 * t;
        #pragma unroll
        for (int i = 0; i < DH / 8; i++)
            *(uint32_t*)(p + i * 8) = pack_bf2(o[i][2 * half] * inv, o[i][2 * half + 1] * inv);
        if (t == 0 && a.lse)
            a.lse[((long)at.seq * a.kv_heads + at.hk) * a.rows + r] = l == 0.f ? -INFINITY : (m + log2f(l)) * LN2;
    }
}

// joins the parts of a split forward: a block per stacked row, whose warps take
// every fourth part and are added in order (single tokens over a long cache
// have few rows, and each has many parts).  A part's maximum comes as the shift
// that its exponentials took, of e in fp32 and of 2 in bf16: turned into the
// other base it would be rounded, and the part's weight be off by that much (554
// half units of 2^-24 at scores of 1000)
template <typename T, int DH>
__global__ void __launch_bounds__(128) k_cross_join(const __grid_constant__ CrossArgs a) {
    constexpr int C = DH / 32;                      // columns a lane
    constexpr bool F32 = sizeof(T) == 4;
    __shared__ float sy[4][DH], sl[4];
    const long row = blockIdx.x;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long b = row / a.rows;
    const int seq = (int)(b / a.kv_heads), hk = (int)(b % a.kv_heads), r = (int)(row - b * a.rows);
    int parts = a.nsplit;
    if (a.want) {
        const unsigned len = even_length(a);
        parts = (int)((even_units(a, seq) + len - 1) / len);
    }
    const float2* ml = a.part_ml + row * a.nsplit;
    float m = -INFINITY;
    for (int i = lane; i < parts; i += 32) m = fmaxf(m, ml[i].x);
    m = warp_max(m);
    const float u = m == -INFINITY ? 0.f : m;
    float l = 0.f, y[C];
    #pragma unroll
    for (int e = 0; e < C; e++) y[e] = 0.f;
    const float* p = a.part + row * a.nsplit * DH + lane;
    #pragma unroll 8
    for (int i = warp; i < parts; i += 4) {
        const float2 x = ml[i];
        const float c = F32 ? expf(x.x - u) : ex2_approx(x.x - u);
        l = fmaf(x.y, c, l);
        #pragma unroll
        for (int e = 0; e < C; e++) y[e] = fmaf(p[(long)i * DH + e * 32], c, y[e]);
    }
    #pragma unroll
    for (int e = 0; e < C; e++) sy[warp][e * 32 + lane] = y[e];
    if (lane == 0) sl[warp] = l;
    __syncthreads();
    l = sl[0] + sl[1] + sl[2] + sl[3];
    const float inv = l == 0.f ? 0.f : 1.f / l;
    for (int d = threadIdx.x; d < DH; d += 128)
        ((T*)a.out + qrow(a, a.so, seq, hk, r))[d] = from_f<T>((sy[0][d] + sy[1][d] + sy[2][d] + sy[3][d]) * inv);
    if (threadIdx.x == 0 && a.lse) a.lse[row] = l == 0.f ? -INFINITY : F32 ? m + logf(l) : (m + log2f(l)) * LN2;
}

// --------------------------------------------------------- bf16 backward
// A quad's accumulators hold two columns of each 8-column piece per lane;
// handed around, lane t has the whole of piece t out of four and stores 16
// bytes: the short backward below took 932 us so, 965 with 4-byte stores (the
// forward has a third of its stores and loses by it, 413 to 418 us).
PTCG_DEV uint4 quad_piece(uint32_t v0, uint32_t v1, uint32_t v2, uint32_t v3, int t) {
    const bool odd = t & 1, hi = t & 2;
    const uint32_t r0 = __shfl_xor_sync(0xffffffffu, odd ? v0 : v1, 1);
    const uint32_t r1 = __shfl_xor_sync(0xffffffffu, odd ? v2 : v3, 1);
    // two words of piece t & 1 and of piece 2 + (t & 1)
    const uint32_t a0 = odd ? r0 : v0, a1 = odd ? v1 : r0, b0 = odd ? r1 : v2, b1 = odd ? v3 : r1;
    const uint32_t c0 = __shfl_xor_sync(0xffffffffu, hi ? a0 : b0, 2);
    const uint32_t c1 = __shfl_xor_sync(0xffffffffu, hi ? a1 : b1, 2);
    return hi ? make_uint4(c0, c1, b0, b1) : make_uint4(a0, a1, c0, c1);
}
// the accumulators' upper or lower row times f as bf16 (zeros where `keep` is not
// all ones); every lane takes part, those with `in` store
template <int DH>
PTCG_DEV void put_acc(bf16* row, int t, bool in, float f, const float (&acc)[DH / 8][4], int half,
                      uint32_t keep = 0xffffffffu) {
    #pragma unroll
    for (int j = 0; j < DH / 8; j += 4) {
        uint32_t v[4];
        #pragma unroll
        for (int i = 0; i < 4; i++) v[i] = pack_bf2(acc[j + i][2 * half] * f, acc[j + i][2 * half + 1] * f);
        const uint4 w = quad_piece(v[0] & keep, v[1] & keep, v[2] & keep, v[3] & keep, t);
        if (in) *(uint4*)(row + (j + t) * 8) = w;
    }
}
template <int DH>
PTCG_DEV void put_zeros(bf16* row, int t) {
    #pragma unroll
    for (int j = 0; j < DH / 8; j += 4) *(uint4*)(row + (j + t) * 8) = make_uint4(0u, 0u, 0u, 0u);
}

// dq: a block owns 64 stacked rows (16 a warp) with q, dout and dq in
// registers and walks the keys; it also writes delta = dout . out for the
// dk / dv kernel.  S is computed again from q and k: reading stored
// probabilities would cost lk numbers a row.
template <int DH>
__global__ void __launch_bounds__(128) k_cross_dq(const __grid_constant__ CrossArgs a) {
    constexpr int THREADS = 128, BM = 64, BN = DH == 128 ? 32 : 64, NT = BN / 8, KS = DH / 16;
    constexpr int TILE = BN * DH * 2;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = (uint8_t*)(((uintptr_t)smem_raw + 255) & ~(uintptr_t)255);
    __shared__ uint32_t bits[3][2];
    __shared__ float s_delta[BM];
    const uint32_t sK = s_addr(sm), sV = sK + 2 * TILE, sQ = sV + 2 * TILE, sG = sQ + BM * DH * 2;
    const Where at = where(a);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t fr = lane_rows<DH>(lane), fc = lane_cols<DH>(lane);
    const int r0 = at.tile * BM, len = kept_len(a, at.seq);
    const int kbeg = min(at.part * a.split, len), kend = min(len, kbeg + a.split);
    const int nt = (kend - kbeg + BN - 1) / BN;
    const bf16 *K = (const bf16*)a.k, *V = (const bf16*)a.v;
    const long row0 = ((long)at.seq * a.kv_heads + at.hk) * a.rows;
    auto mask_byte = [&](int j) {
        const int key = kbeg + j * BN + warp * 32 + lane;
        return warp < BN / 32 && key < kend && kept(a, at.seq, key, len);
    };
    auto put_bits = [&](int j, bool b) {
        const uint32_t m = __ballot_sync(0xffffffffu, b);
        if (warp < 2 && lane == 0) bits[j % 3][warp] = m;
    };
    auto load = [&](int j) {
        if (j < nt) {
            stage_k<DH, BN, THREADS>(sK + (j & 1) * TILE, K, a.sk, at.seq, at.hk, kbeg + j * BN, bits[j % 3]);
            stage_k<DH, BN, THREADS>(sV + (j & 1) * TILE, V, a.sv, at.seq, at.hk, kbeg + j * BN, bits[j % 3]);
        }
        cp_commit();
    };
    put_bits(0, mask_byte(0));
    put_bits(1, mask_byte(1));
    stage_q<DH, BM, THREADS>(sQ, (const bf16*)a.q, a.sq, a, at.seq, at.hk, r0);
    stage_q<DH, BM, THREADS>(sG, (const bf16*)a.dout, a.sdo, a, at.seq, at.hk, r0);
    __syncthreads();
    load(0);
    {   // delta: two threads a row
        const int r = threadIdx.x >> 1, h = threadIdx.x & 1;
        float d = 0.f;
        if (r0 + r < a.rows) {
            const bf16* og = (const bf16*)a.o + qrow(a, a.so, at.seq, at.hk, r0 + r) + h * (DH / 2);
            const bf16* gg = (const bf16*)a.dout + qrow(a, a.sdo, at.seq, at.hk, r0 + r) + h * (DH / 2);
            #pragma unroll
            for (int c = 0; c < DH / 16; c++) {
                float x[8], y[8];
                VecIO<bf16, 8>::ld(x, og + c * 8);
                VecIO<bf16, 8>::ld(y, gg + c * 8);
                #pragma unroll
                for (int e = 0; e < 8; e++) d = fmaf(x[e], y[e], d);
            }
        }
        d += __shfl_xor_sync(0xffffffffu, d, 1);
        if (h == 0) {
            s_delta[r] = d;
            if (r0 + r < a.rows && at.part == 0) a.delta[row0 + r0 + r] = d;
        }
    }
    const int g = lane >> 2, t = lane & 3;
    const int ra = r0 + warp * 16 + g, rb = ra + 8;
    // log2-domain lse; +inf makes the probabilities of a row without keys
    // (and of rows past the end) zero
    float la = ra < a.rows ? a.lse[row0 + ra] : -INFINITY, lb = rb < a.rows ? a.lse[row0 + rb] : -INFINITY;
    la = la == -INFINITY ? INFINITY : la * LOG2E;
    lb = lb == -INFINITY ? INFINITY : lb * LOG2E;
    const float sc = a.scale * LOG2E;
    float dq[DH / 8][4];
    #pragma unroll
    for (int i = 0; i < DH / 8; i++) dq[i][0] = dq[i][1] = dq[i][2] = dq[i][3] = 0.f;
    uint32_t qf[KS][4], gf[KS][4];
    float da = 0.f, db = 0.f;
    for (int j = 0; j < nt; j++) {
        const bool next = mask_byte(j + 2);
        cp_wait<0>();
        __syncthreads();
        load(j + 1);
        if (j == 0) {
            #pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                frag<DH>(qf[ks], sQ + fr, warp * 16, ks);
                frag<DH>(gf[ks], sG + fr, warp * 16, ks);
            }
            da = s_delta[warp * 16 + g];
            db = s_delta[warp * 16 + g + 8];
        }
        const uint32_t w0 = bits[j % 3][0], w1 = BN == 64 ? bits[j % 3][1] : 0u;
        if (w0 | w1) {
            const uint32_t kt = sK + (j & 1) * TILE, vt = sV + (j & 1) * TILE;
            float s[NT][4], p[NT][4];
            #pragma unroll
            for (int i = 0; i < NT; i++) {
                s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
                p[i][0] = p[i][1] = p[i][2] = p[i][3] = 0.f;
            }
            #pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                #pragma unroll
                for (int i = 0; i < NT / 2; i++) {
                    uint32_t b[4];
                    frag<DH>(b, kt + fc, i * 16, ks);
                    mma(s[2 * i], qf[ks], b[0], b[1]);
                    mma(s[2 * i + 1], qf[ks], b[2], b[3]);
                    frag<DH>(b, vt + fc, i * 16, ks);
                    mma(p[2 * i], gf[ks], b[0], b[1]);
                    mma(p[2 * i + 1], gf[ks], b[2], b[3]);
                }
            }
            #pragma unroll
            for (int i = 0; i < NT; i++) {
                const uint32_t w = (i < 4 ? w0 : w1) >> ((i & 3) * 8 + 2 * t);
                const float e0 = w & 1 ? ex2_approx(fmaf(s[i][0], sc, -la)) : 0.f;
                const float e1 = w & 2 ? ex2_approx(fmaf(s[i][1], sc, -la)) : 0.f;
                const float e2 = w & 1 ? ex2_approx(fmaf(s[i][2], sc, -lb)) : 0.f;
                const float e3 = w & 2 ? ex2_approx(fmaf(s[i][3], sc, -lb)) : 0.f;
                s[i][0] = e0 * (p[i][0] - da);
                s[i][1] = e1 * (p[i][1] - da);
                s[i][2] = e2 * (p[i][2] - db);
                s[i][3] = e3 * (p[i][3] - db);
            }
            #pragma unroll
            for (int i = 0; i < NT / 2; i++) {
                const uint32_t f[4] = {pack_bf2(s[2 * i][0], s[2 * i][1]), pack_bf2(s[2 * i][2], s[2 * i][3]),
                                       pack_bf2(s[2 * i + 1][0], s[2 * i + 1][1]),
                                       pack_bf2(s[2 * i + 1][2], s[2 * i + 1][3])};
                #pragma unroll
                for (int d = 0; d < KS; d++) {
                    uint32_t b[4];
                    frag_t<DH>(b, kt + fr, i * 16, d);
                    mma(dq[2 * d], f, b[0], b[1]);
                    mma(dq[2 * d + 1], f, b[2], b[3]);
                }
            }
        }
        put_bits(j + 2, next);
    }
    cp_wait<0>();
    #pragma unroll
    for (int half = 0; half < 2; half++) {
        const int r = half ? rb : ra;
        const bool in = r < a.rows;
        if (a.nsplit > 1) {
            if (!in) continue;
            float* p = a.part + ((row0 + r) * a.nsplit + at.part) * DH;
            #pragma unroll
            for (int i = 0; i < DH / 8; i++)
                *(float2*)(p + i * 8 + 2 * t) = make_float2(dq[i][2 * half] * a.scale, dq[i][2 * half + 1] * a.scale);
        } else {
            put_acc<DH>((bf16*)a.dq + qrow(a, a.sdq, at.seq, at.hk, r), t, in, a.scale, dq, half);
        }
    }
}

// dk, dv: a block owns 64 keys (16 a warp) and walks the stacked rows; S^T and
// dP^T come out with keys as rows, so P^T and dS^T are the left operands of
// dv += P^T dout and dk += dS^T q straight from the accumulators.
template <int DH>
__global__ void __launch_bounds__(128) k_cross_dkv(const __grid_constant__ CrossArgs a) {
    constexpr int THREADS = 128, BK = 64, BQ = DH == 128 ? 32 : 64, NT = BQ / 8, KS = DH / 16;
    constexpr int QT = BQ * DH * 2;
    constexpr bool REGS = DH < 128;              // k and v fragments stay in registers
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = (uint8_t*)(((uintptr_t)smem_raw + 255) & ~(uintptr_t)255);
    __shared__ uint32_t bits[2];
    __shared__ float s_lse[2][BQ], s_delta[2][BQ];
    const uint32_t sK = s_addr(sm), sV = sK + BK * DH * 2, sQ = sV + BK * DH * 2, sG = sQ + 2 * QT;
    const Where at = where(a);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t fr = lane_rows<DH>(lane), fc = lane_cols<DH>(lane);
    const int j0 = at.tile * BK, len = kept_len(a, at.seq);
    const int qbeg = min(at.part * a.split, a.rows), qend = min(a.rows, qbeg + a.split);
    const int nt = (qend - qbeg + BQ - 1) / BQ;
    const long row0 = ((long)at.seq * a.kv_heads + at.hk) * a.rows;
    {
        const int key = j0 + warp * 32 + lane;
        const uint32_t m = __ballot_sync(0xffffffffu, warp < 2 && kept(a, at.seq, key, len));
        if (warp < 2 && lane == 0) bits[warp] = m;
    }
    __syncthreads();
    const uint32_t w0 = bits[0], w1 = bits[1];
    const bool any = (w0 | w1) != 0;
    auto load = [&](int j) {
        if (j < nt) {
            stage_q<DH, BQ, THREADS>(sQ + (j & 1) * QT, (const bf16*)a.q, a.sq, a, at.seq, at.hk, qbeg + j * BQ);
            stage_q<DH, BQ, THREADS>(sG + (j & 1) * QT, (const bf16*)a.dout, a.sdo, a, at.seq, at.hk, qbeg + j * BQ);
        }
        cp_commit();
    };
    float lv = 0.f, dl = 0.f;
    auto load_stat = [&](int j) {
        const int r = qbeg + j * BQ + threadIdx.x;
        const bool in = threadIdx.x < BQ && r < qend;
        lv = in ? a.lse[row0 + r] : -INFINITY;
        lv = lv == -INFINITY ? INFINITY : lv * LOG2E;
        dl = in ? a.delta[row0 + r] : 0.f;
    };
    auto put_stat = [&](int j) {
        if (threadIdx.x < BQ) { s_lse[j & 1][threadIdx.x] = lv; s_delta[j & 1][threadIdx.x] = dl; }
    };
    float dk[DH / 8][4], dv[DH / 8][4];
    #pragma unroll
    for (int i = 0; i < DH / 8; i++) {
        dk[i][0] = dk[i][1] = dk[i][2] = dk[i][3] = 0.f;
        dv[i][0] = dv[i][1] = dv[i][2] = dv[i][3] = 0.f;
    }
    const int g = lane >> 2, t = lane & 3;
    const uint32_t wk = (warp & 2 ? w1 : w0) >> ((warp & 1) * 16);
    const bool ka = (wk >> g) & 1, kb = (wk >> (g + 8)) & 1;
    if (any) {
        stage_k<DH, BK, THREADS>(sK, (const bf16*)a.k, a.sk, at.seq, at.hk, j0, bits);
        stage_k<DH, BK, THREADS>(sV, (const bf16*)a.v, a.sv, at.seq, at.hk, j0, bits);
        load(0);
        load_stat(0);
        const float sc = a.scale * LOG2E;
        uint32_t kf[REGS ? KS : 1][4], vf[REGS ? KS : 1][4];
        for (int j = 0; j < nt; j++) {
            put_stat(j);
            load_stat(j + 1);
            cp_wait<0>();
            __syncthreads();
            load(j + 1);
            if (REGS && j == 0) {
                #pragma unroll
                for (int ks = 0; ks < KS; ks++) {
                    frag<DH>(kf[REGS ? ks : 0], sK + fr, warp * 16, ks);
                    frag<DH>(vf[REGS ? ks : 0], sV + fr, warp * 16, ks);
                }
            }
            const uint32_t qt = sQ + (j & 1) * QT, gt = sG + (j & 1) * QT;
            float s[NT][4], p[NT][4];
            #pragma unroll
            for (int i = 0; i < NT; i++) {
                s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
                p[i][0] = p[i][1] = p[i][2] = p[i][3] = 0.f;
            }
            #pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                if (!REGS) {
                    frag<DH>(kf[0], sK + fr, warp * 16, ks);
                    frag<DH>(vf[0], sV + fr, warp * 16, ks);
                }
                #pragma unroll
                for (int i = 0; i < NT / 2; i++) {
                    uint32_t b[4];
                    frag<DH>(b, qt + fc, i * 16, ks);
                    mma(s[2 * i], kf[REGS ? ks : 0], b[0], b[1]);
                    mma(s[2 * i + 1], kf[REGS ? ks : 0], b[2], b[3]);
                    frag<DH>(b, gt + fc, i * 16, ks);
                    mma(p[2 * i], vf[REGS ? ks : 0], b[0], b[1]);
                    mma(p[2 * i + 1], vf[REGS ? ks : 0], b[2], b[3]);
                }
            }
            #pragma unroll
            for (int i = 0; i < NT; i++) {
                const int c = i * 8 + 2 * t;
                const float x0 = s_lse[j & 1][c], x1 = s_lse[j & 1][c + 1];
                const float d0 = s_delta[j & 1][c], d1 = s_delta[j & 1][c + 1];
                s[i][0] = ka ? ex2_approx(fmaf(s[i][0], sc, -x0)) : 0.f;
                s[i][1] = ka ? ex2_approx(fmaf(s[i][1], sc, -x1)) : 0.f;
                s[i][2] = kb ? ex2_approx(fmaf(s[i][2], sc, -x0)) : 0.f;
                s[i][3] = kb ? ex2_approx(fmaf(s[i][3], sc, -x1)) : 0.f;
                p[i][0] = s[i][0] * (p[i][0] - d0);
                p[i][1] = s[i][1] * (p[i][1] - d1);
                p[i][2] = s[i][2] * (p[i][2] - d0);
                p[i][3] = s[i][3] * (p[i][3] - d1);
            }
            #pragma unroll
            for (int i = 0; i < NT / 2; i++) {
                const uint32_t pf[4] = {pack_bf2(s[2 * i][0], s[2 * i][1]), pack_bf2(s[2 * i][2], s[2 * i][3]),
                                        pack_bf2(s[2 * i + 1][0], s[2 * i + 1][1]),
                                        pack_bf2(s[2 * i + 1][2], s[2 * i + 1][3])};
                const uint32_t df[4] = {pack_bf2(p[2 * i][0], p[2 * i][1]), pack_bf2(p[2 * i][2], p[2 * i][3]),
                                        pack_bf2(p[2 * i + 1][0], p[2 * i + 1][1]),
                                        pack_bf2(p[2 * i + 1][2], p[2 * i + 1][3])};
                #pragma unroll
                for (int d = 0; d < KS; d++) {
                    uint32_t b[4];
                    frag_t<DH>(b, gt + fr, i * 16, d);
                    mma(dv[2 * d], pf, b[0], b[1]);
                    mma(dv[2 * d + 1], pf, b[2], b[3]);
                    frag_t<DH>(b, qt + fr, i * 16, d);
                    mma(dk[2 * d], df, b[0], b[1]);
                    mma(dk[2 * d + 1], df, b[2], b[3]);
                }
            }
        }
        cp_wait<0>();
    }
    #pragma unroll
    for (int half = 0; half < 2; half++) {
        const int j = j0 + warp * 16 + g + half * 8;
        const bool in = j < a.lk, live = half ? kb : ka;
        if (a.nsplit > 1) {
            if (!in) continue;
            const long at_row = (((long)at.seq * a.kv_heads + at.hk) * a.lk + j) * a.nsplit + at.part;
            #pragma unroll
            for (int i = 0; i < DH / 8; i++) {
                const float2 z = make_float2(0.f, 0.f);
                *(float2*)(a.part + at_row * DH + i * 8 + 2 * t) = live ? make_float2(dk[i][2 * half] * a.scale, dk[i][2 * half + 1] * a.scale) : z;
                *(float2*)(a.part2 + at_row * DH + i * 8 + 2 * t) = live ? make_float2(dv[i][2 * half], dv[i][2 * half + 1]) : z;
            }
        } else {
            const uint32_t keep = live ? 0xffffffffu : 0u;
            put_acc<DH>((bf16*)a.dk + krow(a.sdk, at.seq, at.hk, j), t, in, a.scale, dk, half, keep);
            put_acc<DH>((bf16*)a.dv + krow(a.sdv, at.seq, at.hk, j), t, in, 1.f, dv, half, keep);
        }
    }
}

// a dq row of a warp that has its 16-column pieces d0, d0 + DR, .. (all of them
// with 64 rows)
template <int DH, int NR, int N>
PTCG_DEV void put_dq(bf16* row, int t, int d0, bool in, float f, const float (&dq)[N][4], int half) {
    if constexpr (NR == 4) {
        put_acc<DH>(row, t, in, f, dq, half);
    } else {
        #pragma unroll
        for (int i = 0; i < N; i++) {
            const int c = (d0 + (i >> 1) * (4 / NR)) * 16 + (i & 1) * 8;
            if (in && c < DH) *(uint32_t*)(row + c + 2 * t) = pack_bf2(dq[i][2 * half] * f, dq[i][2 * half + 1] * f);
        }
    }
}

// Backward of problems of at most 64 stacked rows in one kernel: the rows stay
// in shared memory while a block walks the keys 64 at a time, so S, P and dS
// are computed once (five products instead of the seven of the pair above) and
// a key tile's dk and dv are finished at once.  S^T and dP^T have keys as rows
// (16 a warp); dS^T goes through shared memory, from where the warps take it
// transposed as the left operand of dq += dS k (16 rows and a share of the
// columns each), which stays in registers over all keys.  512 x 8 problems of 64
// rows on 600 keys of width 64, some 350 of them kept: 416 us (the tiled forward
// 222); bound by latency: two blocks a processor, by their registers.
template <int DH, int NR>                    // 16 NR rows
__global__ void __launch_bounds__(128, DH == 32 ? 4 : 1) k_cross_bwd_rows(const __grid_constant__ CrossArgs a) {
    constexpr int THREADS = 128, BM = NR * 16, BN = 64, KS = DH / 16, TILE = BN * DH * 2;
    constexpr int NT = BM / 8;               // 8-row tiles of the stacked rows
    constexpr int DR = 4 / NR > 0 ? 4 / NR : 1;             // warps that share a group of 16 rows
    constexpr int ND = (KS + DR - 1) / DR;   // 16-column pieces of dq a warp owns
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = (uint8_t*)(((uintptr_t)smem_raw + 255) & ~(uintptr_t)255);
    __shared__ uint32_t bits[3][2];
    __shared__ float s_lse[BM], s_delta[BM];
    const uint32_t sQ = s_addr(sm), sG = sQ + BM * DH * 2, sK = sG + BM * DH * 2, sV = sK + 2 * TILE;
    const uint32_t sD = sV + 2 * TILE;       // dS^T [64 keys][BM rows], rows of 16 bytes permuted
    const Where at = where(a);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t fr = lane_rows<DH>(lane), fc = lane_cols<DH>(lane);
    const int len = kept_len(a, at.seq);
    // parts tile [0, lk), so that the masked tail's dk and dv are written too
    const int kbeg = at.part * a.split, kend = min(a.lk, kbeg + a.split);
    const int nt = (kend - kbeg + BN - 1) / BN;
    const bf16 *K = (const bf16*)a.k, *V = (const bf16*)a.v;
    const long row0 = ((long)at.seq * a.kv_heads + at.hk) * a.rows;
    auto mask_byte = [&](int j) {
        const int key = kbeg + j * BN + warp * 32 + lane;
        return warp < 2 && key < kend && kept(a, at.seq, key, len);
    };
    auto put_bits = [&](int j, bool b) {
        const uint32_t m = __ballot_sync(0xffffffffu, b);
        if (warp < 2 && lane == 0) bits[j % 3][warp] = m;
    };
    auto load = [&](int j) {
        if (j < nt) {
            stage_k<DH, BN, THREADS>(sK + (j & 1) * TILE, K, a.sk, at.seq, at.hk, kbeg + j * BN, bits[j % 3]);
            stage_k<DH, BN, THREADS>(sV + (j & 1) * TILE, V, a.sv, at.seq, at.hk, kbeg + j * BN, bits[j % 3]);
        }
        cp_commit();
    };
    put_bits(0, mask_byte(0));
    put_bits(1, mask_byte(1));
    stage_q<DH, BM, THREADS>(sQ, (const bf16*)a.q, a.sq, a, at.seq, at.hk, 0);
    stage_q<DH, BM, THREADS>(sG, (const bf16*)a.dout, a.sdo, a, at.seq, at.hk, 0);
    __syncthreads();
    load(0);
    {   // delta = dout . out, THREADS / BM threads a row, and the log2-domain lse
        // (+inf makes the probabilities of rows without keys and past the end zero)
        constexpr int TR = THREADS / BM, PC = DH / 8;       // threads a row, 16-byte pieces
        const int r = threadIdx.x / TR, h = threadIdx.x % TR;
        float d = 0.f;
        if (r < a.rows) {
            const bf16* og = (const bf16*)a.o + qrow(a, a.so, at.seq, at.hk, r);
            const bf16* gg = (const bf16*)a.dout + qrow(a, a.sdo, at.seq, at.hk, r);
            for (int c = h; c < PC; c += TR) {
                float x[8], y[8];
                VecIO<bf16, 8>::ld(x, og + c * 8);
                VecIO<bf16, 8>::ld(y, gg + c * 8);
                #pragma unroll
                for (int e = 0; e < 8; e++) d = fmaf(x[e], y[e], d);
            }
        }
        #pragma unroll
        for (int o = 1; o < TR; o <<= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
        if (h == 0) {
            const float x = r < a.rows ? a.lse[row0 + r] : -INFINITY;
            s_lse[r] = x == -INFINITY ? INFINITY : x * LOG2E;
            s_delta[r] = d;
        }
    }
    const int g = lane >> 2, t = lane & 3, mi = lane >> 3;
    const float sc = a.scale * LOG2E;
    const int qr = NR == 1 ? 0 : warp % NR, qd = NR == 1 ? warp : warp / NR;   // dq rows, first column piece
    float dq[2 * ND][4];
    #pragma unroll
    for (int i = 0; i < 2 * ND; i++) dq[i][0] = dq[i][1] = dq[i][2] = dq[i][3] = 0.f;
    // 16-byte piece c (8 rows) of key row k of the dS^T tile
    auto ds_off = [&](int k, int c) {
        return sD + (uint32_t)(k * BM * 2 + ((c ^ (NT == 8 ? k & 7 : NT == 4 ? (k >> 1) & 3 : (k >> 2) & 1)) << 4));
    };
    for (int j = 0; j < nt; j++) {
        const bool next = mask_byte(j + 2);
        cp_wait<0>();
        __syncthreads();
        load(j + 1);
        const uint32_t w0 = bits[j % 3][0], w1 = bits[j % 3][1];
        const uint32_t wk = ((warp & 2 ? w1 : w0) >> ((warp & 1) * 16)) & 0xffffu;
        const uint32_t kt = sK + (j & 1) * TILE, vt = sV + (j & 1) * TILE;
        const int ja = kbeg + j * BN + warp * 16 + g;
        bf16* pk = (bf16*)a.dk + krow(a.sdk, at.seq, at.hk, ja);
        bf16* pv = (bf16*)a.dv + krow(a.sdv, at.seq, at.hk, ja);
        const bool ina = ja < kend, inb = ja + 8 < kend;
        if (wk) {
            float s[NT][4], p[NT][4];
            // the scores of a masked key start, and stay, at -inf
            const float ma = (wk >> g) & 1 ? 0.f : -INFINITY, mb = (wk >> (g + 8)) & 1 ? 0.f : -INFINITY;
            #pragma unroll
            for (int i = 0; i < NT; i++) {
                s[i][0] = s[i][1] = ma;
                s[i][2] = s[i][3] = mb;
                p[i][0] = p[i][1] = p[i][2] = p[i][3] = 0.f;
            }
            #pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                uint32_t kf[4], vf[4];
                frag<DH>(kf, kt + fr, warp * 16, ks);
                frag<DH>(vf, vt + fr, warp * 16, ks);
                #pragma unroll
                for (int i = 0; i < NT / 2; i++) {
                    uint32_t b[4];
                    frag<DH>(b, sQ + fc, i * 16, ks);
                    mma(s[2 * i], kf, b[0], b[1]);
                    mma(s[2 * i + 1], kf, b[2], b[3]);
                    frag<DH>(b, sG + fc, i * 16, ks);
                    mma(p[2 * i], vf, b[0], b[1]);
                    mma(p[2 * i + 1], vf, b[2], b[3]);
                }
            }
            uint32_t pf[NT / 2][4], df[NT / 2][4];
            #pragma unroll
            for (int i = 0; i < NT; i++) {
                const int c = i * 8 + 2 * t;
                const float x0 = s_lse[c], x1 = s_lse[c + 1], d0 = s_delta[c], d1 = s_delta[c + 1];
                const float e0 = ex2_approx(fmaf(s[i][0], sc, -x0)), e1 = ex2_approx(fmaf(s[i][1], sc, -x1));
                const float e2 = ex2_approx(fmaf(s[i][2], sc, -x0)), e3 = ex2_approx(fmaf(s[i][3], sc, -x1));
                pf[i >> 1][(i & 1) * 2] = pack_bf2(e0, e1);
                pf[i >> 1][(i & 1) * 2 + 1] = pack_bf2(e2, e3);
                const uint32_t da = pack_bf2(e0 * (p[i][0] - d0), e1 * (p[i][1] - d1));
                const uint32_t db = pack_bf2(e2 * (p[i][2] - d0), e3 * (p[i][3] - d1));
                df[i >> 1][(i & 1) * 2] = da;
                df[i >> 1][(i & 1) * 2 + 1] = db;
                asm volatile("st.shared.b32 [%0], %1;" :: "r"(ds_off(warp * 16 + g, i) + 4 * t), "r"(da) : "memory");
                asm volatile("st.shared.b32 [%0], %1;" :: "r"(ds_off(warp * 16 + g + 8, i) + 4 * t), "r"(db) : "memory");
            }
            #pragma unroll
            for (int which = 0; which < 2; which++) {
                float acc[DH / 8][4];
                #pragma unroll
                for (int i = 0; i < DH / 8; i++) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
                #pragma unroll
                for (int i = 0; i < NT / 2; i++) {
                    #pragma unroll
                    for (int d = 0; d < KS; d++) {
                        uint32_t b[4];
                        frag_t<DH>(b, (which ? sQ : sG) + fr, i * 16, d);
                        mma(acc[2 * d], which ? df[i] : pf[i], b[0], b[1]);
                        mma(acc[2 * d + 1], which ? df[i] : pf[i], b[2], b[3]);
                    }
                }
                const float f = which ? a.scale : 1.f;
                bf16* out = which ? pk : pv;
                const long down = 8 * (which ? a.sdk.row : a.sdv.row);
                put_acc<DH>(out, t, ina, f, acc, 0, (wk >> g) & 1 ? 0xffffffffu : 0u);
                put_acc<DH>(out + down, t, inb, f, acc, 1, (wk >> (g + 8)) & 1 ? 0xffffffffu : 0u);
            }
        } else {                                 // masked keys: no gradient
            if (ina) { put_zeros<DH>(pk, t); put_zeros<DH>(pv, t); }
            if (inb) { put_zeros<DH>(pk + 8 * a.sdk.row, t); put_zeros<DH>(pv + 8 * a.sdv.row, t); }
        }
        put_bits(j + 2, next);
        if (w0 | w1) {                           // the same for every warp
            __syncthreads();
            #pragma unroll
            for (int k = 0; k < BN / 16; k++) {
                if (!(((k & 2 ? w1 : w0) >> ((k & 1) * 16)) & 0xffffu)) continue;
                uint32_t f[4];                   // dS rows 16 qr .., keys 16 k ..
                ldsm4t(f, ds_off(k * 16 + (mi >> 1) * 8 + (lane & 7), qr * 2 + (mi & 1)));
                #pragma unroll
                for (int i = 0; i < ND; i++) {
                    const int d = qd + i * DR;
                    if (d >= KS) break;
                    uint32_t b[4];
                    frag_t<DH>(b, kt + fr, k * 16, d);
                    mma(dq[2 * i], f, b[0], b[1]);
                    mma(dq[2 * i + 1], f, b[2], b[3]);
                }
            }
        }
    }
    cp_wait<0>();
    #pragma unroll
    for (int half = 0; half < 2; half++) {
        const int r = qr * 16 + g + half * 8;
        if (a.nsplit == 1) {
            put_dq<DH, NR>((bf16*)a.dq + qrow(a, a.sdq, at.seq, at.hk, r), t, qd, r < a.rows, a.scale, dq, half);
            continue;
        }
        if (r >= a.rows) continue;
        float* p = a.part + ((row0 + r) * a.nsplit + at.part) * DH + 2 * t;
        #pragma unroll
        for (int i = 0; i < 2 * ND; i++) {
            const int c = (qd + (i >> 1) * DR) * 16 + (i & 1) * 8;
            if (c < DH) *(float2*)(p + c) = make_float2(dq[i][2 * half] * a.scale, dq[i][2 * half + 1] * a.scale);
        }
    }
}

// The same for keys that fit shared memory whole: every warp takes each fourth
// 16-key group that has a kept key, dS^T of all of them is kept, and dq is one
// product at the end; three barriers in all.  8192 x 8 problems of 64 rows on
// 129 keys, width 32: 915 us (3.6 TB/s; with the forward 1318, in 64-key tiles
// 1730).  Bound: 16 warps a processor, as shared memory allows, with half of
// shared memory's wavefronts (every warp reads q and dout as fragments, dS^T is
// written and read back) and of the issue slots taken, the tensor pipe at 25 %.
template <int DH, int NR>                    // 16 NR rows
__global__ void __launch_bounds__(128, DH == 32 ? 4 : DH == 64 ? 2 : 1) k_cross_bwd_short(const __grid_constant__ CrossArgs a) {
    constexpr int BM = NR * 16, KS = DH / 16, NT = BM / 8;
    constexpr int DR = 4 / NR, ND = (KS + DR - 1) / DR;
    constexpr int TR = 128 / BM, PC = DH / 8 / TR > 0 ? DH / 8 / TR : 1;   // threads a row, pieces each
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = (uint8_t*)(((uintptr_t)smem_raw + 255) & ~(uintptr_t)255);
    __shared__ uint32_t words[SHORT_KEYS / 32];
    __shared__ float bias[SHORT_KEYS];
    __shared__ __align__(8) float s_lse[BM], s_delta[BM];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, keys = (a.lk + 15) & ~15;
    const uint32_t sQ = s_addr(sm), sG = sQ + BM * DH * 2, sK = sG + BM * DH * 2, sV = sK + keys * DH * 2;
    const uint32_t sD = sV + keys * DH * 2;  // dS^T [keys][BM rows], rows of 16 bytes permuted
    const Where at = where(a);
    const int len = kept_len(a, at.seq);
    const long row0 = ((long)at.seq * a.kv_heads + at.hk) * a.rows;
    stage_q<DH, BM, 128>(sQ, (const bf16*)a.q, a.sq, a, at.seq, at.hk, 0);
    stage_q<DH, BM, 128>(sG, (const bf16*)a.dout, a.sdo, a, at.seq, at.hk, 0);
    cp_commit();
    // the row whose delta this thread shares in: out and the log-sum-exp come now
    const int dr = threadIdx.x / TR, dp = threadIdx.x % TR;
    uint4 og[PC];
    float lr = -INFINITY;
    if (dr < a.rows) {
        const uint4* p = (const uint4*)((const bf16*)a.o + qrow(a, a.so, at.seq, at.hk, dr));
        #pragma unroll
        for (int c = 0; c < PC; c++) og[c] = dp + c * TR < DH / 8 ? p[dp + c * TR] : make_uint4(0u, 0u, 0u, 0u);
        lr = a.lse[row0 + dr];
    } else {
        #pragma unroll
        for (int c = 0; c < PC; c++) og[c] = make_uint4(0u, 0u, 0u, 0u);
    }
    short_masks(a, at.seq, len, words, bias);
    __syncthreads();
    short_stage<DH>(a, at, sK, sV, keys, words);
    const uint32_t active = short_groups(a, words, lane);
    cp_commit();
    cp_wait<1>();
    __syncthreads();
    {
        float d = 0.f;
        #pragma unroll
        for (int c = 0; c < PC; c++) {
            if (dp + c * TR >= DH / 8) break;
            uint4 y;
            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(y.x), "=r"(y.y), "=r"(y.z), "=r"(y.w)
                         : "r"(sG + tile_off<DH>(dr, dp + c * TR)));
            const uint32_t u[4] = {og[c].x, og[c].y, og[c].z, og[c].w}, v[4] = {y.x, y.y, y.z, y.w};
            #pragma unroll
            for (int e = 0; e < 4; e++) {
                float u0, u1, v0, v1;
                unpack_bf2(u[e], u0, u1);
                unpack_bf2(v[e], v0, v1);
                d = fmaf(u0, v0, fmaf(u1, v1, d));
            }
        }
        #pragma unroll
        for (int o = 1; o < TR; o <<= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
        if (dp == 0) {
            s_lse[dr] = lr == -INFINITY ? INFINITY : lr * LOG2E;
            s_delta[dr] = d;
        }
    }
    cp_wait<0>();
    __syncthreads();
    const int g = lane >> 2, t = lane & 3, mi = lane >> 3;
    const uint32_t fr = lane_rows<DH>(lane), fc = lane_cols<DH>(lane);
    const float sc = a.scale * LOG2E;
    // 16-byte piece c (8 rows) of key row k of dS^T
    auto ds_off = [&](int k, int c) {
        return sD + (uint32_t)(k * BM * 2 + ((c ^ (NT == 8 ? k & 7 : NT == 4 ? (k >> 1) & 3 : (k >> 2) & 1)) << 4));
    };
    const int groups = keys / 16;
    int turn = 0;
    for (int k = 0; k < groups; k++) {
        const bool on = (active >> k) & 1;
        if (((on ? turn++ : k) & 3) != warp) continue;
        const int ja = k * 16 + g;
        const bool ina = ja < a.lk, inb = ja + 8 < a.lk;
        bf16* pk = (bf16*)a.dk + krow(a.sdk, at.seq, at.hk, ja);
        bf16* pv = (bf16*)a.dv + krow(a.sdv, at.seq, at.hk, ja);
        if (!on) {                               // masked keys: no gradient
            if (ina) { put_zeros<DH>(pk, t); put_zeros<DH>(pv, t); }
            if (inb) { put_zeros<DH>(pk + 8 * a.sdk.row, t); put_zeros<DH>(pv + 8 * a.sdv.row, t); }
            continue;
        }
        float s[NT][4], p[NT][4];
        const float ma = bias[ja], mb = bias[ja + 8];
        #pragma unroll
        for (int i = 0; i < NT; i++) {
            s[i][0] = s[i][1] = ma;
            s[i][2] = s[i][3] = mb;
            p[i][0] = p[i][1] = p[i][2] = p[i][3] = 0.f;
        }
        #pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            uint32_t kf[4], vf[4];
            frag<DH>(kf, sK + fr, k * 16, ks);
            frag<DH>(vf, sV + fr, k * 16, ks);
            #pragma unroll
            for (int i = 0; i < NT / 2; i++) {
                uint32_t b[4];
                frag<DH>(b, sQ + fc, i * 16, ks);
                mma(s[2 * i], kf, b[0], b[1]);
                mma(s[2 * i + 1], kf, b[2], b[3]);
                frag<DH>(b, sG + fc, i * 16, ks);
                mma(p[2 * i], vf, b[0], b[1]);
                mma(p[2 * i + 1], vf, b[2], b[3]);
            }
        }
        uint32_t pf[NT / 2][4], df[NT / 2][4];
        #pragma unroll
        for (int i = 0; i < NT; i++) {
            const float2 x = *(const float2*)(s_lse + i * 8 + 2 * t), d = *(const float2*)(s_delta + i * 8 + 2 * t);
            const float e0 = ex2_approx(fmaf(s[i][0], sc, -x.x)), e1 = ex2_approx(fmaf(s[i][1], sc, -x.y));
            const float e2 = ex2_approx(fmaf(s[i][2], sc, -x.x)), e3 = ex2_approx(fmaf(s[i][3], sc, -x.y));
            pf[i >> 1][(i & 1) * 2] = pack_bf2(e0, e1);
            pf[i >> 1][(i & 1) * 2 + 1] = pack_bf2(e2, e3);
            const uint32_t da = pack_bf2(e0 * (p[i][0] - d.x), e1 * (p[i][1] - d.y));
            const uint32_t db = pack_bf2(e2 * (p[i][2] - d.x), e3 * (p[i][3] - d.y));
            df[i >> 1][(i & 1) * 2] = da;
            df[i >> 1][(i & 1) * 2 + 1] = db;
            asm volatile("st.shared.b32 [%0], %1;" :: "r"(ds_off(ja, i) + 4 * t), "r"(da) : "memory");
            asm volatile("st.shared.b32 [%0], %1;" :: "r"(ds_off(ja + 8, i) + 4 * t), "r"(db) : "memory");
        }
        #pragma unroll
        for (int which = 0; which < 2; which++) {
            float acc[DH / 8][4];
            #pragma unroll
            for (int i = 0; i < DH / 8; i++) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
            #pragma unroll
            for (int i = 0; i < NT / 2; i++) {
                #pragma unroll
                for (int d = 0; d < KS; d++) {
                    uint32_t b[4];
                    frag_t<DH>(b, (which ? sQ : sG) + fr, i * 16, d);
                    mma(acc[2 * d], which ? df[i] : pf[i], b[0], b[1]);
                    mma(acc[2 * d + 1], which ? df[i] : pf[i], b[2], b[3]);
                }
            }
            const float f = which ? a.scale : 1.f;
            bf16* out = which ? pk : pv;
            const long down = 8 * (which ? a.sdk.row : a.sdv.row);
            put_acc<DH>(out, t, ina, f, acc, 0, ma == 0.f ? 0xffffffffu : 0u);
            put_acc<DH>(out + down, t, inb, f, acc, 1, mb == 0.f ? 0xffffffffu : 0u);
        }
    }
    __syncthreads();
    const int qr = NR == 1 ? 0 : warp % NR, qd = NR == 1 ? warp : warp / NR;   // dq rows, first column piece
    float dq[2 * ND][4];
    #pragma unroll
    for (int i = 0; i < 2 * ND; i++) dq[i][0] = dq[i][1] = dq[i][2] = dq[i][3] = 0.f;
    for (uint32_t rem = active; rem; rem &= rem - 1) {
        const int k = __ffs(rem) - 1;
        uint32_t f[4];                           // dS rows 16 qr .., keys 16 k ..
        ldsm4t(f, ds_off(k * 16 + (mi >> 1) * 8 + (lane & 7), qr * 2 + (mi & 1)));
        #pragma unroll
        for (int i = 0; i < ND; i++) {
            const int d = qd + i * DR;
            if (d >= KS) break;
            uint32_t b[4];
            frag_t<DH>(b, sK + fr, k * 16, d);
            mma(dq[2 * i], f, b[0], b[1]);
            mma(dq[2 * i + 1], f, b[2], b[3]);
        }
    }
    #pragma unroll
    for (int half = 0; half < 2; half++) {
        const int r = qr * 16 + g + half * 8;
        put_dq<DH, NR>((bf16*)a.dq + qrow(a, a.sdq, at.seq, at.hk, r), t, qd, r < a.rows, a.scale, dq, half);
    }
}

// sums the parts of a split gradient in order: one 4-column piece a thread.
// keys: the rows are key rows of a.dk (from part) and a.dv (from part2),
// else stacked rows of a.dq
template <typename T, int DH>
__global__ void __launch_bounds__(256) k_cross_sum(const __grid_constant__ CrossArgs a, long nrows, int keys) {
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    const long row = i / (DH / 4);
    const int c = (int)(i % (DH / 4)) * 4;
    if (row >= nrows) return;
    const long per = keys ? a.lk : a.rows, b = row / per;
    const int seq = (int)(b / a.kv_heads), hk = (int)(b % a.kv_heads), r = (int)(row - b * per);
    for (int which = 0; which < 1 + keys; which++) {
        const float* p = (which ? a.part2 : a.part) + row * a.nsplit * DH + c;
        float s[4] = {0.f, 0.f, 0.f, 0.f};
        for (int k = 0; k < a.nsplit; k++) {
            float v[4];
            VecIO<float, 4>::ld(v, p + (long)k * DH);
            #pragma unroll
            for (int e = 0; e < 4; e++) s[e] += v[e];
        }
        T* out = !keys ? (T*)a.dq + qrow(a, a.sdq, seq, hk, r)
                       : which ? (T*)a.dv + krow(a.sdv, seq, hk, r) : (T*)a.dk + krow(a.sdk, seq, hk, r);
        VecIO<T, 4>::st(out + c, s);
    }
}

// ------------------------------------------------------------------ fp32
// fp32 throughout, on the SIMT cores (a tensor core would round the operands).
// 128 threads as 8 x 16: thread (ty, tx) owns RT rows (row_of) and NC columns of every product, computed two multiply-adds
// at a time on the packed f32x2 path.  All tiles are row-major copies of the
// tensors (cp.async, pitch DH + 4 floats, so that the rows a quarter warp
// touches fall into different banks); two forms of product serve them:
//   mm_rows   acc[i][j] = sum_d A[row i][d] B[row tx + 16 j][d], pairs along d
//   mm_outer  acc[i][j] += sum_k A[k][row i] B[k][col j], pairs along the rows,
//             A a probability tile that the threads wrote with k as its row
// Exponentials are expf, right to 2 units in the last place over the whole
// range: the intrinsic's error grows with |x| (54 half units of 2^-24 at e^-82,
// 2 with expf), for 1 to 3 % less time (170 and 399 us below).
// Bound: the multiply-adds and the reads from shared memory that
// feed them: 512 x 8 problems of 61 rows on up to 186 keys of width 32 take
// 176 us forward and 403 backward (18 TFLOP/s over the kept keys); single
// tokens, 8 of them on caches of up to 20000 keys (8 heads on 2 of width 128),
// 86 us, as 16 rows are computed for the 4 there are.
template <int RT> PTCG_DEV int row_of(int ty, int i) {
    return RT == 8 ? (i >> 2) * 32 + ty * 4 + (i & 3) : ty * RT + i;
}
template <int NC> PTCG_DEV int col_of(int tx, int j) {
    return NC == 8 ? (j >> 2) * 64 + tx * 4 + (j & 3) : tx * NC + j;
}
// keys (or stacked rows) per tile of the fp32 kernels, and their pitch
template <int DH> struct F32 { static constexpr int BN = DH == 128 ? 32 : 64, LD = DH + 4; };

template <int RT, int NC, int DH>
PTCG_DEV void mm_rows(float (&acc)[RT][NC], const float* A, const float* B, int ty, int tx) {
    constexpr int LD = F32<DH>::LD;
    unsigned long long c[RT][NC];
    #pragma unroll
    for (int i = 0; i < RT; i++)
        #pragma unroll
        for (int j = 0; j < NC; j++) c[i][j] = 0ull;
    #pragma unroll 2
    for (int d = 0; d < DH; d += 4) {
        ulonglong2 b[NC];
        #pragma unroll
        for (int j = 0; j < NC; j++) b[j] = *reinterpret_cast<const ulonglong2*>(B + (tx + 16 * j) * LD + d);
        #pragma unroll
        for (int i = 0; i < RT; i++) {
            const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(A + row_of<RT>(ty, i) * LD + d);
            #pragma unroll
            for (int j = 0; j < NC; j++) c[i][j] = fma2(x.y, b[j].y, fma2(x.x, b[j].x, c[i][j]));
        }
    }
    #pragma unroll
    for (int i = 0; i < RT; i++)
        #pragma unroll
        for (int j = 0; j < NC; j++) {
            float lo, hi;
            upk2(c[i][j], lo, hi);
            acc[i][j] = lo + hi;
        }
}
template <int RT, int NC, int K>
PTCG_DEV void mm_outer(float (&acc)[RT][NC], const float* A, int lda, const float* B, int ldb, int ty, int tx) {
    unsigned long long c[RT / 2][NC];
    #pragma unroll
    for (int i = 0; i < RT / 2; i++)
        #pragma unroll
        for (int j = 0; j < NC; j++) c[i][j] = pk2(acc[2 * i][j], acc[2 * i + 1][j]);
    #pragma unroll 4
    for (int k = 0; k < K; k++) {
        unsigned long long x[RT / 2];
        #pragma unroll
        for (int i = 0; i < RT; i += 4) {
            const float* p = A + k * lda + row_of<RT>(ty, i);
            if constexpr (RT >= 4) {
                const ulonglong2 u = *reinterpret_cast<const ulonglong2*>(p);
                x[i / 2] = u.x;
                x[i / 2 + 1] = u.y;
            } else {
                x[0] = *reinterpret_cast<const unsigned long long*>(p);
            }
        }
        float y[NC];
        #pragma unroll
        for (int j = 0; j < NC; j += 4) {
            const float* p = B + k * ldb + col_of<NC>(tx, j);
            if constexpr (NC >= 4) {
                const float4 v = *reinterpret_cast<const float4*>(p);
                y[j] = v.x; y[j + 1] = v.y; y[j + 2] = v.z; y[j + 3] = v.w;
            } else {
                const float2 v = *reinterpret_cast<const float2*>(p);
                y[0] = v.x; y[1] = v.y;
            }
        }
        #pragma unroll
        for (int j = 0; j < NC; j++) {
            const unsigned long long s = splat2(y[j]);
            #pragma unroll
            for (int i = 0; i < RT / 2; i++) c[i][j] = fma2(x[i], s, c[i][j]);
        }
    }
    #pragma unroll
    for (int i = 0; i < RT / 2; i++)
        #pragma unroll
        for (int j = 0; j < NC; j++) upk2(c[i][j], acc[2 * i][j], acc[2 * i + 1][j]);
}
template <int RT, int NC> PTCG_DEV void clear(float (&acc)[RT][NC]) {
    #pragma unroll
    for (int i = 0; i < RT; i++)
        #pragma unroll
        for (int j = 0; j < NC; j++) acc[i][j] = 0.f;
}
// the same, the tile's products summed by themselves first: one rounding of the
// running sum per tile, not per row of it, so that long sums stay as exact as
// short ones: out is off by 2.6e-7 of its size at 300 keys and at 20000 (a sum
// over all keys grows with the root of their number); 1 to 3 % of the time
template <int RT, int NC, int K>
PTCG_DEV void mm_outer_add(float (&acc)[RT][NC], const float* A, int lda, const float* B, int ldb, int ty, int tx) {
    float y[RT][NC];
    clear(y);
    mm_outer<RT, NC, K>(y, A, lda, B, ldb, ty, tx);
    #pragma unroll
    for (int i = 0; i < RT; i++)
        #pragma unroll
        for (int j = 0; j < NC; j++) acc[i][j] += y[i][j];
}
// the thread's RT values of column k into row k of a [k][row] tile
template <int RT> PTCG_DEV void put_rows(float* T, int ld, int k, int ty, const float (&v)[RT]) {
    #pragma unroll
    for (int i = 0; i < RT; i += 4) {
        float* p = T + k * ld + row_of<RT>(ty, i);
        if constexpr (RT >= 4) *reinterpret_cast<float4*>(p) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        else *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
    }
}
// one thread's columns of a result row
template <int NC> PTCG_DEV void put_cols(float* p, int tx, const float (&v)[NC], float f) {
    #pragma unroll
    for (int j = 0; j < NC; j += 4) {
        float* q = p + col_of<NC>(tx, j);
        if constexpr (NC >= 4) *reinterpret_cast<float4*>(q) = make_float4(v[j] * f, v[j + 1] * f, v[j + 2] * f, v[j + 3] * f);
        else *reinterpret_cast<float2*>(q) = make_float2(v[0] * f, v[1] * f);
    }
}
// N rows of DH floats, asynchronously; row(r) gives the source or null (zeros)
template <int DH, int N, typename F>
PTCG_DEV void stage_f32(float* dst, const float* any, F row) {
    constexpr int P = DH / 4, STEP = 128 / P;
    const int r0 = threadIdx.x / P, c = threadIdx.x % P * 4;
    const uint32_t to = s_addr(dst + r0 * F32<DH>::LD + c);
    #pragma unroll
    for (int n = 0; n < N; n += STEP) {
        if (N % STEP && r0 + n >= N) break;
        const float* p = row(r0 + n);
        cp16(to + n * F32<DH>::LD * 4, p ? p + c : any, p != nullptr);
    }
}
PTCG_DEV float row16_max(float v) {
    #pragma unroll
    for (int o = 1; o < 16; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
PTCG_DEV float row16_sum(float v) {
    #pragma unroll
    for (int o = 1; o < 16; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
PTCG_DEV const float* q_ptr(const CrossArgs& a, const void* p, const PtcgHeads& s, const Where& at, int r, int end) {
    return r < end ? (const float*)p + qrow(a, s, at.seq, at.hk, r) : nullptr;
}
PTCG_DEV const float* k_ptr(const void* p, const PtcgHeads& s, const Where& at, int j, bool ok) {
    return ok ? (const float*)p + krow(s, at.seq, at.hk, j) : nullptr;
}
// lse as the backward uses it: +inf makes the probabilities of rows without
// keys and of rows past the end zero
PTCG_DEV float lse_or_inf(const CrossArgs& a, long row, bool in) {
    const float x = in ? a.lse[row] : -INFINITY;
    return x == -INFINITY ? INFINITY : x;
}
// delta = dout . out of row r, whose dout lies in shared memory
template <int DH> PTCG_DEV float delta_f32(const CrossArgs& a, const Where& at, int r, const float* g) {
    const float* o = (const float*)a.o + qrow(a, a.so, at.seq, at.hk, r);
    float d = 0.f;
    #pragma unroll 4
    for (int c = 0; c < DH; c += 4) {
        const float4 x = *reinterpret_cast<const float4*>(o + c), y = *reinterpret_cast<const float4*>(g + c);
        d = fmaf(x.x, y.x, fmaf(x.y, y.y, fmaf(x.z, y.z, fmaf(x.w, y.w, d))));
    }
    return d;
}

template <int DH, int RT>
__global__ void __launch_bounds__(128, RT == 8 && DH == 32 ? 4 : 1) k_cross_fwd_f32(const __grid_constant__ CrossArgs a) {
    constexpr int BM = RT * 8, LM = BM + 4, BN = F32<DH>::BN, LD = F32<DH>::LD, NC = BN / 16, ND = DH / 16;
    extern __shared__ __align__(16) float fs[];
    __shared__ uint8_t ok[BN];
    float* Qs = fs;                  // [BM][LD]
    float* Ks = Qs + BM * LD;        // [BN][LD]
    float* Vs = Ks + BN * LD;        // [BN][LD]
    float* Ps = Vs + BN * LD;        // [BN][LM]
    Where at = where(a);
    int kbeg, kend;
    if (RT == 2 && a.want) {
        if (!even_part(a, at, kbeg, kend)) return;
    }
    const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
    const int r0 = at.tile * BM, len = kept_len(a, at.seq);
    if (RT != 2 || !a.want) {
        kbeg = min(at.part * a.split, len);
        kend = min(len, kbeg + a.split);
    }
    stage_f32<DH, BM>(Qs, (const float*)a.q, [&](int r) { return q_ptr(a, a.q, a.sq, at, r0 + r, a.rows); });
    float o[RT][ND], m[RT], l[RT];
    clear(o);
    #pragma unroll
    for (int i = 0; i < RT; i++) { m[i] = -INFINITY; l[i] = 0.f; }
    for (int k0 = kbeg; k0 < kend; k0 += BN) {
        const int key = k0 + threadIdx.x;
        const bool in = threadIdx.x < BN && key < kend && kept(a, at.seq, key, len);
        __syncthreads();                             // the last tile is done with
        if (threadIdx.x < BN) ok[threadIdx.x] = in;
        if (!__syncthreads_or(in)) continue;
        stage_f32<DH, BN>(Ks, (const float*)a.k, [&](int r) { return k_ptr(a.k, a.sk, at, k0 + r, ok[r]); });
        cp_commit();
        stage_f32<DH, BN>(Vs, (const float*)a.v, [&](int r) { return k_ptr(a.v, a.sv, at, k0 + r, ok[r]); });
        cp_commit();
        cp_wait<1>();
        __syncthreads();
        float s[RT][NC];
        mm_rows<RT, NC, DH>(s, Qs, Ks, ty, tx);
        #pragma unroll
        for (int j = 0; j < NC; j++) {
            const bool live = ok[tx + 16 * j];
            #pragma unroll
            for (int i = 0; i < RT; i++) s[i][j] = live ? s[i][j] * a.scale : -INFINITY;
        }
        float c[RT];
        #pragma unroll
        for (int i = 0; i < RT; i++) {
            float x = s[i][0];
            #pragma unroll
            for (int j = 1; j < NC; j++) x = fmaxf(x, s[i][j]);
            const float n = fmaxf(m[i], row16_max(x)), u = n == -INFINITY ? 0.f : n;
            c[i] = expf(m[i] - u);
            m[i] = n;
            float t = 0.f;
            #pragma unroll
            for (int j = 0; j < NC; j++) {
                s[i][j] = expf(s[i][j] - u);
                t += s[i][j];
            }
            l[i] = fmaf(l[i], c[i], t);
        }
        #pragma unroll
        for (int j = 0; j < NC; j++) {
            float v[RT];
            #pragma unroll
            for (int i = 0; i < RT; i++) v[i] = s[i][j];
            put_rows<RT>(Ps, LM, tx + 16 * j, ty, v);
        }
        cp_wait<0>();
        __syncthreads();
        // as mm_outer_add, with the old maximum's factor
        float y[RT][ND];
        clear(y);
        mm_outer<RT, ND, BN>(y, Ps, LM, Vs, LD, ty, tx);
        #pragma unroll
        for (int i = 0; i < RT; i++)
            #pragma unroll
            for (int j = 0; j < ND; j++) o[i][j] = fmaf(o[i][j], c[i], y[i][j]);
    }
    cp_wait<0>();
    #pragma unroll
    for (int i = 0; i < RT; i++) {
        const float t = row16_sum(l[i]);
        const int r = r0 + row_of<RT>(ty, i);
        if (r >= a.rows) continue;
        const long row = ((long)at.seq * a.kv_heads + at.hk) * a.rows + r;
        const float inv = a.nsplit > 1 ? 1.f : t == 0.f ? 0.f : 1.f / t;
        float* p = a.nsplit > 1 ? a.part + (row * a.nsplit + at.part) * DH
                                : (float*)a.out + qrow(a, a.so, at.seq, at.hk, r);
        put_cols<ND>(p, tx, o[i], inv);
        if (tx == 0) {
            if (a.nsplit > 1) a.part_ml[row * a.nsplit + at.part] = make_float2(m[i], t);
            else if (a.lse) a.lse[row] = t == 0.f ? -INFINITY : m[i] + logf(t);
        }
    }
}

template <int DH, int RT>
__global__ void __launch_bounds__(128, DH == 32 ? 3 : 1) k_cross_dq_f32(const __grid_constant__ CrossArgs a) {
    constexpr int BM = RT * 8, LM = BM + 4, BN = F32<DH>::BN, LD = F32<DH>::LD, NC = BN / 16, ND = DH / 16;
    extern __shared__ __align__(16) float fs[];
    __shared__ uint8_t ok[BN];
    __shared__ float s_lse[BM], s_delta[BM];
    float* Qs = fs;                  // [BM][LD]
    float* Gs = Qs + BM * LD;        // [BM][LD]
    float* Ks = Gs + BM * LD;        // [BN][LD]
    float* Vs = Ks + BN * LD;        // [BN][LD]
    float* Ds = Vs + BN * LD;        // [BN][LM]
    const Where at = where(a);
    const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
    const int r0 = at.tile * BM, len = kept_len(a, at.seq);
    const int kbeg = min(at.part * a.split, len), kend = min(len, kbeg + a.split);
    const long row0 = ((long)at.seq * a.kv_heads + at.hk) * a.rows;
    stage_f32<DH, BM>(Qs, (const float*)a.q, [&](int r) { return q_ptr(a, a.q, a.sq, at, r0 + r, a.rows); });
    stage_f32<DH, BM>(Gs, (const float*)a.dout, [&](int r) { return q_ptr(a, a.dout, a.sdo, at, r0 + r, a.rows); });
    cp_commit();
    cp_wait<0>();
    __syncthreads();
    for (int r = threadIdx.x; r < BM; r += 128) {
        const bool in = r0 + r < a.rows;
        const float d = in ? delta_f32<DH>(a, at, r0 + r, Gs + r * LD) : 0.f;
        if (in && at.part == 0) a.delta[row0 + r0 + r] = d;
        s_lse[r] = lse_or_inf(a, row0 + r0 + r, in);
        s_delta[r] = d;
    }
    float dq[RT][ND];
    clear(dq);
    for (int k0 = kbeg; k0 < kend; k0 += BN) {
        const int key = k0 + threadIdx.x;
        const bool in = threadIdx.x < BN && key < kend && kept(a, at.seq, key, len);
        __syncthreads();
        if (threadIdx.x < BN) ok[threadIdx.x] = in;
        if (!__syncthreads_or(in)) continue;
        stage_f32<DH, BN>(Ks, (const float*)a.k, [&](int r) { return k_ptr(a.k, a.sk, at, k0 + r, ok[r]); });
        cp_commit();
        stage_f32<DH, BN>(Vs, (const float*)a.v, [&](int r) { return k_ptr(a.v, a.sv, at, k0 + r, ok[r]); });
        cp_commit();
        cp_wait<1>();
        __syncthreads();
        float s[RT][NC], p[RT][NC];
        mm_rows<RT, NC, DH>(s, Qs, Ks, ty, tx);
        cp_wait<0>();
        __syncthreads();
        mm_rows<RT, NC, DH>(p, Gs, Vs, ty, tx);
        #pragma unroll
        for (int j = 0; j < NC; j++) {
            const bool live = ok[tx + 16 * j];
            float v[RT];
            #pragma unroll
            for (int i = 0; i < RT; i++) {
                const int r = row_of<RT>(ty, i);
                const float e = live ? expf(fmaf(s[i][j], a.scale, -s_lse[r])) : 0.f;
                v[i] = e * (p[i][j] - s_delta[r]);
            }
            put_rows<RT>(Ds, LM, tx + 16 * j, ty, v);
        }
        __syncthreads();
        mm_outer_add<RT, ND, BN>(dq, Ds, LM, Ks, LD, ty, tx);
    }
    #pragma unroll
    for (int i = 0; i < RT; i++) {
        const int r = r0 + row_of<RT>(ty, i);
        if (r >= a.rows) continue;
        put_cols<ND>(a.nsplit > 1 ? a.part + ((row0 + r) * a.nsplit + at.part) * DH
                                  : (float*)a.dq + qrow(a, a.sdq, at.seq, at.hk, r), tx, dq[i], a.scale);
    }
}

// dk and dv of a key tile over the stacked rows (ROWS: at most 64 of them, all
// in one tile, and dq as well: each block then walks the key tiles and S is
// computed once, as in k_cross_bwd_rows; tiles of BQ = 16, 32 or 64 rows, the
// smallest that holds them: 24 rows of width 128 on 93 keys, 512 x 8 of them,
// 1066 us in 32 against 1998 in 64)
template <int DH, bool ROWS, int BQ>
__global__ void __launch_bounds__(128, DH == 32 ? 3 : 1) k_cross_dkv_f32(const __grid_constant__ CrossArgs a) {
    constexpr int RT = 8, BK = 64, LM = BK + 4, LQ = BQ + 4, LD = F32<DH>::LD;
    constexpr int NC = BQ / 16, ND = DH / 16, RQ = ROWS ? BQ / 8 : 1;
    extern __shared__ __align__(16) float fs[];
    __shared__ uint8_t ok[BK];
    __shared__ float s_lse[BQ], s_delta[BQ];
    float* Ks = fs;                  // [BK][LD]
    float* Vs = Ks + BK * LD;        // [BK][LD]
    float* Qs = Vs + BK * LD;        // [BQ][LD]
    float* Gs = Qs + BQ * LD;        // [BQ][LD]
    float* Ps = Gs + BQ * LD;        // [BQ][LM] P, then dS
    float* Ds = Ps + BQ * LM;        // ROWS: [BK][LQ] dS with the keys as rows, else [BQ][LM]
    const Where at = where(a);
    const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
    const int len = kept_len(a, at.seq);
    const long row0 = ((long)at.seq * a.kv_heads + at.hk) * a.rows;
    // ROWS: the key tiles of this part; else one key tile and this part's rows
    const int kfrom = ROWS ? at.part * a.split : at.tile * BK;
    const int kto = ROWS ? min(a.lk, kfrom + a.split) : min(a.lk, kfrom + BK);
    const int qbeg = ROWS ? 0 : min(at.part * a.split, a.rows), qend = ROWS ? a.rows : min(a.rows, qbeg + a.split);
    float dq[RQ][ROWS ? ND : 1];
    clear(dq);
    auto stage_rows = [&](int q0) {
        stage_f32<DH, BQ>(Qs, (const float*)a.q, [&](int r) { return q_ptr(a, a.q, a.sq, at, q0 + r, qend); });
        stage_f32<DH, BQ>(Gs, (const float*)a.dout, [&](int r) { return q_ptr(a, a.dout, a.sdo, at, q0 + r, qend); });
        cp_commit();
    };
    if (ROWS) {
        stage_rows(0);
        cp_wait<0>();
        __syncthreads();
        if (threadIdx.x < BQ) {
            const int r = threadIdx.x;
            s_lse[r] = lse_or_inf(a, row0 + r, r < a.rows);
            s_delta[r] = r < a.rows ? delta_f32<DH>(a, at, r, Gs + r * LD) : 0.f;
        }
    }
    for (int j0 = kfrom; j0 < kto; j0 += BK) {
        const bool in = threadIdx.x < BK && j0 + threadIdx.x < kto && kept(a, at.seq, j0 + threadIdx.x, len);
        __syncthreads();
        if (threadIdx.x < BK) ok[threadIdx.x] = in;
        const bool any = __syncthreads_or(in);
        float dk[RT][ND], dv[RT][ND];
        clear(dk);
        clear(dv);
        if (any) {
            stage_f32<DH, BK>(Ks, (const float*)a.k, [&](int r) { return k_ptr(a.k, a.sk, at, j0 + r, ok[r]); });
            stage_f32<DH, BK>(Vs, (const float*)a.v, [&](int r) { return k_ptr(a.v, a.sv, at, j0 + r, ok[r]); });
            cp_commit();
            for (int q0 = qbeg; q0 < qend; q0 += BQ) {
                if (!ROWS) {
                    __syncthreads();
                    stage_rows(q0);
                    if (threadIdx.x < BQ) {
                        const int r = q0 + threadIdx.x;
                        s_lse[threadIdx.x] = lse_or_inf(a, row0 + r, r < qend);
                        s_delta[threadIdx.x] = r < qend ? a.delta[row0 + r] : 0.f;
                    }
                }
                cp_wait<0>();
                __syncthreads();
                float s[RT][NC], p[RT][NC];
                mm_rows<RT, NC, DH>(s, Ks, Qs, ty, tx);
                mm_rows<RT, NC, DH>(p, Vs, Gs, ty, tx);
                #pragma unroll
                for (int j = 0; j < NC; j++) {
                    const int c = tx + 16 * j;
                    const float x = s_lse[c], d = s_delta[c];
                    float v[RT];
                    #pragma unroll
                    for (int i = 0; i < RT; i++) {
                        v[i] = ok[row_of<RT>(ty, i)] ? expf(fmaf(s[i][j], a.scale, -x)) : 0.f;
                        p[i][j] = v[i] * (p[i][j] - d);
                    }
                    put_rows<RT>(Ps, LM, c, ty, v);
                    #pragma unroll
                    for (int i = 0; i < RT; i++) v[i] = p[i][j];
                    if (ROWS) {
                        #pragma unroll
                        for (int i = 0; i < RT; i++) Ds[row_of<RT>(ty, i) * LQ + c] = v[i];
                    } else {
                        put_rows<RT>(Ds, LM, c, ty, v);
                    }
                }
                __syncthreads();
                if constexpr (ROWS) {                // one tile of rows: nothing to add to
                    mm_outer<RT, ND, BQ>(dv, Ps, LM, Gs, LD, ty, tx);
                    mm_outer_add<RQ, ND, BK>(dq, Ds, LQ, Ks, LD, ty, tx);
                    __syncthreads();
                    #pragma unroll
                    for (int j = 0; j < NC; j++) {
                        float v[RT];
                        #pragma unroll
                        for (int i = 0; i < RT; i++) v[i] = p[i][j];
                        put_rows<RT>(Ps, LM, tx + 16 * j, ty, v);
                    }
                    __syncthreads();
                    mm_outer<RT, ND, BQ>(dk, Ps, LM, Qs, LD, ty, tx);
                } else {
                    mm_outer_add<RT, ND, BQ>(dv, Ps, LM, Gs, LD, ty, tx);
                    mm_outer_add<RT, ND, BQ>(dk, Ds, LM, Qs, LD, ty, tx);
                }
            }
            cp_wait<0>();
        }
        #pragma unroll
        for (int i = 0; i < RT; i++) {
            const int j = j0 + row_of<RT>(ty, i);
            if (j >= kto) continue;
            if (!ok[j - j0]) {
                #pragma unroll
                for (int c = 0; c < ND; c++) dk[i][c] = dv[i][c] = 0.f;
            }
            const bool parts = !ROWS && a.nsplit > 1;
            const long part = ((((long)at.seq * a.kv_heads + at.hk) * a.lk + j) * a.nsplit + at.part) * DH;
            put_cols<ND>(parts ? a.part + part : (float*)a.dk + krow(a.sdk, at.seq, at.hk, j), tx, dk[i], a.scale);
            put_cols<ND>(parts ? a.part2 + part : (float*)a.dv + krow(a.sdv, at.seq, at.hk, j), tx, dv[i], 1.f);
        }
    }
    if constexpr (ROWS) {
        #pragma unroll
        for (int i = 0; i < RQ; i++) {
            const int r = row_of<RQ>(ty, i);
            if (r >= a.rows) continue;
            put_cols<ND>(a.nsplit > 1 ? a.part + ((row0 + r) * a.nsplit + at.part) * DH
                                      : (float*)a.dq + qrow(a, a.sdq, at.seq, at.hk, r), tx, dq[i], a.scale);
        }
    }
}

// ------------------------------------------------------------- host side
// A problem whose tiles leave processors idle is split along its other axis,
// at least 256 rows of it to a part: into about four blocks a processor, or
// (tcgen05: one block fills a processor) as many as run at once.
struct Split { int n, len; };
Split split_of(long tiles, int axis, bool tc = false) {
    Split s = {1, axis > 0 ? axis : 1};
    if (tiles >= (tc ? 75 : 148 * 2) || axis <= 256 || tiles == 0) return s;
    long want = tc ? 148 / tiles : (148 * 4 + tiles - 1) / tiles;
    want = std::min(want, (long)(axis + 255) / 256);
    s.len = (int)((((axis + want - 1) / want) + 63) / 64 * 64);
    s.n = (int)cdiv(axis, s.len);
    return s;
}
void set_tiles(CrossArgs& a, long tiles, const Split& s) {
    a.tiles = (int)tiles;
    a.nsplit = s.n;
    a.split = s.len;
    a.by_tiles = fast_div((unsigned)tiles);
    a.by_nsplit = fast_div(s.n);
}
// Which bf16 forwards run on tcgen05 (256-row blocks, one to a processor) and
// which on mma.sync (64-row blocks, several to a processor).  Measured, us,
// mma.sync / tcgen05: width 128: 4 x 4101 rows on 8191 keys 2260 / 508, 130 on
// 257 153 / 94, 1024 on 100 109 / 68, but 130 on 64 54 / 57; width 64: 4 x 4101
// on 8191 1410 / 450, 130 on 257 99 / 73; width 32, where a tile's products are
// short and half-empty tiles cost most: 512 on 512 54 / 43, 256 on 256 30 / 29,
// 130 on 257 47 / 63.
bool use_tc(const PtcgCross& c, long rows) {
    if (c.dtype != PTCG_BF16 || !gemm_tc_available()) return false;
    return c.dh == 32 ? rows >= 384 && c.lk >= 256 : rows > 64 && c.lk > 64;
}
// Parts of the single-token form: as many blocks as run at once (two of width
// 128 on a processor, four of the others), twice that where the problems alone
// are more than half of it.  Long caches of unequal length take even parts
// instead (cross.cuh), which only pays where the blocks have more to do than
// find their parts: from 4096 keys on (8 caches of up to 4100, 4 key heads of
// width 128: 24.6 us either way).
struct FwdPlan { bool few, tc; int bm; long tiles, blocks; Split sp; int want, most; long o_ml, bytes; };
FwdPlan fwd_plan(const PtcgCross& c) {
    FwdPlan p;
    const long rows = (long)c.heads / c.kv_heads * c.lq, probs = (long)c.nseq * c.kv_heads;
    p.few = rows <= 16;
    p.tc = use_tc(c, rows);
    p.bm = p.few ? 16 : c.dtype == PTCG_FP32 && rows <= 32 ? 32 : p.tc ? TC_ROWS : 64;
    p.tiles = (rows + p.bm - 1) / p.bm;
    p.sp = split_of(p.tiles * probs, c.lk, p.tc);
    p.want = 0;
    if (p.few && p.sp.n > 1) {
        long slots = 148 * (c.dh == 128 ? 2 : 4);
        if (2 * probs > slots) slots *= 2;
        p.sp.len = (int)((cdiv(c.lk, std::min(slots / probs, ((long)c.lk + 255) / 256)) + 63) / 64 * 64);
        p.sp.n = (int)cdiv(c.lk, p.sp.len);
        if (c.lk >= 4096) p.want = (int)(slots / c.kv_heads);
    }
    p.blocks = p.tiles * probs * p.sp.n;
    p.most = p.want ? std::max(std::min((int)cdiv(c.lk, EVEN_KEYS), p.want), p.sp.n) : p.sp.n;
    const long parts = p.most > 1 ? rows * probs * p.most : 0;
    p.o_ml = (4 * parts * c.dh + 255) / 256 * 256;
    p.bytes = p.most > 1 ? p.o_ml + 8 * parts : 0;
    return p;
}
struct BwdPlan { bool rows; long qtiles, qblocks, ktiles, kblocks; Split qs, ks; long o_part, o_part2, bytes; };
BwdPlan bwd_plan(const PtcgCross& c, bool tc) {
    BwdPlan p;
    const long group = c.heads / c.kv_heads, rows = group * c.lq, probs = (long)c.nseq * c.kv_heads;
    const long tile = tc ? TC_TILE : 64;
    p.rows = rows > 0 && rows <= 64;
    p.qtiles = (rows + tile - 1) / tile;
    p.ktiles = (c.lk + tile - 1) / tile;
    // dq: split over keys; dk and dv: over rows (tcgen05: in whole blocks of a head)
    p.qs = split_of(p.qtiles * probs, c.lk, tc);
    p.ks = split_of(p.ktiles * probs, (int)(tc ? group * cdiv(c.lq, TC_BLOCK) * TC_BLOCK : rows), tc);
    p.qblocks = p.qtiles * probs * p.qs.n;
    p.kblocks = p.ktiles * probs * p.ks.n;
    p.o_part = (4 * rows * probs + 255) / 256 * 256;       // delta first
    const long q = p.qs.n > 1 ? 4 * rows * probs * p.qs.n * c.dh : 0;
    const long k = p.ks.n > 1 ? 4 * (long)c.lk * probs * p.ks.n * c.dh : 0;
    p.o_part2 = p.o_part + k;
    p.bytes = p.o_part + std::max(q, 2 * k);               // one after the other
    return p;
}
// Which bf16 backwards run on tcgen05.  Measured, us, mma.sync / tcgen05 (rows
// x keys).  dq, width 128: 4 x 4101 x 8191 2690 / 757, 256 x 256 126 / 98,
// 130 x 257 194 / 175, but 130 x 70 101 / 140; width 64: 1354 / 549, but
// 130 x 257 100 / 118; width 32: 776 / 470, 512 x 512 61 / 59, but 256 x 256
// 37 / 45.  dk and dv, width 128: 3361 / 1068, 130 x 70 92 / 61; width 64:
// 1620 / 820, 130 x 257 134 / 136, 130 x 70 55 / 45; width 32: 922 / 794,
// 1024 x 100 40 / 33, but 512 x 512 68 / 69 and 256 x 256 40 / 46.
bool use_tc_dq(const PtcgCross& c) {
    if (c.dtype != PTCG_BF16 || !gemm_tc_available()) return false;
    const long rows = (long)c.heads / c.kv_heads * c.lq;
    return c.dh == 128 ? rows > 64 && c.lk >= 256
           : c.dh == 64 ? rows > 64 && c.lk >= 384 : rows >= 384 && c.lk >= 512;
}
// dk and dv take their row blocks per query head: not where short heads would
// leave them half empty
bool use_tc_dkv(const PtcgCross& c) {
    if (c.dtype != PTCG_BF16 || !gemm_tc_available()) return false;
    const long rows = (long)c.heads / c.kv_heads * c.lq;
    return 2L * cdiv(c.lq, TC_BLOCK) * TC_BLOCK <= 3L * c.lq && c.lk > 64 && rows > (c.dh == 32 ? 768 : 64);
}
long bwd_bytes(const PtcgCross& c) {
    const long b = bwd_plan(c, false).bytes;
    return use_tc_dq(c) || use_tc_dkv(c) ? std::max(b, bwd_plan(c, true).bytes) : b;
}

// kernels with more than 48 KB of shared memory, their static arrays (under
// 4 KB here) included, need the limit raised on the current device; a cheap
// call, repeated so that no state is kept
template <typename F>
cudaError_t smem_limit(F f, int bytes) {
    return bytes > 44 * 1024 ? cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes)
                             : cudaSuccess;
}

template <int DH, int WM, int WN, int NST>
cudaError_t launch_fwd(const CrossArgs& a, long blocks, cudaStream_t s) {
    int bytes = WM * 16 * DH * 2 + 2 * NST * 64 * DH * 2 + 256;
    if (WN > 1) bytes = std::max(bytes, (WN * 32 + WN * 16 * DH) * 4 + 256);
    const cudaError_t e = smem_limit(k_cross_fwd<DH, WM, WN, NST>, bytes);
    if (e != cudaSuccess) return e;
    ++g_ptcg_launches, k_cross_fwd<DH, WM, WN, NST><<<(unsigned)blocks, WM * WN * 32, bytes, s>>>(a);
    return cudaSuccess;
}
// dynamic shared memory of the kernels for short keys; they take problems whose
// keys leave room for two blocks on a processor
int short_fwd_bytes(int dh, int lk) { return (64 + 2 * ((lk + 15) & ~15)) * dh * 2 + 256; }
int short_bwd_bytes(int dh, int lk, int rows) {
    const int keys = (lk + 15) & ~15;
    return (2 * rows + 2 * keys) * dh * 2 + keys * rows * 2 + 256;
}
bool is_short(int lk, int bytes) { return lk <= SHORT_KEYS && bytes <= 108 * 1024; }
template <int DH>
cudaError_t launch_fwd_short(const CrossArgs& a, long blocks, cudaStream_t s) {
    const int bytes = short_fwd_bytes(DH, a.lk);
    const cudaError_t e = smem_limit(k_cross_fwd_short<DH>, bytes);
    if (e != cudaSuccess) return e;
    ++g_ptcg_launches, k_cross_fwd_short<DH><<<(unsigned)blocks, 128, bytes, s>>>(a);
    return cudaSuccess;
}
template <int DH, int RT>
cudaError_t launch_fwd_f32(const CrossArgs& a, long blocks, cudaStream_t s) {
    constexpr int BM = RT * 8, BN = F32<DH>::BN;
    const int bytes = 4 * ((BM + 2 * BN) * F32<DH>::LD + BN * (BM + 4));
    const cudaError_t e = smem_limit(k_cross_fwd_f32<DH, RT>, bytes);
    if (e != cudaSuccess) return e;
    ++g_ptcg_launches, k_cross_fwd_f32<DH, RT><<<(unsigned)blocks, 128, bytes, s>>>(a);
    return cudaSuccess;
}
template <int DH>
cudaError_t launch_dq(const CrossArgs& a, long blocks, cudaStream_t s) {
    constexpr int BN = DH == 128 ? 32 : 64;
    const int bytes = 4 * BN * DH * 2 + 2 * 64 * DH * 2 + 256;
    const cudaError_t e = smem_limit(k_cross_dq<DH>, bytes);
    if (e != cudaSuccess) return e;
    ++g_ptcg_launches, k_cross_dq<DH><<<(unsigned)blocks, 128, bytes, s>>>(a);
    return cudaSuccess;
}
template <int DH>
cudaError_t launch_dkv(const CrossArgs& a, long blocks, cudaStream_t s) {
    constexpr int BQ = DH == 128 ? 32 : 64;
    const int bytes = 2 * 64 * DH * 2 + 4 * BQ * DH * 2 + 256;
    const cudaError_t e = smem_limit(k_cross_dkv<DH>, bytes);
    if (e != cudaSuccess) return e;
    ++g_ptcg_launches, k_cross_dkv<DH><<<(unsigned)blocks, 128, bytes, s>>>(a);
    return cudaSuccess;
}
template <int DH, int RT>
cudaError_t launch_dq_f32(const CrossArgs& a, long blocks, cudaStream_t s) {
    constexpr int BM = RT * 8, BN = F32<DH>::BN;
    const int bytes = 4 * (2 * (BM + BN) * F32<DH>::LD + BN * (BM + 4));
    const cudaError_t e = smem_limit(k_cross_dq_f32<DH, RT>, bytes);
    if (e != cudaSuccess) return e;
    ++g_ptcg_launches, k_cross_dq_f32<DH, RT><<<(unsigned)blocks, 128, bytes, s>>>(a);
    return cudaSuccess;
}
template <int DH, bool ROWS, int BQ>
cudaError_t launch_dkv_f32(const CrossArgs& a, long blocks, cudaStream_t s) {
    const int bytes = 4 * (2 * (64 + BQ) * F32<DH>::LD + BQ * 68 + std::max(BQ * 68, 64 * (BQ + 4)));
    const cudaError_t e = smem_limit(k_cross_dkv_f32<DH, ROWS, BQ>, bytes);
    if (e != cudaSuccess) return e;
    ++g_ptcg_launches, k_cross_dkv_f32<DH, ROWS, BQ><<<(unsigned)blocks, 128, bytes, s>>>(a);
    return cudaSuccess;
}
template <int DH>
cudaError_t fwd_dh(CrossArgs a, const PtcgCross& c, const FwdPlan& p, cudaStream_t s) {
    cudaError_t e;
    bool taken = false;
    long blocks = p.blocks;
    if (p.want && a.kv_len) {
        a.want = p.want;
        a.nsplit = p.most;
        blocks = (long)p.want * c.kv_heads;
    }
    if (p.tc) {
        e = fwd_tc(DH, a, p.blocks, s, &taken);
        if (e != cudaSuccess) return e;
    }
    if (p.tc && !taken) {                          // the same parts, in 64-row tiles
        const long tiles = (a.rows + 63) / 64;
        set_tiles(a, tiles, p.sp);
        e = launch_fwd<DH, 4, 1, 2>(a, tiles * c.nseq * c.kv_heads * p.sp.n, s);
    } else if (!p.tc && c.dtype == PTCG_BF16)
        e = p.few ? launch_fwd<DH, 1, 4, 3>(a, blocks, s)
            : p.sp.n == 1 && is_short(c.lk, short_fwd_bytes(DH, c.lk)) ? launch_fwd_short<DH>(a, p.blocks, s)
            : launch_fwd<DH, 4, 1, 2>(a, p.blocks, s);
    else if (!p.tc)
        e = p.few ? launch_fwd_f32<DH, 2>(a, blocks, s)
            : p.bm == 32 ? launch_fwd_f32<DH, 4>(a, p.blocks, s) : launch_fwd_f32<DH, 8>(a, p.blocks, s);
    if (e != cudaSuccess || a.nsplit == 1) return e;
    const long nrows = (long)c.nseq * c.kv_heads * a.rows;
    ++g_ptcg_launches;
    if (c.dtype == PTCG_BF16) k_cross_join<bf16, DH><<<(unsigned)nrows, 128, 0, s>>>(a);
    else k_cross_join<float, DH><<<(unsigned)nrows, 128, 0, s>>>(a);
    return cudaSuccess;
}
template <int DH, int NR>
cudaError_t launch_bwd_rows(const CrossArgs& a, long blocks, cudaStream_t s) {
    const int whole = short_bwd_bytes(DH, a.lk, NR * 16);
    if (a.nsplit == 1 && is_short(a.lk, whole)) {
        const cudaError_t e = smem_limit(k_cross_bwd_short<DH, NR>, whole);
        if (e != cudaSuccess) return e;
        ++g_ptcg_launches, k_cross_bwd_short<DH, NR><<<(unsigned)blocks, 128, whole, s>>>(a);
        return cudaSuccess;
    }
    const int bytes = 2 * NR * 16 * DH * 2 + 4 * 64 * DH * 2 + 64 * NR * 16 * 2 + 256;
    const cudaError_t e = smem_limit(k_cross_bwd_rows<DH, NR>, bytes);
    if (e != cudaSuccess) return e;
    ++g_ptcg_launches, k_cross_bwd_rows<DH, NR><<<(unsigned)blocks, 128, bytes, s>>>(a);
    return cudaSuccess;
}
template <int DH>
void sum_parts(const CrossArgs& a, bool bf, long nrows, int keys, cudaStream_t s) {
    const unsigned grid = cdiv(nrows * (DH / 4), 256);
    ++g_ptcg_launches;
    if (bf) k_cross_sum<bf16, DH><<<grid, 256, 0, s>>>(a, nrows, keys);
    else k_cross_sum<float, DH><<<grid, 256, 0, s>>>(a, nrows, keys);
}
template <int DH>
cudaError_t bwd_dh(CrossArgs a, const PtcgCross& c, uint8_t* scratch, cudaStream_t s) {
    cudaError_t e = cudaSuccess;
    const bool bf = c.dtype == PTCG_BF16;
    const long probs = (long)c.nseq * c.kv_heads, nrows = probs * a.rows, nkeys = probs * a.lk;
    const BwdPlan plain = bwd_plan(c, false);
    auto parts = [&](const BwdPlan& p) {
        a.part = (float*)(scratch + p.o_part);
        a.part2 = (float*)(scratch + p.o_part2);
    };
    a.delta = (float*)scratch;
    parts(plain);
    if (plain.rows && plain.qblocks) {
        set_tiles(a, 1, plain.qs);
        e = !bf ? (a.rows <= 16 ? launch_dkv_f32<DH, true, 16>(a, plain.qblocks, s)
                   : a.rows <= 32 ? launch_dkv_f32<DH, true, 32>(a, plain.qblocks, s)
                                  : launch_dkv_f32<DH, true, 64>(a, plain.qblocks, s))
            : a.rows <= 16 ? launch_bwd_rows<DH, 1>(a, plain.qblocks, s)
            : a.rows <= 32 ? launch_bwd_rows<DH, 2>(a, plain.qblocks, s) : launch_bwd_rows<DH, 4>(a, plain.qblocks, s);
        if (e == cudaSuccess && a.nsplit > 1) sum_parts<DH>(a, bf, nrows, 0, s);
        return e;
    }
    const BwdPlan tc = bwd_plan(c, true);
    if (plain.qblocks) {
        bool taken = false;
        if (use_tc_dq(c)) {
            parts(tc);
            set_tiles(a, tc.qtiles, tc.qs);
            e = dq_tc(DH, a, tc.qblocks, s, &taken);
        }
        if (e == cudaSuccess && !taken) {
            parts(plain);
            set_tiles(a, plain.qtiles, plain.qs);
            e = bf ? launch_dq<DH>(a, plain.qblocks, s) : launch_dq_f32<DH, 8>(a, plain.qblocks, s);
        }
        if (e != cudaSuccess) return e;
        if (a.nsplit > 1) sum_parts<DH>(a, bf, nrows, 0, s);
    }
    if (plain.kblocks) {
        bool taken = false;
        if (use_tc_dkv(c)) {
            parts(tc);
            set_tiles(a, tc.ktiles, tc.ks);
            e = dkv_tc(DH, a, tc.kblocks, s, &taken);
        }
        if (e == cudaSuccess && !taken) {
            parts(plain);
            set_tiles(a, plain.ktiles, plain.ks);
            e = bf ? launch_dkv<DH>(a, plain.kblocks, s) : launch_dkv_f32<DH, false, F32<DH>::BN>(a, plain.kblocks, s);
        }
        if (e == cudaSuccess && a.nsplit > 1) sum_parts<DH>(a, bf, nkeys, 1, s);
    }
    return e;
}

bool heads_ok(const PtcgHeads& s, const void* p, int dtype) {
    const long sz = dt_size(dtype);
    return (uintptr_t)p % 16 == 0 && (s.seq * sz) % 16 == 0 && (s.row * sz) % 16 == 0 && (s.head * sz) % 16 == 0;
}
// a written tensor: no two of its rows may share elements along one axis
bool apart(const PtcgHeads& s, long nseq, long n, long nh, int dh) {
    if (nseq == 0 || n == 0 || nh == 0) return true;
    return (nseq <= 1 || s.seq >= dh) && (n <= 1 || s.row >= dh) && (nh <= 1 || s.head >= dh);
}
// 0, or an error code with its message set
int check(const PtcgCross* c) {
    OP_REQ(c, PTCG_EINVAL, "cross attention: null description");
    OP_REQ(dt_ok(c->dtype), PTCG_EINVAL, "cross attention: unknown dtype %d", c->dtype);
    OP_REQ(c->nseq >= 0 && c->lq >= 0 && c->lk >= 0 && c->heads > 0 && c->kv_heads > 0 &&
           c->heads % c->kv_heads == 0, PTCG_EINVAL,
           "cross attention: bad sizes (nseq %d, lq %d, lk %d, heads %d, kv_heads %d)", c->nseq, c->lq,
           c->lk, c->heads, c->kv_heads);
    OP_REQ(c->dh == 32 || c->dh == 64 || c->dh == 128, PTCG_EINVAL,
           "cross attention: head width %d is not 32, 64 or 128", c->dh);
    // the exponentials are of 2
    OP_REQ(c->scale > 0.f && c->scale * LOG2E < INFINITY, PTCG_EINVAL,
           "cross attention: scale must be positive and finite, scale * log2 e too");
    const long rows = (long)c->heads / c->kv_heads * c->lq;
    OP_REQ(rows <= (1L << 30) && c->lk <= (1 << 30), PTCG_EINVAL, "cross attention: more than 2^30 rows");
    return PTCG_OK;
}
CrossArgs args(const PtcgCross& c) {
    CrossArgs a = {};
    a.sq = c.q; a.sk = c.k; a.sv = c.v; a.so = c.out;
    a.sdo = c.dout; a.sdq = c.dq; a.sdk = c.dk; a.sdv = c.dv;
    a.nseq = c.nseq; a.lq = c.lq; a.lk = c.lk; a.heads = c.heads; a.kv_heads = c.kv_heads;
    a.group = c.heads / c.kv_heads;
    a.rows = a.group * c.lq;
    a.scale = c.scale;
    a.by_lq = fast_div(c.lq > 0 ? c.lq : 1);
    a.by_kv = fast_div(c.kv_heads);
    return a;
}

}  // namespace

extern "C" {

long ptcg_cross_attention_fwd_scratch(const PtcgCross* c) {
    return check(c) ? -1 : fwd_plan(*c).bytes;
}

int ptcg_cross_attention_fwd(const PtcgCross* c, const void* q, const void* k, const void* v,
                             const unsigned char* keep, const int* kv_len, void* out, float* lse,
                             void* scratch, long scratch_bytes, void* stream) {
    const int rc = check(c);
    if (rc) return rc;
    if (c->nseq == 0 || c->lq == 0) return PTCG_OK;
    OP_REQ(q && out && (c->lk == 0 || (k && v)), PTCG_EINVAL, "cross attention: null pointer");
    OP_REQ(heads_ok(c->q, q, c->dtype) && heads_ok(c->k, k, c->dtype) && heads_ok(c->v, v, c->dtype) &&
           heads_ok(c->out, out, c->dtype) && (uintptr_t)lse % 4 == 0 && (uintptr_t)kv_len % 4 == 0, PTCG_EINVAL,
           "cross attention: rows must start on 16-byte boundaries");
    OP_REQ(apart(c->out, c->nseq, c->lq, c->heads, c->dh), PTCG_EINVAL, "cross attention: out rows overlap");
    const FwdPlan p = fwd_plan(*c);
    OP_REQ(p.bytes == 0 || ((uintptr_t)scratch % 16 == 0 && scratch && scratch_bytes >= p.bytes), PTCG_ERANGE,
           "cross attention: scratch of %ld bytes, %ld needed (16-byte aligned)", scratch ? scratch_bytes : 0L, p.bytes);
    OP_REQ(p.blocks <= 0x7fffffffL, PTCG_EINVAL, "cross attention: too many tiles");
    CrossArgs a = args(*c);
    a.q = q; a.k = k; a.v = v; a.keep = keep; a.kv_len = kv_len; a.out = out; a.lse = lse;
    a.part = (float*)scratch;
    a.part_ml = (float2*)((uint8_t*)scratch + p.o_ml);
    set_tiles(a, p.tiles, p.sp);
    cudaStream_t s = (cudaStream_t)stream;
    OP_CK(c->dh == 32 ? fwd_dh<32>(a, *c, p, s) : c->dh == 64 ? fwd_dh<64>(a, *c, p, s) : fwd_dh<128>(a, *c, p, s));
    OP_CKL();
    return PTCG_OK;
}

long ptcg_cross_attention_bwd_scratch(const PtcgCross* c) {
    return check(c) ? -1 : bwd_bytes(*c);
}

int ptcg_cross_attention_bwd(const PtcgCross* c, const void* q, const void* k, const void* v,
                             const unsigned char* keep, const int* kv_len, const void* out,
                             const float* lse, const void* dout, void* dq, void* dk, void* dv,
                             void* scratch, long scratch_bytes, void* stream) {
    const int rc = check(c);
    if (rc) return rc;
    if (c->nseq == 0 || (c->lq == 0 && c->lk == 0)) return PTCG_OK;
    OP_REQ((c->lq == 0 || (q && out && lse && dout && dq)) && (c->lk == 0 || (k && v && dk && dv)),
           PTCG_EINVAL, "cross attention gradient: null pointer");
    OP_REQ(heads_ok(c->q, q, c->dtype) && heads_ok(c->k, k, c->dtype) && heads_ok(c->v, v, c->dtype) &&
           heads_ok(c->out, out, c->dtype) && heads_ok(c->dout, dout, c->dtype) &&
           heads_ok(c->dq, dq, c->dtype) && heads_ok(c->dk, dk, c->dtype) && heads_ok(c->dv, dv, c->dtype) &&
           (uintptr_t)lse % 4 == 0 && (uintptr_t)kv_len % 4 == 0, PTCG_EINVAL,
           "cross attention gradient: rows must start on 16-byte boundaries");
    OP_REQ(apart(c->dq, c->nseq, c->lq, c->heads, c->dh) && apart(c->dk, c->nseq, c->lk, c->kv_heads, c->dh) &&
           apart(c->dv, c->nseq, c->lk, c->kv_heads, c->dh), PTCG_EINVAL,
           "cross attention gradient: rows of a gradient overlap");
    const BwdPlan p = bwd_plan(*c, false);
    const long need = bwd_bytes(*c);
    OP_REQ(need == 0 || ((uintptr_t)scratch % 16 == 0 && scratch && scratch_bytes >= need), PTCG_ERANGE,
           "cross attention gradient: scratch of %ld bytes, %ld needed (16-byte aligned)",
           scratch ? scratch_bytes : 0L, need);
    OP_REQ(p.qblocks <= 0x7fffffffL && p.kblocks <= 0x7fffffffL, PTCG_EINVAL, "cross attention gradient: too many tiles");
    CrossArgs a = args(*c);
    a.q = q; a.k = k; a.v = v; a.keep = keep; a.kv_len = kv_len; a.o = out; a.lse = (float*)lse;
    a.dout = dout; a.dq = dq; a.dk = dk; a.dv = dv;
    uint8_t* base = (uint8_t*)scratch;
    cudaStream_t s = (cudaStream_t)stream;
    OP_CK(c->dh == 32 ? bwd_dh<32>(a, *c, base, s) : c->dh == 64 ? bwd_dh<64>(a, *c, base, s) : bwd_dh<128>(a, *c, base, s));
    OP_CKL();
    return PTCG_OK;
}

}  // extern "C"
