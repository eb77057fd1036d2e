// Layer norm over rows, its backward pass and the reduction of the weight
// gradients, for any row width up to PTCG_LN_MAX_WIDTH.
//   forward   mu = mean x, r = (mean (x - mu)^2 + eps)^(-1/2),
//             h = (x - mu) r, y = h gamma + beta
//   backward  g = dy gamma, dx = r (g - mean g - h mean(g h)) (+ dres),
//             dgamma = sum over rows of dy h, dbeta = sum over rows of dy
// (torch nn.LayerNorm; the model's own norms, ptcg/rl/model.py:70-91, run
// kernels tied to its row layouts.)  The statistics are two passes over the
// row in registers, so no cancellation between sums of squares; everything
// is fp32 until the one rounding to the output's type.  An fp32 mean is off by
// some of its last places, which in a row far from 0 are not small beside its
// deviations or sqrt(eps) (at 12345 one of them moves a constant row's y by 0.3
// gamma) or, squared, lie past its range.  Such rows take the mean of the
// deviations as well, a third sum, and are normed about both, their variance
// too; summed beside the squares in every row it would cost 3 to 20 % of the
// time (50000 x 2048, fp32 to bf16: 117 us without it, 137 so, 124 by need, or 156
// where every row lies 100 deviations from 0; 2.1 M x 256 508 and 518).
#include <algorithm>
#include <initializer_list>

#include "vec.cuh"

namespace {

constexpr int MAXW = PTCG_LN_MAX_WIDTH;
// one warp holds rows of up to 1024 columns, NV pieces of V columns per lane;
// wider rows are shared by the warps of a block, 256 columns each, so that the
// backward's registers per column still fit 1024 threads; blocks of up to 640
// have registers, 96 each, for two rows at once (forward) or the next row's
// loads (backward): 47 + 90 us at 8192 x 5120 in bf16 against 58 + 118 under the
// bound of 1024.  A bound of 672 threads, which would leave 96 registers too, takes
// 57 + 111 there and no less at 5376
constexpr int WARP_COLS = 1024, SHARED_COLS = 256, MID_THREADS = 640, MAX_THREADS = MAXW / SHARED_COLS * 32;

// Bound: HBM (2.1 M rows of 256, fp32 to bf16: forward 502 us, 6.5 TB/s; backward
// with the residual's gradient 1146 us, 6.6 TB/s); wider rows are bound by the
// latency of a row's loads and barriers (fp32 to bf16, 50000 x 1024: 54 us, 5.7
// TB/s, and 101, 5.1; 50000 x 2048: 123, 5.0, and 237, 4.3; in bf16, 4099 x 5001:
// 31, 2.7, and 57, 2.2; 8192 x 8192: 78, 3.5, and 133, 3.0).  A row
// belongs to one warp (width <= 1024, eight rows to a block) or to the W warps
// of a block (MULTI).  Lane l of warp w owns pieces w * 32 * NV + l, + 32, .. so
// that a warp's accesses are contiguous.
template <int V, int NV>
PTCG_DEV int piece_at(int w, int lane, int k) { return (w * NV + k) * 32 + lane; }

// sums of N values over the row's warps; `slot` alternates so that one barrier
// per reduction is enough
template <int MULTI, int N>
PTCG_DEV void row_sums(float (&v)[N], float (*red)[N][32], int slot, int w, int lane, int W) {
    #pragma unroll
    for (int i = 0; i < N; i++) v[i] = warp_sum(v[i]);
    if (!MULTI) return;
    if (lane == 0) {
        #pragma unroll
        for (int i = 0; i < N; i++) red[slot][i][w] = v[i];
    }
    __syncthreads();
    #pragma unroll
    for (int i = 0; i < N; i++) v[i] = warp_sum(lane < W ? red[slot][i][lane] : 0.f);
}

// Columns of a row: `body` pieces of V from `head` on, and up to 2 (V - 1) single
// ones at its ends, one each to the first lanes of the row's first warp.  Rows
// that start on V-element boundaries have none of those; other rows are taken
// PHASED: every row of a warp (or block) starts at the same phase, so that its
// pieces are aligned and its lanes keep their columns (row steps are multiples
// of V for that).
template <int V, bool PHASED> struct Columns {
    int head, body, edge;                           // edge: this lane's single column, or -1
    PTCG_DEV Columns(int phase, int width, bool first_warp, int lane) {
        head = PHASED ? (V - phase) & (V - 1) : 0;
        if (PHASED && head > width) head = width;
        body = (width - head) / V;
        const int tail = width - head - body * V;
        edge = !PHASED || !first_warp ? -1 : lane < head ? lane : lane < head + tail ? width - tail + lane - head : -1;
    }
    PTCG_DEV bool has(int p) const { return p < body; }
    PTCG_DEV int at(int p) const { return head + p * V; }
};

template <typename TX, typename TY, int V, int NV, int MULTI, bool PHASED>
__global__ void __launch_bounds__(MULTI ? MULTI : 256) k_layer_norm_fwd(
        TY* y, long ldy, float* mean, float* rstd, const TX* x, long ldx,
        const float* __restrict__ gamma, const float* __restrict__ beta, long rows, int width,
        float eps) {
    constexpr int R = MULTI == MID_THREADS ? 2 : 1;
    __shared__ float red[4][R][32], far_red[2][R][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = blockDim.x >> 5;
    const int w = MULTI ? warp : 0;
    const float inv = 1.f / (float)width;
    const long step = MULTI ? gridDim.x : (long)gridDim.x * W;
    long r0 = MULTI ? blockIdx.x : (long)blockIdx.x * W + warp;
    const int phase = PHASED ? (int)(((uintptr_t)x / sizeof(TX) + r0 * ldx) & (V - 1)) : 0;
    const Columns<V, PHASED> cols(phase, width, w == 0, lane);
    const bool edge = PHASED && cols.edge >= 0;
    float gm[NV][V], bt[NV][V];
    #pragma unroll
    for (int k = 0; k < NV; k++) {
        const int p = piece_at<V, NV>(w, lane, k);
        #pragma unroll
        for (int e = 0; e < V; e++) {
            gm[k][e] = gamma && cols.has(p) ? gamma[cols.at(p) + e] : 1.f;
            bt[k][e] = beta && cols.has(p) ? beta[cols.at(p) + e] : 0.f;
        }
    }
    const float ge = edge && gamma ? gamma[cols.edge] : 1.f, be = edge && beta ? beta[cols.edge] : 0.f;
    // R rows at a time, the next ones' loads in flight while these are reduced,
    // where the registers allow it
    constexpr bool AHEAD = NV * V <= 8;
    Raw<TX, V> row[R][NV];
    Raw<TX, 1> single[R];
    auto fetch = [&](long i0) {
        #pragma unroll
        for (int j = 0; j < R; j++) {
            const long i = i0 + j * step;
            const TX* xr = x + i * ldx;
            #pragma unroll
            for (int k = 0; k < NV; k++) {
                const int p = piece_at<V, NV>(w, lane, k);
                row[j][k].zero();
                if (i < rows && cols.has(p)) row[j][k].ld(xr + cols.at(p));
            }
            if (PHASED) {
                single[j].zero();
                if (i < rows && edge) single[j].ld(xr + cols.edge);
            }
        }
    };
    int slot = 0;
    if (AHEAD) fetch(r0);
    for (; r0 < rows; r0 += R * step) {
        float v[R][NV][V], s[R], mu[R], dm[R], se[R][1];
        if (!AHEAD) fetch(r0);
        #pragma unroll
        for (int j = 0; j < R; j++) {
            #pragma unroll
            for (int k = 0; k < NV; k++) row[j][k].get(v[j][k]);
            se[j][0] = 0.f;
            if (PHASED) single[j].get(se[j]);
            s[j] = se[j][0];
        }
        if (AHEAD) fetch(r0 + R * step);
        #pragma unroll
        for (int j = 0; j < R; j++)
            #pragma unroll
            for (int k = 0; k < NV; k++)
                #pragma unroll
                for (int e = 0; e < V; e++) s[j] += v[j][k][e];
        row_sums<MULTI>(s, red, slot, w, lane, W);
        #pragma unroll
        for (int j = 0; j < R; j++) {
            // rounded here, so that x - mu is the same whether or not mean is stored
            mu[j] = __fmul_rn(s[j], inv);
            s[j] = 0.f;
            #pragma unroll
            for (int k = 0; k < NV; k++) {
                const float in = cols.has(piece_at<V, NV>(w, lane, k)) ? 1.f : 0.f;
                #pragma unroll
                for (int e = 0; e < V; e++) {
                    const float d = (v[j][k][e] - mu[j]) * in;
                    s[j] = fmaf(d, d, s[j]);
                }
            }
            if (edge) s[j] = fmaf(se[j][0] - mu[j], se[j][0] - mu[j], s[j]);
        }
        row_sums<MULTI>(s, red, slot + 1, w, lane, W);
        slot ^= 2;
        // mean squares of up to 16 times the variance (+ eps): the mean's last
        // places are below those of h itself.  The same answer in all warps of a row
        bool far = false;
        #pragma unroll
        for (int j = 0; j < R; j++) {
            dm[j] = 0.f;
            const float t = fmaf(s[j], inv, eps);
            far = far || mu[j] * mu[j] > 16.f * t || t == INFINITY;
        }
        if (__builtin_expect(far, 0)) {
            float d[R];
            #pragma unroll
            for (int j = 0; j < R; j++) {
                d[j] = edge ? se[j][0] - mu[j] : 0.f;
                #pragma unroll
                for (int k = 0; k < NV; k++) {
                    const bool in = cols.has(piece_at<V, NV>(w, lane, k));
                    #pragma unroll
                    for (int e = 0; e < V; e++) d[j] += in ? v[j][k][e] - mu[j] : 0.f;
                }
            }
            row_sums<MULTI>(d, far_red, 0, w, lane, W);
            // sum (d - dm)^2 = sum d^2 - dm sum d, or summed again where little is
            // left of it or it was past fp32's range
            bool again = false;
            #pragma unroll
            for (int j = 0; j < R; j++) {
                // divided, so that equal deviations (a constant row) leave nothing
                dm[j] = d[j] / (float)width;
                const float left = fmaf(-d[j], dm[j], s[j]);
                again = again || !(left >= 0.25f * s[j]) || s[j] == INFINITY;
                s[j] = left;
            }
            if (again) {
                #pragma unroll
                for (int j = 0; j < R; j++) {
                    s[j] = edge ? se[j][0] - mu[j] - dm[j] : 0.f;
                    s[j] *= s[j];
                    #pragma unroll
                    for (int k = 0; k < NV; k++) {
                        const bool in = cols.has(piece_at<V, NV>(w, lane, k));
                        #pragma unroll
                        for (int e = 0; e < V; e++) {
                            const float x = in ? v[j][k][e] - mu[j] - dm[j] : 0.f;
                            s[j] = fmaf(x, x, s[j]);
                        }
                    }
                }
                row_sums<MULTI>(s, far_red, 1, w, lane, W);
            }
        }
        #pragma unroll
        for (int j = 0; j < R; j++) {
            const long r = r0 + j * step;
            if (j && r >= rows) break;
            const float rs = rsqrtf(fmaf(s[j], inv, eps));
            if (lane == 0 && w == 0) {
                if (mean) mean[r] = mu[j] + dm[j];
                if (rstd) rstd[r] = rs;
            }
            #pragma unroll
            for (int k = 0; k < NV; k++) {
                #pragma unroll
                for (int e = 0; e < V; e++) v[j][k][e] = fmaf((v[j][k][e] - mu[j] - dm[j]) * rs, gm[k][e], bt[k][e]);
                const int p = piece_at<V, NV>(w, lane, k);
                if (cols.has(p)) VecIO<TY, V>::st(y + r * ldy + cols.at(p), v[j][k]);
            }
            if (edge) y[r * ldy + cols.edge] = from_f<TY>(fmaf((se[j][0] - mu[j] - dm[j]) * rs, ge, be));
        }
    }
}

// Backward: the same ownership, each lane keeping the weight-gradient sums of
// its columns in registers over all its rows.  They leave once per block, in
// warp order through shared memory, as one partial row of dgamma and dbeta;
// k_layer_norm_wgrad adds the blocks' partials in a fixed order.  No atomics,
// so equal inputs give equal bits.
template <typename TX, typename TY, int V, int NV, int MULTI, bool PHASED>
__global__ void __launch_bounds__(MULTI ? MULTI : 256) k_layer_norm_bwd(
        TX* dx, long lddx, const TY* dy, long lddy, const TX* x, long ldx,
        const TX* dres, long lddres, const float* __restrict__ gamma,
        const float* __restrict__ mean, const float* __restrict__ rstd, long rows, int width,
        float* __restrict__ partial) {
    __shared__ float red[2][2][32];
    extern __shared__ float wsum[];                 // [2][width] of a one-warp-per-row block
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = blockDim.x >> 5;
    const int w = MULTI ? warp : 0;
    const float inv = 1.f / (float)width;
    const long step = MULTI ? gridDim.x : (long)gridDim.x * W;
    long r = MULTI ? blockIdx.x : (long)blockIdx.x * W + warp;
    const int phase = PHASED ? (int)(((uintptr_t)x / sizeof(TX) + r * ldx) & (V - 1)) : 0;
    const Columns<V, PHASED> cols(phase, width, w == 0, lane);
    const bool edge = PHASED && cols.edge >= 0;
    float gm[NV][V], ag[NV][V], ab[NV][V];
    #pragma unroll
    for (int k = 0; k < NV; k++) {
        const int p = piece_at<V, NV>(w, lane, k);
        #pragma unroll
        for (int e = 0; e < V; e++) {
            gm[k][e] = gamma && cols.has(p) ? gamma[cols.at(p) + e] : 1.f;
            ag[k][e] = ab[k][e] = 0.f;
        }
    }
    const float ge = edge && gamma ? gamma[cols.edge] : 1.f;
    float age = 0.f, abe = 0.f;
    int slot = 0;
    // as in the forward, a row at a time
    constexpr bool AHEAD = MULTI != MAX_THREADS && NV * V <= 8;
    struct Row { Raw<TX, V> x[NV], r[NV]; Raw<TY, V> g[NV]; Raw<TX, 1> xe, re; Raw<TY, 1> ge; float mu, rs; } row;
    auto fetch = [&](long i) {
        #pragma unroll
        for (int k = 0; k < NV; k++) {
            const int p = piece_at<V, NV>(w, lane, k);
            row.x[k].zero(); row.g[k].zero(); row.r[k].zero();
            if (i < rows && cols.has(p)) {
                row.x[k].ld(x + i * ldx + cols.at(p));
                row.g[k].ld(dy + i * lddy + cols.at(p));
                if (dres) row.r[k].ld(dres + i * lddres + cols.at(p));
            }
        }
        if (PHASED) {
            row.xe.zero(); row.ge.zero(); row.re.zero();
            if (i < rows && edge) {
                row.xe.ld(x + i * ldx + cols.edge);
                row.ge.ld(dy + i * lddy + cols.edge);
                if (dres) row.re.ld(dres + i * lddres + cols.edge);
            }
        }
        row.mu = i < rows ? mean[i] : 0.f;
        row.rs = i < rows ? rstd[i] : 0.f;
    };
    if (AHEAD) fetch(r);
    for (; r < rows; r += step) {
        float h[NV][V], g[NV][V], d[NV][V], s[2] = {0.f, 0.f};
        if (!AHEAD) fetch(r);
        const float mu = row.mu, rs = row.rs;
        #pragma unroll
        for (int k = 0; k < NV; k++) {
            row.x[k].get(h[k]);
            row.g[k].get(g[k]);
            row.r[k].get(d[k]);
        }
        float xe[1] = {0.f}, gy[1] = {0.f}, re[1] = {0.f};
        if (PHASED) {
            row.xe.get(xe);
            row.ge.get(gy);
            row.re.get(re);
        }
        if (AHEAD) fetch(r + step);
        // past the row g is 0, but mu rs need not be finite: no h there in the sums
        if (PHASED) {                               // 0 gradient where there is no edge column
            xe[0] = (xe[0] - mu) * (edge ? rs : 0.f);
            age = fmaf(gy[0], xe[0], age);
            abe += gy[0];
            gy[0] *= ge;
            s[0] = gy[0];
            s[1] = gy[0] * xe[0];
        }
        #pragma unroll
        for (int k = 0; k < NV; k++) {
            #pragma unroll
            for (int e = 0; e < V; e++) {
                const float hh = (h[k][e] - mu) * rs;
                ag[k][e] = fmaf(g[k][e], hh, ag[k][e]);
                ab[k][e] += g[k][e];
                g[k][e] *= gm[k][e];
                h[k][e] = hh;
                s[0] += g[k][e];
                s[1] = cols.has(piece_at<V, NV>(w, lane, k)) ? fmaf(g[k][e], hh, s[1]) : s[1];
            }
        }
        row_sums<MULTI>(s, red, slot, w, lane, W);
        slot ^= 1;
        const float m1 = __fmul_rn(s[0], inv), m2 = __fmul_rn(s[1], inv);
        #pragma unroll
        for (int k = 0; k < NV; k++) {
            #pragma unroll
            for (int e = 0; e < V; e++) {
                const float t = (g[k][e] - m1 - h[k][e] * m2) * rs;
                h[k][e] = dres ? t + d[k][e] : t;
            }
            const int p = piece_at<V, NV>(w, lane, k);
            if (cols.has(p)) VecIO<TX, V>::st(dx + r * lddx + cols.at(p), h[k]);
        }
        if (edge) {
            const float t = (gy[0] - m1 - xe[0] * m2) * rs;
            dx[r * lddx + cols.edge] = from_f<TX>(dres ? t + re[0] : t);
        }
    }
    if (!partial) return;
    float* out = partial + (long)blockIdx.x * 2 * width;
    if constexpr (MULTI) {
        #pragma unroll
        for (int k = 0; k < NV; k++) {
            const int p = piece_at<V, NV>(w, lane, k);
            if (!cols.has(p)) continue;
            #pragma unroll
            for (int e = 0; e < V; e++) {
                out[cols.at(p) + e] = ag[k][e];
                out[width + cols.at(p) + e] = ab[k][e];
            }
        }
        if (edge) {
            out[cols.edge] = age;
            out[width + cols.edge] = abe;
        }
    } else {
        auto add = [&](int c, float g, float b, bool first) {
            wsum[c] = first ? g : wsum[c] + g;
            wsum[width + c] = first ? b : wsum[width + c] + b;
        };
        for (int t = 0; t < W; t++) {
            if (warp == t) {
                #pragma unroll
                for (int k = 0; k < NV; k++) {
                    const int p = piece_at<V, NV>(0, lane, k);
                    if (!cols.has(p)) continue;
                    #pragma unroll
                    for (int e = 0; e < V; e++) add(cols.at(p) + e, ag[k][e], ab[k][e], t == 0);
                }
                if (edge) add(cols.edge, age, abe, t == 0);
            }
            __syncthreads();
        }
        for (int i = threadIdx.x; i < 2 * width; i += blockDim.x) out[i] = wsum[i];
    }
}

// out[c] (+)= sum over the blocks of partial[block][c], c over dgamma then
// dbeta: 32 columns a block, 8 threads over the rows of each, joined in order
__global__ void __launch_bounds__(256) k_layer_norm_wgrad(
        float* dgamma, float* dbeta, const float* __restrict__ partial, int nparts, int width,
        int accumulate) {
    __shared__ float part[8][33];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const long c = (long)blockIdx.x * 32 + tx;
    float s = 0.f;
    if (c < 2L * width) {
        #pragma unroll 8
        for (int j = ty; j < nparts; j += 8) s += partial[(long)j * 2 * width + c];
    }
    part[ty][tx] = s;
    __syncthreads();
    if (ty == 0 && c < 2L * width) {
        #pragma unroll
        for (int k = 1; k < 8; k++) s += part[k][tx];
        float* out = c < width ? dgamma + c : dbeta + (c - width);
        *out = accumulate ? *out + s : s;
    }
}

// The variant of a row width: V-column pieces, NV of them per lane, W warps a
// row (0: one warp a row, eight rows a block).  Rows that start on 4-element
// boundaries and a width of fours take them whole, other rows PHASED where all
// tensors' rows start at the same phase (4099 x 5001 fp32 to bf16: 39 + 64 us
// forward and backward against 43 + 82 with single elements, in bf16 31 + 71
// against 43 + 72; 50000 x 634 in fp32: 78 + 121 against 90 + 113), the rest
// single elements.
enum { SINGLE = 0, WHOLE = 1, PHASED4 = 2 };
struct Cfg { int mode, NV, W; };
Cfg cfg_of(int width, int mode) {
    Cfg c;
    c.mode = mode;
    const int V = mode == SINGLE ? 1 : 4, w = width;
    c.W = 0;
    if (w > WARP_COLS) {
        c.NV = SHARED_COLS / (32 * V);
        c.W = (int)cdiv(w, SHARED_COLS);
        return c;
    }
    c.NV = 1;
    while (c.NV * 32 * V < w) c.NV *= 2;
    if (V == 1) c.NV = c.NV <= 8 ? 8 : 32;
    return c;
}
// how the rows of some tensors (up to four; null: none) can be taken
struct Rows { const void* p; int dtype; long ld; };
int mode_of(int width, std::initializer_list<Rows> all) {
    bool whole = width % 4 == 0, same = true;
    long start = -1, pitch = -1;
    for (const Rows& t : all) {
        if (!t.p) continue;
        const long s = (long)((uintptr_t)t.p / dt_size(t.dtype) % 4), l = t.ld % 4;
        whole = whole && s == 0 && l == 0;
        if (start < 0) { start = s; pitch = l; }
        same = same && s == start && l == pitch;
    }
    return whole ? WHOLE : same ? PHASED4 : SINGLE;
}
// blocks of W warps that a processor's registers hold: each then takes its
// share of the rows in one go (twice as many blocks, fp32 to bf16: 41 + 70 us
// forward and backward at 4099 x 5001 instead of 39 + 64, 133 + 280 at 50000 x 2048
// instead of 123 + 237)
int resident(int W) { return std::max(MID_THREADS / 32 / W, 1); }
// blocks of the backward pass: as many as the registers of a processor hold, some
// 128 a thread up to 512 columns and 250 above (a multiple of 4, as 148 is, for
// the phases), at most one per row group, so that each leaves one partial row of
// the weight gradients.  1 / 2 / 4 blocks a processor, us: 2.1 M x 256, fp32 to
// bf16, 1413 / 969 / 978; 100000 x 512 129 / 100 / 111; 50000 x 634 113 / 125 / 145; 50000
// x 1024 113 / 129 / 158
int bwd_blocks(long rows, int width) {
    const long units = width > WARP_COLS ? rows : (rows + 7) / 8;
    const long most = 148L * (width > WARP_COLS ? resident((int)cdiv(width, SHARED_COLS)) : width > 512 ? 1 : 2);
    return (int)(units < most ? units : most);
}

template <typename TX, typename TY, int V, int NV, int MULTI, bool PH>
void fwd(void* y, long ldy, float* mean, float* rstd, const void* x, long ldx, const float* gamma,
         const float* beta, long rows, int width, float eps, int W, cudaStream_t s) {
    const long units = MULTI ? rows : (rows + 7) / 8;
    const long most = 148L * (MULTI ? resident(W) : 8);
    ++g_ptcg_launches;
    k_layer_norm_fwd<TX, TY, V, NV, MULTI, PH><<<(unsigned)(units < most ? units : most), MULTI ? W * 32 : 256, 0, s>>>(
        (TY*)y, ldy, mean, rstd, (const TX*)x, ldx, gamma, beta, rows, width, eps);
}
// LN(V, NV, MULTI, PHASED) of a configuration; MULTI: the most threads of a
// block whose warps share rows (a bound that leaves each its registers), 0: a
// warp takes rows alone
#define LN_WIDE(c, V, NV, PH) do { \
    if ((c).W * 32 <= MID_THREADS) LN(V, NV, MID_THREADS, PH); else LN(V, NV, MAX_THREADS, PH); } while (0)
#define LN_BY_CFG(c) do { \
    if ((c).mode == SINGLE) { \
        if ((c).W) LN(1, 8, MAX_THREADS, false); else if ((c).NV == 8) LN(1, 8, 0, false); else LN(1, 32, 0, false); \
    } else if ((c).mode == WHOLE) { \
        if ((c).W) LN_WIDE(c, 4, 2, false); else if ((c).NV == 1) LN(4, 1, 0, false); \
        else if ((c).NV == 2) LN(4, 2, 0, false); else if ((c).NV == 4) LN(4, 4, 0, false); \
        else LN(4, 8, 0, false); \
    } else { \
        if ((c).W) LN_WIDE(c, 4, 2, true); else if ((c).NV == 1) LN(4, 1, 0, true); \
        else if ((c).NV == 2) LN(4, 2, 0, true); else if ((c).NV == 4) LN(4, 4, 0, true); \
        else LN(4, 8, 0, true); \
    } } while (0)
template <typename TX, typename TY>
void fwd(const Cfg& c, void* y, long ldy, float* mean, float* rstd, const void* x, long ldx,
         const float* gamma, const float* beta, long rows, int width, float eps, cudaStream_t s) {
    #define LN(V, NV, M, PH) fwd<TX, TY, V, NV, M, PH>(y, ldy, mean, rstd, x, ldx, gamma, beta, rows, width, eps, c.W, s)
    LN_BY_CFG(c);
    #undef LN
}

struct BwdArgs {
    void* dx; long lddx; const void* dy; long lddy; const void* x; long ldx;
    const void* dres; long lddres; const float* gamma; const float* mean; const float* rstd;
    long rows; int width; float* partial;
};
template <typename TX, typename TY, int V, int NV, int MULTI, bool PH>
void bwd(const BwdArgs& a, int blocks, int W, cudaStream_t s) {
    ++g_ptcg_launches;
    k_layer_norm_bwd<TX, TY, V, NV, MULTI, PH><<<blocks, MULTI ? W * 32 : 256, MULTI ? 0 : 8 * a.width, s>>>(
        (TX*)a.dx, a.lddx, (const TY*)a.dy, a.lddy, (const TX*)a.x, a.ldx, (const TX*)a.dres,
        a.lddres, a.gamma, a.mean, a.rstd, a.rows, a.width, a.partial);
}
template <typename TX, typename TY>
void bwd(const Cfg& c, const BwdArgs& a, int blocks, cudaStream_t s) {
    #define LN(V, NV, M, PH) bwd<TX, TY, V, NV, M, PH>(a, blocks, c.W, s)
    LN_BY_CFG(c);
    #undef LN
}
#undef LN_BY_CFG
#undef LN_WIDE

}  // namespace

extern "C" {

int ptcg_layer_norm_fwd(const void* x, int x_dtype, long ldx, const float* gamma,
                        const float* beta, float eps, void* y, int y_dtype, long ldy, float* mean,
                        float* rstd, long rows, int width, void* stream) {
    OP_REQ(dt_ok(x_dtype) && dt_ok(y_dtype), PTCG_EINVAL, "layer norm: unknown dtype");
    OP_REQ(rows >= 0 && width > 0 && width <= MAXW && ldx >= width && ldy >= width, PTCG_EINVAL,
           "layer norm: bad sizes (rows %ld, width %d of at most %d, ldx %ld, ldy %ld)", rows, width,
           MAXW, ldx, ldy);
    if (rows == 0) return PTCG_OK;
    OP_REQ(x && y, PTCG_EINVAL, "layer norm: null pointer");
    OP_REQ(el_ok(x, x_dtype) && el_ok(y, y_dtype) && el_ok(gamma, PTCG_FP32) && el_ok(beta, PTCG_FP32) &&
           el_ok(mean, PTCG_FP32) && el_ok(rstd, PTCG_FP32), PTCG_EINVAL,
           "layer norm: pointer not aligned to its element");
    const Cfg c = cfg_of(width, mode_of(width, {{x, x_dtype, ldx}, {y, y_dtype, ldy}}));
    cudaStream_t s = (cudaStream_t)stream;
    #define LN(TX, TY) fwd<TX, TY>(c, y, ldy, mean, rstd, x, ldx, gamma, beta, rows, width, eps, s)
    if (x_dtype == PTCG_BF16) { if (y_dtype == PTCG_BF16) LN(bf16, bf16); else LN(bf16, float); }
    else { if (y_dtype == PTCG_BF16) LN(float, bf16); else LN(float, float); }
    #undef LN
    OP_CKL();
    return PTCG_OK;
}

long ptcg_layer_norm_bwd_scratch(long rows, int width) {
    OP_REQ(rows >= 0 && width > 0 && width <= MAXW, -1,
           "layer norm gradient: bad sizes (rows %ld, width %d of at most %d)", rows, width, MAXW);
    return 8L * width * bwd_blocks(rows, width);    // the same for every variant
}

int ptcg_layer_norm_bwd(const void* dy, int dy_dtype, long lddy, const void* x, int x_dtype,
                        long ldx, const float* gamma, const float* mean, const float* rstd,
                        const void* dres, long lddres, void* dx, long lddx, float* dgamma,
                        float* dbeta, int accumulate, long rows, int width, void* scratch,
                        long scratch_bytes, void* stream) {
    OP_REQ(dt_ok(x_dtype) && dt_ok(dy_dtype), PTCG_EINVAL, "layer norm gradient: unknown dtype");
    OP_REQ(rows >= 0 && width > 0 && width <= MAXW && lddy >= width && ldx >= width && lddx >= width &&
           (!dres || lddres >= width), PTCG_EINVAL,
           "layer norm gradient: bad sizes (rows %ld, width %d of at most %d)", rows, width, MAXW);
    OP_REQ(!dgamma == !dbeta, PTCG_EINVAL, "layer norm gradient: dgamma and dbeta come together");
    OP_REQ(el_ok(x, x_dtype) && el_ok(dy, dy_dtype) && el_ok(dx, x_dtype) && el_ok(dres, x_dtype) &&
           el_ok(gamma, PTCG_FP32) && el_ok(mean, PTCG_FP32) && el_ok(rstd, PTCG_FP32) &&
           el_ok(dgamma, PTCG_FP32) && el_ok(dbeta, PTCG_FP32) && el_ok(scratch, PTCG_FP32), PTCG_EINVAL,
           "layer norm gradient: pointer not aligned to its element");
    cudaStream_t s = (cudaStream_t)stream;
    if (rows == 0) {
        if (dgamma && !accumulate) {
            OP_CK(cudaMemsetAsync(dgamma, 0, 4L * width, s));
            OP_CK(cudaMemsetAsync(dbeta, 0, 4L * width, s));
        }
        return PTCG_OK;
    }
    OP_REQ(dy && x && mean && rstd && dx, PTCG_EINVAL, "layer norm gradient: null pointer");
    const long need = ptcg_layer_norm_bwd_scratch(rows, width);
    OP_REQ(!dgamma || (scratch && scratch_bytes >= need), PTCG_ERANGE,
           "layer norm gradient: scratch of %ld bytes, %ld needed", scratch ? scratch_bytes : 0L, need);
    const Cfg c = cfg_of(width, mode_of(width, {{x, x_dtype, ldx}, {dy, dy_dtype, lddy}, {dx, x_dtype, lddx},
                                                {dres, x_dtype, lddres}}));
    const int blocks = bwd_blocks(rows, width);
    const BwdArgs a = {dx, lddx, dy, lddy, x, ldx, dres, lddres, gamma, mean, rstd, rows, width,
                       dgamma ? (float*)scratch : nullptr};
    if (x_dtype == PTCG_BF16) { if (dy_dtype == PTCG_BF16) bwd<bf16, bf16>(c, a, blocks, s); else bwd<bf16, float>(c, a, blocks, s); }
    else { if (dy_dtype == PTCG_BF16) bwd<float, bf16>(c, a, blocks, s); else bwd<float, float>(c, a, blocks, s); }
    if (dgamma)
        ++g_ptcg_launches, k_layer_norm_wgrad<<<cdiv(2L * width, 32), 256, 0, s>>>(
            dgamma, dbeta, (const float*)scratch, blocks, width, accumulate);
    OP_CKL();
    return PTCG_OK;
}

}  // extern "C"
