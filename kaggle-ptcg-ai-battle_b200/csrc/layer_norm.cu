// Layer norm over rows, its backward pass and the reduction of the weight
// gradients, for any row width up to PTCG_LN_MAX_WIDTH.
//   forward   mu = mean x, r = (mean (x - mu)^2 + eps)^(-1/2),
//             h = (x - mu) r, y = h gamma + beta
//   backward  g = dy gamma, dx = r (g - mean g - h mean(g h)) (+ dres),
//             dgamma = sum over rows of dy h, dbeta = sum over rows of dy
// (torch nn.LayerNorm; the model's own norms, ptcg/rl/model.py:70-91, run
// kernels tied to its row layouts.)  The statistics are two passes over the
// row in registers, so no cancellation between sums of squares; everything
// is fp32 until the one rounding to the output's type.
#include <algorithm>

#include "vec.cuh"

namespace {

constexpr int MAXW = PTCG_LN_MAX_WIDTH;
// one warp holds rows of up to 1024 columns, NV pieces of V columns per lane;
// wider rows are shared by the warps of a block, 256 columns each, so that the
// backward's registers per column still fit 1024 threads
constexpr int WARP_COLS = 1024, SHARED_COLS = 256, MAX_THREADS = MAXW / SHARED_COLS * 32;

// Bound: HBM.  A row belongs to one warp (width <= 1024, eight rows to a
// block) or to the W warps of a block (MULTI).  Lane l of warp w owns pieces
// w * 32 * NV + l, + 32, .. so that a warp's accesses are contiguous.
template <int V, int NV>
PTCG_DEV int piece_at(int w, int lane, int k) { return (w * NV + k) * 32 + lane; }

// sum of v over the row's warps; `slot` alternates so that one barrier per
// reduction is enough
template <bool MULTI>
PTCG_DEV float row_sum(float v, float (*red)[32], int slot, int w, int lane, int W) {
    v = warp_sum(v);
    if (!MULTI) return v;
    if (lane == 0) red[slot][w] = v;
    __syncthreads();
    return warp_sum(lane < W ? red[slot][lane] : 0.f);
}

template <typename TX, typename TY, int V, int NV, bool MULTI>
__global__ void __launch_bounds__(MULTI ? MAX_THREADS : 256) k_layer_norm_fwd(
        TY* y, long ldy, float* mean, float* rstd, const TX* x, long ldx,
        const float* __restrict__ gamma, const float* __restrict__ beta, long rows, int width,
        float eps) {
    __shared__ float red[4][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = blockDim.x >> 5;
    const int w = MULTI ? warp : 0, pieces = width / V;
    const float inv = 1.f / (float)width;
    float gm[NV][V], bt[NV][V];
    #pragma unroll
    for (int k = 0; k < NV; k++) {
        const int p = piece_at<V, NV>(w, lane, k);
        #pragma unroll
        for (int e = 0; e < V; e++) { gm[k][e] = 1.f; bt[k][e] = 0.f; }
        if (p < pieces) {
            #pragma unroll
            for (int e = 0; e < V; e++) {
                if (gamma) gm[k][e] = gamma[p * V + e];
                if (beta) bt[k][e] = beta[p * V + e];
            }
        }
    }
    const long step = MULTI ? gridDim.x : (long)gridDim.x * W;
    // the next row's loads are in flight while this one is reduced, where the
    // registers allow it
    constexpr bool AHEAD = NV * V <= 8;
    Raw<TX, V> row[NV];
    auto fetch = [&](long r) {
        #pragma unroll
        for (int k = 0; k < NV; k++) {
            const int p = piece_at<V, NV>(w, lane, k);
            row[k].zero();
            if (r < rows && p < pieces) row[k].ld(x + r * ldx + (long)p * V);
        }
    };
    int slot = 0;
    long r = MULTI ? blockIdx.x : (long)blockIdx.x * W + warp;
    if (AHEAD) fetch(r);
    for (; r < rows; r += step) {
        float v[NV][V];
        float s = 0.f;
        if (!AHEAD) fetch(r);
        #pragma unroll
        for (int k = 0; k < NV; k++) row[k].get(v[k]);
        if (AHEAD) fetch(r + step);
        #pragma unroll
        for (int k = 0; k < NV; k++)
            #pragma unroll
            for (int e = 0; e < V; e++) s += v[k][e];
        // rounded here, so that x - mu is the same whether or not mean is stored
        const float mu = __fmul_rn(row_sum<MULTI>(s, red, slot, w, lane, W), inv);
        float q = 0.f;
        #pragma unroll
        for (int k = 0; k < NV; k++) {
            const float in = piece_at<V, NV>(w, lane, k) < pieces ? 1.f : 0.f;
            #pragma unroll
            for (int e = 0; e < V; e++) { const float d = (v[k][e] - mu) * in; q = fmaf(d, d, q); }
        }
        const float rs = rsqrtf(fmaf(row_sum<MULTI>(q, red, slot + 1, w, lane, W), inv, eps));
        slot ^= 2;
        if (lane == 0 && w == 0) {
            if (mean) mean[r] = mu;
            if (rstd) rstd[r] = rs;
        }
        #pragma unroll
        for (int k = 0; k < NV; k++) {
            const int p = piece_at<V, NV>(w, lane, k);
            if (p < pieces) {
                #pragma unroll
                for (int e = 0; e < V; e++) v[k][e] = fmaf((v[k][e] - mu) * rs, gm[k][e], bt[k][e]);
                VecIO<TY, V>::st(y + r * ldy + (long)p * V, v[k]);
            }
        }
    }
}

// Backward: the same ownership, each lane keeping the weight-gradient sums of
// its columns in registers over all its rows.  They leave once per block, in
// warp order through shared memory, as one partial row of dgamma and dbeta;
// k_layer_norm_wgrad adds the blocks' partials in a fixed order.  No atomics,
// so equal inputs give equal bits.
template <typename TX, typename TY, int V, int NV, bool MULTI>
__global__ void __launch_bounds__(MULTI ? MAX_THREADS : 256) k_layer_norm_bwd(
        TX* dx, long lddx, const TY* dy, long lddy, const TX* x, long ldx,
        const TX* dres, long lddres, const float* __restrict__ gamma,
        const float* __restrict__ mean, const float* __restrict__ rstd, long rows, int width,
        float* __restrict__ partial) {
    __shared__ float red[4][32];
    extern __shared__ float cols[];                 // [2][width] of a one-warp-per-row block
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = blockDim.x >> 5;
    const int w = MULTI ? warp : 0, pieces = width / V;
    const float inv = 1.f / (float)width;
    float gm[NV][V], ag[NV][V], ab[NV][V];
    #pragma unroll
    for (int k = 0; k < NV; k++) {
        const int p = piece_at<V, NV>(w, lane, k);
        #pragma unroll
        for (int e = 0; e < V; e++) {
            gm[k][e] = gamma && p < pieces ? gamma[p * V + e] : 1.f;
            ag[k][e] = ab[k][e] = 0.f;
        }
    }
    const long step = MULTI ? gridDim.x : (long)gridDim.x * W;
    int slot = 0;
    // the next row's loads are in flight while this one is reduced, where the
    // registers allow it
    constexpr bool AHEAD = !MULTI && NV * V <= 8;
    struct Row { Raw<TX, V> x[NV], r[NV]; Raw<TY, V> g[NV]; float mu, rs; } row;
    auto fetch = [&](long r) {
        #pragma unroll
        for (int k = 0; k < NV; k++) {
            const int p = piece_at<V, NV>(w, lane, k);
            row.x[k].zero(); row.g[k].zero(); row.r[k].zero();
            if (r < rows && p < pieces) {
                row.x[k].ld(x + r * ldx + (long)p * V);
                row.g[k].ld(dy + r * lddy + (long)p * V);
                if (dres) row.r[k].ld(dres + r * lddres + (long)p * V);
            }
        }
        row.mu = r < rows ? mean[r] : 0.f;
        row.rs = r < rows ? rstd[r] : 0.f;
    };
    long r = MULTI ? blockIdx.x : (long)blockIdx.x * W + warp;
    if (AHEAD) fetch(r);
    for (; r < rows; r += step) {
        float h[NV][V], g[NV][V], d[NV][V];
        if (!AHEAD) fetch(r);
        const float mu = row.mu, rs = row.rs;
        #pragma unroll
        for (int k = 0; k < NV; k++) {
            row.x[k].get(h[k]);
            row.g[k].get(g[k]);
            row.r[k].get(d[k]);
        }
        if (AHEAD) fetch(r + step);
        float s1 = 0.f, s2 = 0.f;
        #pragma unroll
        for (int k = 0; k < NV; k++) {
            #pragma unroll
            for (int e = 0; e < V; e++) {
                const float hh = (h[k][e] - mu) * rs;
                ag[k][e] = fmaf(g[k][e], hh, ag[k][e]);
                ab[k][e] += g[k][e];
                g[k][e] *= gm[k][e];
                h[k][e] = hh;
                s1 += g[k][e];
                s2 = fmaf(g[k][e], hh, s2);
            }
        }
        if (MULTI) {
            s1 = warp_sum(s1);
            s2 = warp_sum(s2);
            if (lane == 0) { red[slot][w] = s1; red[slot + 1][w] = s2; }
            __syncthreads();
            s1 = warp_sum(lane < W ? red[slot][lane] : 0.f);
            s2 = warp_sum(lane < W ? red[slot + 1][lane] : 0.f);
            slot ^= 2;
        } else {
            s1 = warp_sum(s1);
            s2 = warp_sum(s2);
        }
        const float m1 = __fmul_rn(s1, inv), m2 = __fmul_rn(s2, inv);
        #pragma unroll
        for (int k = 0; k < NV; k++) {
            const int p = piece_at<V, NV>(w, lane, k);
            if (p < pieces) {
                #pragma unroll
                for (int e = 0; e < V; e++) {
                    const float t = (g[k][e] - m1 - h[k][e] * m2) * rs;
                    h[k][e] = dres ? t + d[k][e] : t;
                }
                VecIO<TX, V>::st(dx + r * lddx + (long)p * V, h[k]);
            }
        }
    }
    if (!partial) return;
    float* out = partial + (long)blockIdx.x * 2 * width;
    if constexpr (MULTI) {
        #pragma unroll
        for (int k = 0; k < NV; k++) {
            const int p = piece_at<V, NV>(w, lane, k);
            if (p < pieces) {
                #pragma unroll
                for (int e = 0; e < V; e++) {
                    out[p * V + e] = ag[k][e];
                    out[width + p * V + e] = ab[k][e];
                }
            }
        }
    } else {
        for (int t = 0; t < W; t++) {
            if (warp == t) {
                #pragma unroll
                for (int k = 0; k < NV; k++) {
                    const int p = piece_at<V, NV>(0, lane, k);
                    if (p < pieces) {
                        #pragma unroll
                        for (int e = 0; e < V; e++) {
                            float* c = cols + p * V + e;
                            c[0] = t ? c[0] + ag[k][e] : ag[k][e];
                            c[width] = t ? c[width] + ab[k][e] : ab[k][e];
                        }
                    }
                }
            }
            __syncthreads();
        }
        for (int i = threadIdx.x; i < 2 * width; i += blockDim.x) out[i] = cols[i];
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

// the variant of a row width: V-column pieces, NV of them per lane, W warps a
// row (0: one warp a row, eight rows a block)
struct Cfg { int V, NV, W; };
Cfg cfg_of(int width, bool vec) {
    Cfg c;
    c.V = vec ? 4 : 1;
    if (width > WARP_COLS) {
        c.NV = SHARED_COLS / (32 * c.V);
        c.W = (int)cdiv(width, SHARED_COLS);
        return c;
    }
    c.W = 0;
    c.NV = 1;
    while (c.NV * 32 * c.V < width) c.NV *= 2;
    if (c.V == 1 && c.NV < 4) c.NV = 4;
    return c;
}
// blocks of the backward pass: as many as the processors hold, at most one
// per row group, so that each leaves one partial row of the weight gradients
int bwd_blocks(long rows, const Cfg& c) {
    const long units = c.W ? rows : (rows + 7) / 8;
    const long most = c.W ? std::max(148 * 32 / c.W, 148) : 148 * 4;
    return (int)(units < most ? units : most);
}

template <typename TX, typename TY, int V, int NV, bool MULTI>
void fwd(void* y, long ldy, float* mean, float* rstd, const void* x, long ldx, const float* gamma,
         const float* beta, long rows, int width, float eps, int W, cudaStream_t s) {
    const long units = MULTI ? rows : (rows + 7) / 8;
    const long most = MULTI ? std::max(148 * 64 / W, 148) : 148 * 8;
    ++g_ptcg_launches;
    k_layer_norm_fwd<TX, TY, V, NV, MULTI><<<(unsigned)(units < most ? units : most), MULTI ? W * 32 : 256, 0, s>>>(
        (TY*)y, ldy, mean, rstd, (const TX*)x, ldx, gamma, beta, rows, width, eps);
}
template <typename TX, typename TY>
void fwd(const Cfg& c, void* y, long ldy, float* mean, float* rstd, const void* x, long ldx,
         const float* gamma, const float* beta, long rows, int width, float eps, cudaStream_t s) {
    #define LN(V, NV, M) fwd<TX, TY, V, NV, M>(y, ldy, mean, rstd, x, ldx, gamma, beta, rows, width, eps, c.W, s)
    if (c.V == 4) {
        if (c.W) LN(4, 2, true);
        else if (c.NV == 1) LN(4, 1, false);
        else if (c.NV == 2) LN(4, 2, false);
        else if (c.NV == 4) LN(4, 4, false);
        else LN(4, 8, false);
    } else {
        if (c.W) LN(1, 8, true);
        else if (c.NV == 4) LN(1, 4, false);
        else if (c.NV == 8) LN(1, 8, false);
        else if (c.NV == 16) LN(1, 16, false);
        else LN(1, 32, false);
    }
    #undef LN
}

struct BwdArgs {
    void* dx; long lddx; const void* dy; long lddy; const void* x; long ldx;
    const void* dres; long lddres; const float* gamma; const float* mean; const float* rstd;
    long rows; int width; float* partial;
};
template <typename TX, typename TY, int V, int NV, bool MULTI>
void bwd(const BwdArgs& a, int blocks, int W, cudaStream_t s) {
    ++g_ptcg_launches;
    k_layer_norm_bwd<TX, TY, V, NV, MULTI><<<blocks, MULTI ? W * 32 : 256, MULTI ? 0 : 8 * a.width, s>>>(
        (TX*)a.dx, a.lddx, (const TY*)a.dy, a.lddy, (const TX*)a.x, a.ldx, (const TX*)a.dres,
        a.lddres, a.gamma, a.mean, a.rstd, a.rows, a.width, a.partial);
}
template <typename TX, typename TY>
void bwd(const Cfg& c, const BwdArgs& a, int blocks, cudaStream_t s) {
    #define LN(V, NV, M) bwd<TX, TY, V, NV, M>(a, blocks, c.W, s)
    if (c.V == 4) {
        if (c.W) LN(4, 2, true);
        else if (c.NV == 1) LN(4, 1, false);
        else if (c.NV == 2) LN(4, 2, false);
        else if (c.NV == 4) LN(4, 4, false);
        else LN(4, 8, false);
    } else {
        if (c.W) LN(1, 8, true);
        else if (c.NV == 4) LN(1, 4, false);
        else if (c.NV == 8) LN(1, 8, false);
        else if (c.NV == 16) LN(1, 16, false);
        else LN(1, 32, false);
    }
    #undef LN
}

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
    const Cfg c = cfg_of(width, width % 4 == 0 && vec_ok(x, x_dtype, ldx, 4) && vec_ok(y, y_dtype, ldy, 4));
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
    // the scalar and the vector variant use the same number of blocks
    return 8L * width * bwd_blocks(rows, cfg_of(width, true));
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
    const Cfg c = cfg_of(width, width % 4 == 0 && vec_ok(x, x_dtype, ldx, 4) && vec_ok(dy, dy_dtype, lddy, 4) &&
                         vec_ok(dx, x_dtype, lddx, 4) && vec_ok(dres, x_dtype, lddres, 4));
    const int blocks = bwd_blocks(rows, c);
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
