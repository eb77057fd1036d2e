// Cross attention of long bf16 problems on the 5th-generation tensor cores
// (tcgen05 / TMEM): the formulas, masks and row stacking of
// cross_attention.cu.
//
// Operand tiles have the layouts the MMA descriptors read: rows of 128 bytes
// (64 for head width 32) with their 16-byte pieces permuted by the row, DH in
// blocks of 64 columns, as TMA writes them; the same tile serves as a K-major
// operand (rows are M or N) and as an MN-major one (rows are K).  A masked
// key's scores are replaced after the product, so its K row may hold anything;
// its V row is overwritten with zeros in shared memory before the product
// (0 * NaN would be NaN).
//
// Every mbarrier wait is bounded; on expiry the block records an error code
// (ptcg_device_error), its roles stop, copies and MMAs in flight land, TMEM is
// freed and the kernel returns.
#include "cross.cuh"
#include "tc_ptx.cuh"

namespace {

using namespace cross;
using namespace tcx;

__device__ int g_cross_tc_error;

PTCG_DEV bool wait_bar(uint32_t b, uint32_t parity, volatile int* abort_flag, int code) {
    return bar_try(b, parity) || tcx::bar_wait(b, parity, abort_flag, &g_cross_tc_error, code);
}
// warp-uniform outcome: the TMEM accesses after it are warp-collective
PTCG_DEV bool wait_warp(uint32_t b, uint32_t parity, volatile int* abort_flag, int code) {
    return __all_sync(0xffffffffu, wait_bar(b, parity, abort_flag, code));
}
PTCG_DEV void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
PTCG_DEV void tmem_ld32(uint32_t taddr, float* v) {
    uint32_t r[32];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]),
                   "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
                   "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
                   "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                   "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]),
                   "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr));
    #pragma unroll
    for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[i]);
}
PTCG_DEV void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
                 "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 :: "r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]),
                    "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]),
                    "r"(v[13]), "r"(v[14]), "r"(v[15]) : "memory");
}
PTCG_DEV void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// D (TMEM) (+)= A B, A from TMEM
PTCG_DEV void mma_bf16_ts(uint32_t d, uint32_t a_tmem, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "setp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 :: "r"(d), "r"(a_tmem), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
// one lane of a converged warp, the same one each time.  The MMA warps run
// their loops on all lanes and issue under this predicate: addresses and
// descriptors then stay in uniform registers
PTCG_DEV bool elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "elect.sync _|p, 0xffffffff;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}
PTCG_DEV float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// N-row tiles of DH columns
template <int DH, int N> struct Tile {
    static constexpr int ROWB = DH == 32 ? 64 : 128;          // bytes of a row in a block
    static constexpr uint32_t LAYOUT = DH == 32 ? 4 : 2, SBO = ROWB * 8;
    static constexpr int BLOCK = N * ROWB;                    // bytes of a 64-column block
    static constexpr int KPB = ROWB / 32, BYTES = N * DH * 2;
    // 16-byte piece c of row r
    static PTCG_DEV uint32_t off(int r, int c) {
        const int x = DH == 32 ? (r >> 1) & 3 : r & 7;
        return (c / (ROWB / 16)) * BLOCK + r * ROWB + (((c % (ROWB / 16)) ^ x) << 4);
    }
    // Shared-memory descriptors, low and high word apart: a K step adds a
    // constant to the low word (building 64 bits per MMA made its issue the
    // bound: 32 MMAs a step at some 25 instructions of one thread).
    static constexpr uint32_t HI = (SBO >> 4) | (1u << 14) | (LAYOUT << 29);
    static PTCG_DEV uint32_t lo_k(uint32_t base) { return (base >> 4) | ((16u >> 4) << 16); }
    static PTCG_DEV uint32_t lo_mn(uint32_t base) { return (base >> 4) | ((uint32_t)(BLOCK >> 4) << 16); }
    // columns 16 s .. as the K step of a K-major operand
    static PTCG_DEV uint64_t kmajor(uint32_t lo, int s) {
        return ((uint64_t)HI << 32) | (lo + (((s / KPB) * BLOCK + (s % KPB) * 32) >> 4));
    }
    // rows 16 s .. as the K step of an MN-major operand
    static PTCG_DEV uint64_t mnmajor(uint32_t lo, int s) {
        return ((uint64_t)HI << 32) | (lo + ((s * 16 * ROWB) >> 4));
    }
};

// the kept bits of keys k0 .. k0 + 32 W - 1, word i = keys k0 + 32 i ..
template <int W> struct KeyBits {
    bool in[W];
    PTCG_DEV void fetch(const CrossArgs& a, int seq, int k0, int kend, int len, int lane) {
        #pragma unroll
        for (int i = 0; i < W; i++) {
            const int key = k0 + i * 32 + lane;
            in[i] = key < kend && kept(a, seq, key, len);
        }
    }
    PTCG_DEV void words(uint32_t (&w)[W]) const {
        #pragma unroll
        for (int i = 0; i < W; i++) w[i] = __ballot_sync(0xffffffffu, in[i]);
    }
};

// zeros in the rows of a tile whose bit is clear
template <int DH, int N>
PTCG_DEV void clear_rows(uint8_t* tile, const uint32_t (&w)[N / 32], int lane) {
    #pragma unroll
    for (int c = 0; c < N / 32; c++) {
        if ((w[c] >> lane) & 1) continue;
        #pragma unroll
        for (int q = 0; q < DH / 8; q++)
            *(uint4*)(tile + Tile<DH, N>::off(c * 32 + lane, q)) = make_uint4(0u, 0u, 0u, 0u);
    }
}
// 128 stacked query rows from r0 by the 128 threads of a warpgroup; rows past
// the end are zeros.  Returns when this thread's pieces are there
template <int DH>
PTCG_DEV void stage_q(uint32_t dst, const CrossArgs& a, const Where& at, int r0, int tid) {
    constexpr int P = DH / 8, STEP = 128 / P;
    const int pr = tid / P, pc = tid % P;
    const bf16* q = (const bf16*)a.q + at.seq * a.sq.seq + (long)(at.hk * a.group) * a.sq.head + pc * 8;
    #pragma unroll 4
    for (int n = 0; n < 128; n += STEP) {
        const int r = r0 + pr + n;
        const bool in = r < a.rows;
        const int g = a.by_lq.div(in ? r : 0), i = (in ? r : 0) - g * a.lq;
        cp16(dst + Tile<DH, 128>::off(pr + n, pc), q + i * a.sq.row + g * a.sq.head, in);
    }
    cp_commit();
    cp_wait<0>();
}

// start and end of a block's life with TMEM; warp 10 allocates and frees
PTCG_DEV void tmem_alloc(uint32_t* slot) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 :: "r"(s_addr(slot)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
PTCG_DEV void tmem_free(uint32_t tmem) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(512) : "memory");
}

// ------------------------------------------------------------------ forward
// One block per SM takes two 128-row tiles of the stacked rows and walks the
// keys 128 at a time.  Warps 0-3 and 4-7 are the softmax of one tile each (a
// row per thread, its 128 scores in registers: 12 warps leave 168 a thread,
// 13 would leave 128); a lane of warp 8 loads K and V by TMA, warp 9 clears
// the masked rows of V, and warp 10 issues the MMAs:
//   S_t = Q_t K_j^T (M = 128 rows, N = 128 keys), O_t += P_t V_j (A = P from
//   TMEM, over the columns of S_t; N = DH)
// in the order PV_0(j) S_0(j+1) PV_1(j) S_1(j+1), so that one tile's products
// run while the other's softmax does.  MMAs of one thread complete in order:
// once S_t(j+1) is there, PV_t(j) is done and O_t may be rescaled.  A row's
// maximum is raised (and O_t rescaled) only when it grew by more than 2^8:
// until then the probabilities are at most 2^8 and the sum stays exact enough
// in fp32, and the final division takes the common factor out.  P is rounded to
// bf16 as an operand, at most 2^-8 of each probability, the size of the output's
// own rounding; its sum is taken before that.
// TMEM: S_0 0-127, S_1 128-255, O_0 256.., O_1 256 + DH.. .
// Bound: the exponentials (16 a clock and SM) and, at DH 128, equally the
// tensor core: 2048 clocks each per 256 x 128 scores.  131232 stacked rows on
// 8191 keys of width 128: 508 us, 1083 TFLOP/s; the tensor and the exponentials'
// pipes are busy 69 % each.  In a loop with the backward the power cap holds the
// clock at 1792 of 1965 MHz.
template <int DH> struct Fwd {
    static constexpr int NS = DH == 128 ? 2 : DH == 64 ? 4 : 7;       // K and V stages
    using T = Tile<DH, 128>;
    // barriers: kfull[NS] vfull[NS] vready[NS] kfree[NS] vfree[NS] qfull[2] sfull[2] pready[2][2]
    // ofull[2] drain
    static constexpr int BARS = 5 * NS + 11;
    static constexpr int SMEM = 1024 + (2 + 2 * NS) * T::BYTES + BARS * 8 + 16;
    static constexpr int THREADS = 384;
};
PTCG_DEV void tma_4d(uint32_t dst, const CUtensorMap* map, uint32_t b, int x, int y, int z, int w) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
                 " [%0], [%1, {%3, %4, %5, %6}], [%2];"
                 :: "r"(dst), "l"((uint64_t)map), "r"(b), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
// a tensor of rows for TMA: dimensions (column, row, head, sequence); a
// dimension that the tensor repeats (stride 0) has one entry and coordinate 0
struct RowMap { CUtensorMap map; int heads, seqs; };
// rows row .. + N - 1 of one head into a tile; the barrier has been told the bytes
template <int DH, int N>
PTCG_DEV void load_rows(uint32_t dst, const RowMap& m, uint32_t b, int row, int head, int seq) {
    using T = Tile<DH, N>;
    #pragma unroll
    for (int c = 0; c < DH * 2 / T::ROWB; c++)
        tma_4d(dst + c * T::BLOCK, &m.map, b, c * (T::ROWB / 2), row, head * m.heads, seq * m.seqs);
}

template <int DH>
__global__ void __launch_bounds__(Fwd<DH>::THREADS, 1) k_cross_fwd_tc(
        const __grid_constant__ CrossArgs a, const __grid_constant__ RowMap kmap, const __grid_constant__ RowMap vmap) {
    using F = Fwd<DH>;
    using T = Tile<DH, 128>;
    constexpr int NS = F::NS, KS = DH / 16, BN = 128;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const uint32_t sQ = s_addr(smem), sK = sQ + 2 * T::BYTES, sV = sK + NS * T::BYTES;
    uint64_t* bars = (uint64_t*)(smem + (2 + 2 * NS) * T::BYTES);
    const uint32_t kfull = s_addr(bars), vfull = kfull + 8 * NS, vready = vfull + 8 * NS,
                   kfree = vready + 8 * NS, vfree = kfree + 8 * NS, qfull = vfree + 8 * NS,
                   sfull = qfull + 16, pready = sfull + 16, ofull = pready + 32, drain = ofull + 16;
    uint32_t* tmem_slot = (uint32_t*)(bars + F::BARS);
    volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Where at = where(a);
    const int r0 = at.tile * TC_ROWS, len = kept_len(a, at.seq);
    const int kbeg = min(at.part * a.split, len), kend = min(len, kbeg + a.split);
    const int nt = (kend - kbeg + BN - 1) / BN;
    const bool two = r0 + 128 < a.rows;
    if (threadIdx.x == 0) {
        for (int i = 0; i < NS; i++) {
            bar_init(kfull + 8 * i, 1); bar_init(vfull + 8 * i, 1); bar_init(vready + 8 * i, 1);
            bar_init(kfree + 8 * i, 1); bar_init(vfree + 8 * i, 1);
        }
        for (int t = 0; t < 2; t++) {
            bar_init(qfull + 8 * t, 128); bar_init(sfull + 8 * t, 1);
            bar_init(pready + 16 * t, 128); bar_init(pready + 16 * t + 8, 128); bar_init(ofull + 8 * t, 1);
        }
        bar_init(drain, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async();
    }
    if (warp == 10) tmem_alloc(tmem_slot);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    if (warp == 8) {
        // ------------------------------------------------- TMA lane
        if (lane == 0) {
            int j = 0;
            for (; j < nt; j++) {
                const int s = j % NS;
                const uint32_t parity = (uint32_t)(((j / NS) & 1) ^ 1);
                if (!wait_bar(kfree + 8 * s, parity, abort_flag, 1)) break;
                bar_expect_tx(kfull + 8 * s, T::BYTES);
                load_rows<DH, BN>(sK + s * T::BYTES, kmap, kfull + 8 * s, kbeg + j * BN, at.hk, at.seq);
                if (!wait_bar(vfree + 8 * s, parity, abort_flag, 2)) { j++; break; }
                bar_expect_tx(vfull + 8 * s, T::BYTES);
                load_rows<DH, BN>(sV + s * T::BYTES, vmap, vfull + 8 * s, kbeg + j * BN, at.hk, at.seq);
            }
            // on an abort, let the copies still in flight land before exiting
            if (*abort_flag)
                for (int i = max(0, j - NS); i < j; i++) {
                    bar_drain(kfull + 8 * (i % NS), (i / NS) & 1);
                    if (i < nt) bar_drain(vfull + 8 * (i % NS), (i / NS) & 1);
                }
        }
        __syncwarp();
    } else if (warp == 9) {
        // ------------------------------------ masked rows of V become zeros
        KeyBits<4> kb;
        kb.fetch(a, at.seq, kbeg, kend, len, lane);
        for (int j = 0; j < nt; j++) {
            uint32_t w[4];
            kb.words(w);
            kb.fetch(a, at.seq, kbeg + (j + 1) * BN, kend, len, lane);
            const int s = j % NS;
            if (!wait_warp(vfull + 8 * s, (j / NS) & 1, abort_flag, 3)) break;
            if ((w[0] & w[1] & w[2] & w[3]) != 0xffffffffu) {
                clear_rows<DH, BN>(smem + (2 + NS + s) * T::BYTES, w, lane);
                fence_async();
                __syncwarp();
            }
            if (lane == 0) bar_arrive(vready + 8 * s);
        }
    } else if (warp >= 10) {
        // ---------------------------------------------------- MMA warp
        if (warp == 10 && nt > 0) {
            const uint32_t ids = idesc_bf16(BN, 0, 0), ido = idesc_bf16(DH, 0, 1);
            const uint32_t qlo = T::lo_k(sQ), klo = T::lo_k(sK), vlo = T::lo_mn(sV);
            const int T2 = two ? 2 : 1;
            bool ok = true;
            int ks = 0, vs = 0;                             // stages, and their phases
            uint32_t kp = 0, vp = 0;
            for (int j = 0; ok && j <= nt; j++) {
                // the operands of this step are waited for before the
                // probabilities, off the path from them to the next scores
                ok = (j == 0 || wait_warp(vready + 8 * vs, vp, abort_flag, 5)) &&
                     (j == nt || wait_warp(kfull + 8 * ks, kp, abort_flag, 7));
                const uint32_t v = vlo + ((vs * T::BYTES) >> 4), k = klo + ((ks * T::BYTES) >> 4);
                for (int t = 0; t < T2 && ok; t++) {
                    const uint32_t ts = tmem + t * 128, to = tmem + 256 + t * DH;
                    const uint32_t q = qlo + ((t * T::BYTES) >> 4);
                    if (j == 0) {
                        ok = wait_warp(qfull + 8 * t, 0, abort_flag, 4);
                        tc_fence_after();
                    }
                    #pragma unroll
                    for (int h = 0; h < 2; h++) {           // O_t += P_t V of tile j - 1, 64 keys at a time
                        if (j == 0 || !ok) continue;
                        ok = wait_warp(pready + 16 * t + 8 * h, (j - 1) & 1, abort_flag, 6);
                        tc_fence_after();
                        if (ok && elect_one()) {
                            #pragma unroll
                            for (int s = 4 * h; s < 4 * h + 4; s++)
                                mma_bf16_ts(to, ts + 8 * s, T::mnmajor(v, s), ido, s > 0 ? 1u : j > 1);
                        }
                        __syncwarp();
                    }
                    if (ok && elect_one()) {
                        if (j > 0 && t == T2 - 1) mma_commit_to(vfree + 8 * vs);
                        if (j < nt) {                       // S_t of tile j
                            #pragma unroll
                            for (int s = 0; s < KS; s++)
                                mma_bf16(ts, T::kmajor(q, s), T::kmajor(k, s), ids, s > 0);
                            mma_commit_to(sfull + 8 * t);
                            if (t == T2 - 1) mma_commit_to(kfree + 8 * ks);
                        } else {
                            mma_commit_to(ofull + 8 * t);
                        }
                    }
                    __syncwarp();
                }
                if (j > 0 && ++vs == NS) { vs = 0; vp ^= 1; }
                if (++ks == NS) { ks = 0; kp ^= 1; }
            }
            // no MMA may still be in flight when TMEM is released
            if (elect_one()) {
                mma_commit_to(drain);
                bar_drain(drain, 0);
            }
            __syncwarp();
        }
    } else if (warp < 8) {
        // ----------------------------------------------------- softmax
        const int t = warp >> 2, quad = warp & 3, row = quad * 32 + lane;
        const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
        const uint32_t ts = tmem + lane_off + t * 128, to = tmem + lane_off + 256 + t * DH;
        const float sc = a.scale * LOG2E;
        float m = -INFINITY, l = 0.f;                       // the shift in use, and the row sum
        bool ok = t == 0 || two;
        if (ok && nt > 0) {
            stage_q<DH>(sQ + t * T::BYTES, a, at, r0 + t * 128, threadIdx.x & 127);
            fence_async();
            bar_arrive(qfull + 8 * t);
        }
        KeyBits<4> kb;
        kb.fetch(a, at.seq, kbeg, kend, len, lane);
        for (int j = 0; ok && j < nt; j++) {
            uint32_t w[4];
            kb.words(w);
            kb.fetch(a, at.seq, kbeg + (j + 1) * BN, kend, len, lane);
            ok = wait_warp(sfull + 8 * t, j & 1, abort_flag, 8);
            if (!ok) break;
            tc_fence_after();
            float v[128];
            #pragma unroll
            for (int c = 0; c < 4; c++) tmem_ld32(ts + 32 * c, v + 32 * c);
            tmem_wait_ld();
            if ((w[0] & w[1] & w[2] & w[3]) != 0xffffffffu) {
                #pragma unroll
                for (int i = 0; i < 128; i++) if (!((w[i / 32] >> (i % 32)) & 1)) v[i] = -INFINITY;
            }
            float x4[4];
            #pragma unroll
            for (int c = 0; c < 4; c++) {
                x4[c] = fmaxf(v[c], v[c + 4]);
                #pragma unroll
                for (int i = c + 8; i < 128; i += 8) x4[c] = max3(x4[c], v[i], v[i + 4]);
            }
            const float x = fmaxf(fmaxf(x4[0], x4[1]), fmaxf(x4[2], x4[3])) * sc;
            const bool first = m == -INFINITY, grow = !first && x > m + 8.f;
            if (j > 0 && __any_sync(0xffffffffu, grow)) {
                const float f = grow ? ex2_approx(m - x) : 1.f;
                l *= f;
                #pragma unroll 1
                for (int c = 0; c < DH / 16; c++) {
                    float o[16];
                    tmem_ld32x32_x16(to + 16 * c, o);
                    tmem_wait_ld();
                    uint32_t u[16];
                    #pragma unroll
                    for (int i = 0; i < 16; i++) u[i] = __float_as_uint(o[i] * f);
                    tmem_st16(to + 16 * c, u);
                }
            }
            if (first || grow) m = x;
            // a row without a kept key so far shifts by 0 (all its terms are 0)
            const float shift = m == -INFINITY ? 0.f : m;
            const unsigned long long sc2 = splat2(sc), nm2 = splat2(-shift);
            unsigned long long sum2[2] = {0ull, 0ull};
            #pragma unroll
            for (int c = 0; c < 4; c++) {
                uint32_t p[16];
                #pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    float e0, e1;
                    upk2(fma2(pk2(v[c * 32 + i], v[c * 32 + i + 1]), sc2, nm2), e0, e1);
                    e0 = ex2_approx(e0);
                    e1 = ex2_approx(e1);
                    sum2[(i / 2) & 1] = add2(sum2[(i / 2) & 1], pk2(e0, e1));
                    p[i / 2] = pack_bf2(e0, e1);
                }
                tmem_st16(ts + 16 * c, p);                  // over scores that were read
                if (c & 1) {                                // 64 keys' probabilities are there
                    tmem_wait_st();
                    tc_fence_before();
                    bar_arrive(pready + 16 * t + 8 * (c >> 1));
                }
            }
            float s0, s1;
            upk2(add2(sum2[0], sum2[1]), s0, s1);
            l += s0 + s1;
        }
        const int r = r0 + t * 128 + row;
        if (ok && nt > 0) ok = wait_warp(ofull + 8 * t, 0, abort_flag, 9);
        if (ok) {
            tc_fence_after();
            const bool in = r < a.rows;
            const long prow = ((long)at.seq * a.kv_heads + at.hk) * a.rows + r;
            const float inv = l == 0.f ? 0.f : 1.f / l;
            #pragma unroll
            for (int c = 0; c < DH / 32; c++) {
                float o[32];
                if (nt > 0) {
                    tmem_ld32(to + 32 * c, o);
                    tmem_wait_ld();
                } else {
                    #pragma unroll
                    for (int i = 0; i < 32; i++) o[i] = 0.f;
                }
                if (in && a.nsplit > 1) {
                    float4* p = (float4*)(a.part + (prow * a.nsplit + at.part) * DH + 32 * c);
                    #pragma unroll
                    for (int i = 0; i < 8; i++) p[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                } else if (in) {
                    uint4* p = (uint4*)((bf16*)a.out + qrow(a, a.so, at.seq, at.hk, r) + 32 * c);
                    #pragma unroll
                    for (int i = 0; i < 4; i++)
                        p[i] = make_uint4(pack_bf2(o[8 * i] * inv, o[8 * i + 1] * inv), pack_bf2(o[8 * i + 2] * inv, o[8 * i + 3] * inv),
                                          pack_bf2(o[8 * i + 4] * inv, o[8 * i + 5] * inv), pack_bf2(o[8 * i + 6] * inv, o[8 * i + 7] * inv));
                }
            }
            if (in && a.nsplit > 1) a.part_ml[prow * a.nsplit + at.part] = make_float2(m, l);
            else if (in && a.lse) a.lse[prow] = l == 0.f ? -INFINITY : (m + log2f(l)) * LN2;
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 10) tmem_free(tmem);
}

// ----------------------------------------------------------------- backward
// Two kernels, so that every gradient is written by one block in a fixed
// order: dk and dv of a key tile over all rows, and dq of a row tile over all
// keys (S and dP are computed in both: 7 products instead of 5, but no sums
// across blocks).  In both, blocks of 64 of the walked axis alternate between
// two TMEM buffers, each with its own warpgroup, so that one block's products
// run while the other's probabilities are computed; P and dS go to TMEM as
// bf16 (2^-8 of each, as the gradients' own rounding) over the scores and are the
// A operands of the products after them.
// Warps 0-3 and 4-7 compute (a TMEM lane per thread), a lane of warp 8 loads
// by TMA, warp 9 prepares, warp 10 issues the MMAs.
// Bound: the tensor core; a block of 128 x 64 scores takes 1024 clocks of
// products in the first kernel and 768 in the second, 512 of exponentials.
// The rows and keys above: dk and dv 1068 us (1030 TFLOP/s of its own four
// products), dq 757 us (1090 of three); the tensor pipe is busy 62 and 59 %.
constexpr int BB = 64;                       // rows or keys of a block
constexpr int ONE_PER_SM = 120 * 1024;       // shared memory that keeps a second block off the processor

// 64 fp32 values of this lane, 32 columns at a time
PTCG_DEV void tmem_ld64(uint32_t taddr, float (&v)[64]) {
    tmem_ld32(taddr, v);
    tmem_ld32(taddr + 32, v + 32);
    tmem_wait_ld();
}
// x[i] y[i] as bf16, ANDed with `mask`, over 32 columns
template <typename F>
PTCG_DEV void tmem_put64(uint32_t taddr, uint32_t mask, F pair) {
    #pragma unroll
    for (int h = 0; h < 2; h++) {
        uint32_t p[16];
        #pragma unroll
        for (int i = 0; i < 16; i++) p[i] = pair(32 * h + 2 * i) & mask;
        tmem_st16(taddr + 16 * h, p);
    }
    tmem_wait_st();
    tc_fence_before();
}
// 32 columns of an accumulator row to a bf16 (or fp32 part) row, times f; rows
// that are not `live` get zeros
PTCG_DEV void write32(uint32_t taddr, float f, bool live, bool in, bf16* out, float* part) {
    float o[32];
    tmem_ld32(taddr, o);
    tmem_wait_ld();
    #pragma unroll
    for (int i = 0; i < 32; i++) o[i] = live ? o[i] * f : 0.f;
    if (!in) return;
    if (part) {
        #pragma unroll
        for (int i = 0; i < 8; i++) ((float4*)part)[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
    } else {
        #pragma unroll
        for (int i = 0; i < 4; i++)
            ((uint4*)out)[i] = make_uint4(pack_bf2(o[8 * i], o[8 * i + 1]), pack_bf2(o[8 * i + 2], o[8 * i + 3]),
                                          pack_bf2(o[8 * i + 4], o[8 * i + 5]), pack_bf2(o[8 * i + 6], o[8 * i + 7]));
    }
}
// dk, dv of 128 keys (M, a TMEM lane each).  Row blocks are taken per query
// head (TMA fills rows past lq with zeros; their log-sum-exp counts as +inf).
//   S^T = K Q^T, dP^T = V dO^T (N = 64 rows);  dV += P^T dO, dK += dS^T Q
// TMEM: buffer b: S^T at 128 b, dP^T at 128 b + 64; dV at 256, dK at 256 + DH.
template <int DH> struct Dkv {
    using T = Tile<DH, 128>;
    using R = Tile<DH, BB>;
    static constexpr int NS = DH == 128 ? 4 : DH == 64 ? 6 : 8;     // row stages (dout and q)
    // barriers: kvfull full[NS] stat[NS] free[NS] sfull[2] dpfull[2] pready[2] dsready[2] ofull drain
    static constexpr int BARS = 3 * NS + 11;
    static constexpr int BYTES = 1024 + 2 * T::BYTES + 2 * NS * R::BYTES + NS * 2 * BB * 4 + BARS * 8 + 16;
    static constexpr int SMEM = BYTES > ONE_PER_SM ? BYTES : ONE_PER_SM;
    static constexpr int THREADS = 384;
};

template <int DH>
__global__ void __launch_bounds__(Dkv<DH>::THREADS, 1) k_cross_dkv_tc(
        const __grid_constant__ CrossArgs a, const __grid_constant__ RowMap kmap,
        const __grid_constant__ RowMap vmap, const __grid_constant__ RowMap qmap,
        const __grid_constant__ RowMap gmap, FastDiv by_blocks) {
    using F = Dkv<DH>;
    using T = typename F::T;
    using R = typename F::R;
    constexpr int NS = F::NS;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const uint32_t sK = s_addr(smem), sV = sK + T::BYTES, sQ = sV + T::BYTES, sG = sQ + NS * R::BYTES;
    float* stats = (float*)(smem + 2 * T::BYTES + 2 * NS * R::BYTES);  // [NS][-lse2 | -delta][64]
    uint64_t* bars = (uint64_t*)(stats + NS * 2 * BB);
    const uint32_t kvfull = s_addr(bars), full = kvfull + 8, stat = full + 8 * NS, free_ = stat + 8 * NS,
                   sfull = free_ + 8 * NS, dpfull = sfull + 16, pready = dpfull + 16,
                   dsready = pready + 16, ofull = dsready + 16, drain = ofull + 8;
    uint32_t* tmem_slot = (uint32_t*)(bars + F::BARS);
    volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Where at = where(a);
    const int j0 = at.tile * 128, len = kept_len(a, at.seq);
    // the row blocks of this part: block n is rows 64 (n % per head) .. of head n / per head
    const int n0 = at.part * (a.split / BB), n1 = min((int)by_blocks.d * a.group, n0 + a.split / BB);
    KeyBits<4> kb;
    kb.fetch(a, at.seq, j0, a.lk, len, lane);
    uint32_t w[4];
    kb.words(w);
    const int nb = (w[0] | w[1] | w[2] | w[3]) ? n1 - n0 : 0;           // nothing to add for masked keys
    if (threadIdx.x == 0) {
        bar_init(kvfull, 1);
        for (int i = 0; i < NS; i++) { bar_init(full + 8 * i, 1); bar_init(stat + 8 * i, 1); bar_init(free_ + 8 * i, 1); }
        for (int b = 0; b < 2; b++) {
            bar_init(sfull + 8 * b, 1); bar_init(dpfull + 8 * b, 1);
            bar_init(pready + 8 * b, 128); bar_init(dsready + 8 * b, 128);
        }
        bar_init(ofull, 1);
        bar_init(drain, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async();
    }
    if (warp == 10) tmem_alloc(tmem_slot);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    if (warp == 8) {
        // ------------------------------------------------- TMA lane
        if (lane == 0 && nb > 0) {
            bar_expect_tx(kvfull, 2 * T::BYTES);
            load_rows<DH, 128>(sK, kmap, kvfull, j0, at.hk, at.seq);
            load_rows<DH, 128>(sV, vmap, kvfull, j0, at.hk, at.seq);
            int n = 0;
            for (; n < nb; n++) {
                const int s = n % NS, g = by_blocks.div(n0 + n), i0 = (n0 + n - g * by_blocks.d) * BB;
                if (!wait_bar(free_ + 8 * s, (uint32_t)(((n / NS) & 1) ^ 1), abort_flag, 11)) break;
                bar_expect_tx(full + 8 * s, 2 * R::BYTES);
                load_rows<DH, BB>(sQ + s * R::BYTES, qmap, full + 8 * s, i0, at.hk * a.group + g, at.seq);
                load_rows<DH, BB>(sG + s * R::BYTES, gmap, full + 8 * s, i0, at.hk * a.group + g, at.seq);
            }
            if (*abort_flag) {                       // copies still in flight land before the exit
                bar_drain(kvfull, 0);
                for (int i = max(0, n - NS); i < n; i++) bar_drain(full + 8 * (i % NS), (i / NS) & 1);
            }
        }
        __syncwarp();
    } else if (warp == 9) {
        // -------------------------------- log-sum-exp and delta of each block
        for (int n = 0; n < nb; n++) {
            const int s = n % NS, g = by_blocks.div(n0 + n), i0 = (n0 + n - g * by_blocks.d) * BB;
            const long base = ((long)at.seq * a.heads + at.hk * a.group + g) * a.lq;
            float x[2], d[2];
            #pragma unroll
            for (int e = 0; e < 2; e++) {
                const int i = i0 + 32 * e + lane;
                const float v = i < a.lq ? a.lse[base + i] : -INFINITY;
                x[e] = v == -INFINITY ? -INFINITY : -v * LOG2E;
                d[e] = i < a.lq ? -a.delta[base + i] : 0.f;
            }
            if (!wait_warp(free_ + 8 * s, (uint32_t)(((n / NS) & 1) ^ 1), abort_flag, 12)) break;
            #pragma unroll
            for (int e = 0; e < 2; e++) {
                stats[s * 2 * BB + 32 * e + lane] = x[e];
                stats[s * 2 * BB + BB + 32 * e + lane] = d[e];
            }
            __syncwarp();
            if (lane == 0) bar_arrive(stat + 8 * s);
        }
    } else if (warp >= 10) {
        // ---------------------------------------------------- MMA warp
        if (warp == 10 && nb > 0) {
            const uint32_t ids = idesc_bf16(BB, 0, 0), ido = idesc_bf16(DH, 0, 1);
            const uint32_t klo = T::lo_k(sK), vlo = T::lo_k(sV);
            const uint32_t qk = R::lo_k(sQ), gk = R::lo_k(sG), qm = R::lo_mn(sQ), gm = R::lo_mn(sG);
            bool ok = wait_warp(kvfull, 0, abort_flag, 13);
            int s_in = 0, s_out = 0;                 // stages of the next scores and of the next sums
            uint32_t p_in = 0;
            for (int n = -2; ok && n < nb; n++) {
                const int b = n & 1;                 // buffer of blocks n and n + 2
                const bool more = n + 2 < nb;
                if (more) ok = wait_warp(full + 8 * s_in, p_in, abort_flag, 14);
                const uint32_t off_in = (s_in * R::BYTES) >> 4, off_out = (s_out * R::BYTES) >> 4;
                if (n >= 0) {
                    ok = ok && wait_warp(pready + 8 * b, (n >> 1) & 1, abort_flag, 15);
                    tc_fence_after();
                    if (ok && elect_one()) {
                        #pragma unroll
                        for (int s = 0; s < BB / 16; s++)
                            mma_bf16_ts(tmem + 256, tmem + 128 * b + 8 * s, R::mnmajor(gm + off_out, s), ido, s > 0 ? 1u : n > 0);
                    }
                    __syncwarp();
                    ok = ok && wait_warp(dsready + 8 * b, (n >> 1) & 1, abort_flag, 16);
                }
                tc_fence_after();
                if (ok && elect_one()) {
                    if (n >= 0) {
                        #pragma unroll
                        for (int s = 0; s < BB / 16; s++)
                            mma_bf16_ts(tmem + 256 + DH, tmem + 128 * b + 64 + 8 * s, R::mnmajor(qm + off_out, s), ido, s > 0 ? 1u : n > 0);
                        mma_commit_to(free_ + 8 * s_out);
                        if (n == nb - 1) mma_commit_to(ofull);
                    }
                    if (more) {
                        #pragma unroll
                        for (int s = 0; s < DH / 16; s++)
                            mma_bf16(tmem + 128 * b, T::kmajor(klo, s), R::kmajor(qk + off_in, s), ids, s > 0);
                        mma_commit_to(sfull + 8 * b);
                        #pragma unroll
                        for (int s = 0; s < DH / 16; s++)
                            mma_bf16(tmem + 128 * b + 64, T::kmajor(vlo, s), R::kmajor(gk + off_in, s), ids, s > 0);
                        mma_commit_to(dpfull + 8 * b);
                    }
                }
                __syncwarp();
                if (more && ++s_in == NS) { s_in = 0; p_in ^= 1; }
                if (n >= 0 && ++s_out == NS) s_out = 0;
            }
            // no MMA may still be in flight when TMEM is released
            if (elect_one()) {
                mma_commit_to(drain);
                bar_drain(drain, 0);
            }
            __syncwarp();
        }
    } else {
        // ------------------------------------------------ P^T and dS^T
        const int b = warp >> 2, quad = warp & 3, row = quad * 32 + lane;
        const uint32_t lane_off = (uint32_t)(quad * 32) << 16, tb = tmem + lane_off + 128 * b;
        const bool live = ((quad < 2 ? (quad ? w[1] : w[0]) : (quad == 2 ? w[2] : w[3])) >> lane) & 1;
        const uint32_t mask = live ? 0xffffffffu : 0u;
        const unsigned long long sc2 = splat2(a.scale * LOG2E);
        bool ok = true;
        for (int n = b; ok && n < nb; n += 2) {
            const uint32_t ph = (n >> 1) & 1;
            const float* nl = stats + (n % NS) * 2 * BB;
            const float* nd = nl + BB;
            ok = wait_warp(stat + 8 * (n % NS), (n / NS) & 1, abort_flag, 17) && wait_warp(sfull + 8 * b, ph, abort_flag, 18);
            if (!ok) break;
            tc_fence_after();
            float v[64];
            tmem_ld64(tb, v);
            #pragma unroll
            for (int i = 0; i < 64; i += 4) {
                const ulonglong2 l = *reinterpret_cast<const ulonglong2*>(nl + i);
                upk2(fma2(pk2(v[i], v[i + 1]), sc2, l.x), v[i], v[i + 1]);
                upk2(fma2(pk2(v[i + 2], v[i + 3]), sc2, l.y), v[i + 2], v[i + 3]);
                #pragma unroll
                for (int e = 0; e < 4; e++) v[i + e] = ex2_approx(v[i + e]);
            }
            tmem_put64(tb, mask, [&](int i) { return pack_bf2(v[i], v[i + 1]); });
            bar_arrive(pready + 8 * b);
            ok = wait_warp(dpfull + 8 * b, ph, abort_flag, 19);
            if (!ok) break;
            tc_fence_after();
            #pragma unroll
            for (int h = 0; h < 2; h++) {
                float d[32];
                tmem_ld32(tb + 64 + 32 * h, d);
                tmem_wait_ld();
                #pragma unroll
                for (int i = 0; i < 32; i += 4) {
                    const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(nd + 32 * h + i);
                    float* e = v + 32 * h + i;
                    upk2(mul2(pk2(e[0], e[1]), add2(pk2(d[i], d[i + 1]), x.x)), e[0], e[1]);
                    upk2(mul2(pk2(e[2], e[3]), add2(pk2(d[i + 2], d[i + 3]), x.y)), e[2], e[3]);
                }
            }
            tmem_put64(tb + 64, mask, [&](int i) { return pack_bf2(v[i], v[i + 1]); });
            bar_arrive(dsready + 8 * b);
        }
        if (ok && nb > 0) ok = wait_warp(ofull, 0, abort_flag, 20);
        if (ok) {
            tc_fence_after();
            // warpgroup 0 writes dv, warpgroup 1 dk
            const int j = j0 + row;
            const bool in = j < a.lk;
            const long prow = (((long)at.seq * a.kv_heads + at.hk) * a.lk + j) * a.nsplit + at.part;
            const long orow = in ? krow(b ? a.sdk : a.sdv, at.seq, at.hk, j) : 0;
            bf16* out = (bf16*)(b ? a.dk : a.dv) + orow;
            float* part = a.nsplit > 1 ? (b ? a.part : a.part2) + prow * DH : nullptr;
            #pragma unroll
            for (int c = 0; c < DH / 32; c++)
                write32(tmem + lane_off + 256 + b * DH + 32 * c, b ? a.scale : 1.f, live && nb > 0, in,
                        out + 32 * c, part ? part + 32 * c : nullptr);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 10) tmem_free(tmem);
}

// dq of 128 stacked rows (M, a TMEM lane each), which hold q and dout in TMEM:
//   S = Q K^T, dP = dO V^T (A from TMEM, N = 64 keys);  dQ += dS K
// also delta = dout . out, for the kernel above.  K rows of masked keys are
// zeroed in shared memory (dS = 0 there, but 0 * NaN is NaN).
// TMEM: dQ at 0, buffer b: S at 128 + 128 b, dP 64 on; q at 384, dout at 448.
template <int DH> struct Dq {
    using R = Tile<DH, BB>;
    static constexpr int NS = DH == 128 ? 5 : 8;                    // key stages (K and V)
    // barriers: qfull kfull[NS] kready[NS] vfull[NS] free[NS] sfull[2] dpfull[2] dsready[2] ofull drain
    static constexpr int BARS = 4 * NS + 9;
    static constexpr int BYTES = 1024 + 2 * NS * R::BYTES + 2 * 128 * 4 + BARS * 8 + 16;
    static constexpr int SMEM = BYTES > ONE_PER_SM ? BYTES : ONE_PER_SM;
    static constexpr int THREADS = 384;
};

template <int DH>
__global__ void __launch_bounds__(Dq<DH>::THREADS, 1) k_cross_dq_tc(
        const __grid_constant__ CrossArgs a, const __grid_constant__ RowMap kmap,
        const __grid_constant__ RowMap vmap) {
    using F = Dq<DH>;
    using R = typename F::R;
    constexpr int NS = F::NS;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const uint32_t sK = s_addr(smem), sV = sK + NS * R::BYTES;
    float* s_lse = (float*)(smem + 2 * NS * R::BYTES);               // [128] -lse2, [128] -delta
    float* s_delta = s_lse + 128;
    uint64_t* bars = (uint64_t*)(s_delta + 128);
    const uint32_t qfull = s_addr(bars), kfull = qfull + 8, kready = kfull + 8 * NS, vfull = kready + 8 * NS,
                   free_ = vfull + 8 * NS, sfull = free_ + 8 * NS, dpfull = sfull + 16,
                   dsready = dpfull + 16, ofull = dsready + 16, drain = ofull + 8;
    uint32_t* tmem_slot = (uint32_t*)(bars + F::BARS);
    volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Where at = where(a);
    const int r0 = at.tile * 128, len = kept_len(a, at.seq);
    const int kbeg = min(at.part * a.split, len), kend = min(len, kbeg + a.split);
    const int nb = (kend - kbeg + BB - 1) / BB;
    if (threadIdx.x == 0) {
        bar_init(qfull, 256);
        for (int i = 0; i < NS; i++) {
            bar_init(kfull + 8 * i, 1); bar_init(kready + 8 * i, 1);
            bar_init(vfull + 8 * i, 1); bar_init(free_ + 8 * i, 1);
        }
        for (int b = 0; b < 2; b++) {
            bar_init(sfull + 8 * b, 1); bar_init(dpfull + 8 * b, 1); bar_init(dsready + 8 * b, 128);
        }
        bar_init(ofull, 1);
        bar_init(drain, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async();
    }
    if (warp == 10) tmem_alloc(tmem_slot);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    if (warp == 8) {
        // ------------------------------------------------- TMA lane
        if (lane == 0) {
            int n = 0;
            for (; n < nb; n++) {
                const int s = n % NS;
                if (!wait_bar(free_ + 8 * s, (uint32_t)(((n / NS) & 1) ^ 1), abort_flag, 31)) break;
                bar_expect_tx(kfull + 8 * s, R::BYTES);
                load_rows<DH, BB>(sK + s * R::BYTES, kmap, kfull + 8 * s, kbeg + n * BB, at.hk, at.seq);
                bar_expect_tx(vfull + 8 * s, R::BYTES);
                load_rows<DH, BB>(sV + s * R::BYTES, vmap, vfull + 8 * s, kbeg + n * BB, at.hk, at.seq);
            }
            if (*abort_flag)                         // copies still in flight land before the exit
                for (int i = max(0, n - NS); i < n; i++) {
                    bar_drain(kfull + 8 * (i % NS), (i / NS) & 1);
                    bar_drain(vfull + 8 * (i % NS), (i / NS) & 1);
                }
        }
        __syncwarp();
    } else if (warp == 9) {
        // ------------------------------------ masked rows of K become zeros
        KeyBits<2> kb;
        kb.fetch(a, at.seq, kbeg, kend, len, lane);
        for (int n = 0; n < nb; n++) {
            uint32_t w[2];
            kb.words(w);
            kb.fetch(a, at.seq, kbeg + (n + 1) * BB, kend, len, lane);
            const int s = n % NS;
            if (!wait_warp(kfull + 8 * s, (n / NS) & 1, abort_flag, 32)) break;
            if ((w[0] & w[1]) != 0xffffffffu) {
                clear_rows<DH, BB>(smem + s * R::BYTES, w, lane);
                fence_async();
                __syncwarp();
            }
            if (lane == 0) bar_arrive(kready + 8 * s);
        }
    } else if (warp >= 10) {
        // ---------------------------------------------------- MMA warp
        if (warp == 10 && nb > 0) {
            const uint32_t ids = idesc_bf16(BB, 0, 0), ido = idesc_bf16(DH, 0, 1);
            const uint32_t kk = R::lo_k(sK), vk = R::lo_k(sV), km = R::lo_mn(sK);
            bool ok = wait_warp(qfull, 0, abort_flag, 33);
            int s_in = 0, s_out = 0;
            uint32_t p_in = 0;
            for (int n = -2; ok && n < nb; n++) {
                const int b = n & 1;
                const bool more = n + 2 < nb;
                if (more) ok = wait_warp(kready + 8 * s_in, p_in, abort_flag, 34) && wait_warp(vfull + 8 * s_in, p_in, abort_flag, 35);
                const uint32_t off_in = (s_in * R::BYTES) >> 4, off_out = (s_out * R::BYTES) >> 4;
                const uint32_t tb = tmem + 128 + 128 * b;
                if (n >= 0) ok = ok && wait_warp(dsready + 8 * b, (n >> 1) & 1, abort_flag, 36);
                tc_fence_after();
                if (ok && elect_one()) {
                    if (n >= 0) {
                        #pragma unroll
                        for (int s = 0; s < BB / 16; s++)
                            mma_bf16_ts(tmem, tb + 8 * s, R::mnmajor(km + off_out, s), ido, s > 0 ? 1u : n > 0);
                        mma_commit_to(free_ + 8 * s_out);
                        if (n == nb - 1) mma_commit_to(ofull);
                    }
                    if (more) {
                        #pragma unroll
                        for (int s = 0; s < DH / 16; s++)
                            mma_bf16_ts(tb, tmem + 384 + 8 * s, R::kmajor(kk + off_in, s), ids, s > 0);
                        mma_commit_to(sfull + 8 * b);
                        #pragma unroll
                        for (int s = 0; s < DH / 16; s++)
                            mma_bf16_ts(tb + 64, tmem + 448 + 8 * s, R::kmajor(vk + off_in, s), ids, s > 0);
                        mma_commit_to(dpfull + 8 * b);
                    }
                }
                __syncwarp();
                if (more && ++s_in == NS) { s_in = 0; p_in ^= 1; }
                if (n >= 0 && ++s_out == NS) s_out = 0;
            }
            if (elect_one()) {
                mma_commit_to(drain);
                bar_drain(drain, 0);
            }
            __syncwarp();
        }
    } else {
        // ------------------------------------------------------------ dS
        const int b = warp >> 2, quad = warp & 3, row = quad * 32 + lane, r = r0 + row;
        const uint32_t lane_off = (uint32_t)(quad * 32) << 16, tb = tmem + lane_off + 128 + 128 * b;
        const bool in = r < a.rows;
        const long row0 = ((long)at.seq * a.kv_heads + at.hk) * a.rows + r;
        {   // warpgroup 0 brings q to TMEM, warpgroup 1 dout, and both make the row's numbers
            const uint4* src = (const uint4*)((const bf16*)(b ? a.dout : a.q) + (in ? qrow(a, b ? a.sdo : a.sq, at.seq, at.hk, r) : 0));
            const uint4* og = (const uint4*)((const bf16*)a.o + (in ? qrow(a, a.so, at.seq, at.hk, r) : 0));
            float d = 0.f;
            #pragma unroll
            for (int c = 0; c < DH / 32; c++) {
                uint32_t p[16];
                #pragma unroll
                for (int q = 0; q < 4; q++) {
                    const uint4 x = in ? src[4 * c + q] : make_uint4(0u, 0u, 0u, 0u);
                    p[4 * q] = x.x; p[4 * q + 1] = x.y; p[4 * q + 2] = x.z; p[4 * q + 3] = x.w;
                    if (b == 1 && in) {
                        const uint4 y = og[4 * c + q];
                        const uint32_t u[4] = {y.x, y.y, y.z, y.w};
                        #pragma unroll
                        for (int e = 0; e < 4; e++) {
                            float x0, x1, y0, y1;
                            unpack_bf2(p[4 * q + e], x0, x1);
                            unpack_bf2(u[e], y0, y1);
                            d = fmaf(x0, y0, fmaf(x1, y1, d));
                        }
                    }
                }
                tmem_st16(tmem + lane_off + (b ? 448 : 384) + 16 * c, p);
            }
            if (b == 1) {
                s_delta[row] = -d;
                if (in && at.part == 0) a.delta[row0] = d;
            } else {
                const float x = in ? a.lse[row0] : -INFINITY;
                s_lse[row] = x == -INFINITY ? -INFINITY : -x * LOG2E;
            }
            tmem_wait_st();
            tc_fence_before();
            bar_arrive(qfull);
            asm volatile("bar.sync 1, 256;" ::: "memory");
        }
        const unsigned long long sc2 = splat2(a.scale * LOG2E), nl2 = splat2(s_lse[row]), nd2 = splat2(s_delta[row]);
        bool ok = true;
        KeyBits<2> kb;
        kb.fetch(a, at.seq, kbeg + b * BB, kend, len, lane);
        for (int n = b; ok && n < nb; n += 2) {
            const uint32_t ph = (n >> 1) & 1;
            uint32_t w[2];
            kb.words(w);
            kb.fetch(a, at.seq, kbeg + (n + 2) * BB, kend, len, lane);
            ok = wait_warp(sfull + 8 * b, ph, abort_flag, 37);
            if (!ok) break;
            tc_fence_after();
            float v[64];
            tmem_ld64(tb, v);
            #pragma unroll
            for (int i = 0; i < 64; i += 2) {
                upk2(fma2(pk2(v[i], v[i + 1]), sc2, nl2), v[i], v[i + 1]);
                v[i] = ex2_approx(v[i]);
                v[i + 1] = ex2_approx(v[i + 1]);
            }
            ok = wait_warp(dpfull + 8 * b, ph, abort_flag, 38);
            if (!ok) break;
            tc_fence_after();
            #pragma unroll
            for (int h = 0; h < 2; h++) {
                float d[32];
                tmem_ld32(tb + 64 + 32 * h, d);
                tmem_wait_ld();
                #pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    float* e = v + 32 * h + i;
                    upk2(mul2(pk2(e[0], e[1]), add2(pk2(d[i], d[i + 1]), nd2)), e[0], e[1]);
                }
                if (w[h] != 0xffffffffu) {
                    #pragma unroll
                    for (int i = 0; i < 32; i++) if (!((w[h] >> i) & 1)) v[32 * h + i] = 0.f;
                }
            }
            tmem_put64(tb, 0xffffffffu, [&](int i) { return pack_bf2(v[i], v[i + 1]); });
            bar_arrive(dsready + 8 * b);
        }
        if (ok && nb > 0) ok = wait_warp(ofull, 0, abort_flag, 39);
        if (ok) {
            tc_fence_after();
            // 32-column pieces of dq, in turn to the two warpgroups
            bf16* out = (bf16*)a.dq + (in ? qrow(a, a.sdq, at.seq, at.hk, r) : 0);
            float* part = a.nsplit > 1 ? a.part + (row0 * a.nsplit + at.part) * DH : nullptr;
            #pragma unroll
            for (int c = 0; c < DH / 32; c++)
                if ((c & 1) == b)
                    write32(tmem + lane_off + 32 * c, a.scale, nb > 0, in, out + 32 * c, part ? part + 32 * c : nullptr);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 10) tmem_free(tmem);
}

// ------------------------------------------------------------------- host
// the map of a tensor with `rows` rows and `heads` heads, or false
template <int DH>
bool row_map(RowMap* m, const void* p, const PtcgHeads& s, long rows, int heads, int nseq, int box_rows) {
    m->seqs = s.seq != 0;
    m->heads = s.head != 0;
    const long dims[4] = {DH, rows, m->heads ? heads : 1, m->seqs ? nseq : 1};
    // a dimension of one entry may have any stride
    const long strides[3] = {rows > 1 ? s.row : DH, dims[2] > 1 ? s.head : DH, dims[3] > 1 ? s.seq : DH};
    for (long x : strides)
        if (x <= 0) return false;
    const int rowb = Tile<DH, 128>::ROWB;
    return tc_make_map_4d(&m->map, p, dims, strides, rowb / 2, box_rows, rowb);
}
template <typename F>
cudaError_t smem_limit(F f, int bytes) {
    return cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

template <int DH>
cudaError_t launch_fwd(const CrossArgs& a, long blocks, cudaStream_t s, bool* taken) {
    RowMap km, vm;
    *taken = row_map<DH>(&km, a.k, a.sk, a.lk, a.kv_heads, a.nseq, 128) &&
             row_map<DH>(&vm, a.v, a.sv, a.lk, a.kv_heads, a.nseq, 128);
    if (!*taken) return cudaSuccess;
    const cudaError_t e = smem_limit(k_cross_fwd_tc<DH>, Fwd<DH>::SMEM);
    if (e != cudaSuccess) return e;
    ++g_ptcg_launches, k_cross_fwd_tc<DH><<<(unsigned)blocks, Fwd<DH>::THREADS, Fwd<DH>::SMEM, s>>>(a, km, vm);
    return cudaSuccess;
}
template <int DH>
cudaError_t launch_dq(const CrossArgs& a, long blocks, cudaStream_t s, bool* taken) {
    RowMap km, vm;
    *taken = row_map<DH>(&km, a.k, a.sk, a.lk, a.kv_heads, a.nseq, BB) &&
             row_map<DH>(&vm, a.v, a.sv, a.lk, a.kv_heads, a.nseq, BB);
    if (!*taken) return cudaSuccess;
    const cudaError_t e = smem_limit(k_cross_dq_tc<DH>, Dq<DH>::SMEM);
    if (e != cudaSuccess) return e;
    ++g_ptcg_launches, k_cross_dq_tc<DH><<<(unsigned)blocks, Dq<DH>::THREADS, Dq<DH>::SMEM, s>>>(a, km, vm);
    return cudaSuccess;
}
template <int DH>
cudaError_t launch_dkv(const CrossArgs& a, long blocks, cudaStream_t s, bool* taken) {
    RowMap km, vm, qm, gm;
    *taken = row_map<DH>(&km, a.k, a.sk, a.lk, a.kv_heads, a.nseq, 128) &&
             row_map<DH>(&vm, a.v, a.sv, a.lk, a.kv_heads, a.nseq, 128) &&
             row_map<DH>(&qm, a.q, a.sq, a.lq, a.heads, a.nseq, BB) &&
             row_map<DH>(&gm, a.dout, a.sdo, a.lq, a.heads, a.nseq, BB);
    if (!*taken) return cudaSuccess;
    const cudaError_t e = smem_limit(k_cross_dkv_tc<DH>, Dkv<DH>::SMEM);
    if (e != cudaSuccess) return e;
    ++g_ptcg_launches, k_cross_dkv_tc<DH><<<(unsigned)blocks, Dkv<DH>::THREADS, Dkv<DH>::SMEM, s>>>(
        a, km, vm, qm, gm, fast_div((a.lq + BB - 1) / BB));
    return cudaSuccess;
}

}  // namespace

namespace cross {

#define BY_DH(F) (dh == 32 ? F<32>(a, blocks, s, taken) : dh == 64 ? F<64>(a, blocks, s, taken) : F<128>(a, blocks, s, taken))
cudaError_t fwd_tc(int dh, const CrossArgs& a, long blocks, cudaStream_t s, bool* taken) { return BY_DH(launch_fwd); }
cudaError_t dq_tc(int dh, const CrossArgs& a, long blocks, cudaStream_t s, bool* taken) { return BY_DH(launch_dq); }
cudaError_t dkv_tc(int dh, const CrossArgs& a, long blocks, cudaStream_t s, bool* taken) { return BY_DH(launch_dkv); }
#undef BY_DH

}  // namespace cross

int cross_tc_error_read_reset() {
    int v = 0, zero = 0;
    cudaMemcpyFromSymbol(&v, g_cross_tc_error, sizeof(int));
    cudaMemcpyToSymbol(g_cross_tc_error, &zero, sizeof(int));
    return v;
}
