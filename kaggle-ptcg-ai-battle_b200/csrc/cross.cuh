// What the cross-attention kernels share: the launch arguments, the addresses
// of stacked query rows and key rows, the key masks and asynchronous copies.
#pragma once
#include "vec.cuh"

namespace cross {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// n / d for 0 <= n < 2^31 as a multiply-high, an add and a shift: with
// 2^(l-1) < d <= 2^l and mul = floor(2^32 (2^l - d) / d) + 1, the quotient is
// (mulhi(n, mul) + n) >> l (the divisions by sizes known only at the launch
// were a sixth of the short problems' instructions)
struct FastDiv {
    unsigned mul, shift, d;
    PTCG_DEV unsigned div(unsigned n) const { return (__umulhi(n, mul) + n) >> shift; }
};
inline FastDiv fast_div(unsigned d) {
    FastDiv f = {0, 0, d};
    while ((1ull << f.shift) < d) f.shift++;
    f.mul = (unsigned)(((1ull << 32) * ((1ull << f.shift) - d)) / d + 1);
    return f;
}

struct CrossArgs {
    const void *q, *k, *v, *o, *dout;
    const uint8_t* keep;
    const int* kv_len;
    void *out, *dq, *dk, *dv;
    float *lse, *delta;
    // split work: fp32 partial rows and, in the forward, their (max, sum)
    float *part, *part2;
    float2* part_ml;
    PtcgHeads sq, sk, sv, so, sdo, sdq, sdk, sdv;
    int nseq, lq, lk, heads, kv_heads, group, rows;      // rows = group * lq
    int tiles, nsplit, split;                      // `split` rows of the split axis per part
    int want;                                      // or even parts (below), at most so many per key head
    FastDiv by_lq, by_tiles, by_nsplit, by_kv;
    float scale;
};

// element offset of stacked row r of key head hk in a query-like tensor
PTCG_DEV long qrow(const CrossArgs& a, const PtcgHeads& s, int seq, int hk, int r) {
    const int g = a.by_lq.div(r);
    return seq * s.seq + (r - g * a.lq) * s.row + (long)(hk * a.group + g) * s.head;
}
PTCG_DEV long krow(const PtcgHeads& s, int seq, int hk, int j) {
    return seq * s.seq + j * s.row + hk * s.head;
}
PTCG_DEV int kept_len(const CrossArgs& a, int seq) {
    return a.kv_len ? min(max(a.kv_len[seq], 0), a.lk) : a.lk;
}
PTCG_DEV bool kept(const CrossArgs& a, int seq, int j, int len) {
    return j < len && (!a.keep || a.keep[(long)seq * a.lk + j] != 0);
}
// block index -> (tile of the problem, part of the split axis, key head, sequence)
struct Where { int tile, part, hk, seq; };
PTCG_DEV Where where(const CrossArgs& a) {
    Where w;
    const unsigned b = blockIdx.x, c = a.by_tiles.div(b), d = a.by_nsplit.div(c), e = a.by_kv.div(d);
    w.tile = b - c * a.by_tiles.d;
    w.part = c - d * a.by_nsplit.d;
    w.hk = d - e * a.by_kv.d;
    w.seq = e;
    return w;
}

// Even parts: caches of unequal length (kv_len) as at most `want` parts of one
// length, so that all blocks run at once and end together.  Parts of a fixed
// share of lk left processors idle behind the longest caches (8 caches of 12653
// to 65181 keys, 4 key heads of width 128: 162 us, 120 in even parts).  The length is the
// smallest multiple of 256 keys that gives no more parts; every warp works it
// out from the lengths, which are known on the device only.
constexpr int EVEN_KEYS = 256;
PTCG_DEV unsigned even_units(const CrossArgs& a, int seq) {
    return ((unsigned)kept_len(a, seq) + EVEN_KEYS - 1) / EVEN_KEYS;
}
PTCG_DEV unsigned warp_sum_u(unsigned v) {
    #pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
PTCG_DEV unsigned even_length(const CrossArgs& a) {      // in units
    const int lane = threadIdx.x & 31;
    const unsigned want = a.want;
    unsigned all = 0;                                    // at most 2^22 units of each of 296 sequences
    for (int s = lane; s < a.nseq; s += 32) all += even_units(a, s);
    all = warp_sum_u(all);
    unsigned lo = max((all + want - 1) / want, 1u), hi = max(all / (want - a.nseq) + 1, lo);
    while (lo < hi) {
        const unsigned mid = (lo + hi) / 2;
        unsigned n = 0;
        for (int s = lane; s < a.nseq; s += 32) n += (even_units(a, s) + mid - 1) / mid;
        if (warp_sum_u(n) <= want) hi = mid; else lo = mid + 1;
    }
    return lo;
}
// this block's part, and its keys; false: no part is left for it
PTCG_DEV bool even_part(const CrossArgs& a, Where& w, int& kbeg, int& kend) {
    const int lane = threadIdx.x & 31;
    const unsigned len = even_length(a), i = a.by_kv.div(blockIdx.x);
    unsigned base = 0;
    for (int s0 = 0; s0 < a.nseq; s0 += 32) {
        const unsigned n = s0 + lane < a.nseq ? (even_units(a, s0 + lane) + len - 1) / len : 0;
        unsigned x = n;
        #pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        const unsigned m = __ballot_sync(0xffffffffu, i < base + x);
        if (m) {
            const int at = __ffs(m) - 1;
            w.tile = 0;
            w.hk = blockIdx.x - i * a.by_kv.d;
            w.seq = s0 + at;
            w.part = i - base - __shfl_sync(0xffffffffu, x - n, at);
            const int keys = kept_len(a, w.seq), step = (int)len * EVEN_KEYS;
            kbeg = w.part * step;
            kend = keys - kbeg < step ? keys : kbeg + step;
            return true;
        }
        base += __shfl_sync(0xffffffffu, x, 31);
    }
    return false;
}

PTCG_DEV uint32_t s_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
PTCG_DEV void cp16(uint32_t dst, const void* src, bool take) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                 :: "r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}
PTCG_DEV void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> PTCG_DEV void cp_wait() { asm volatile("cp.async.wait_group %0;" :: "n"(N) : "memory"); }

// tcgen05 kernels (cross_attention_tc.cu), bf16, over `blocks` blocks: the
// forward in tiles of 256 stacked rows, dq in tiles of 128 stacked rows (and
// delta), dk and dv in tiles of 128 keys, whose split is in 64-row blocks of
// one query head.  *taken = false: strides that TMA does not address; nothing ran
constexpr int TC_ROWS = 256, TC_TILE = 128, TC_BLOCK = 64;
cudaError_t fwd_tc(int dh, const CrossArgs& a, long blocks, cudaStream_t s, bool* taken);
cudaError_t dq_tc(int dh, const CrossArgs& a, long blocks, cudaStream_t s, bool* taken);
cudaError_t dkv_tc(int dh, const CrossArgs& a, long blocks, cudaStream_t s, bool* taken);

}  // namespace cross
