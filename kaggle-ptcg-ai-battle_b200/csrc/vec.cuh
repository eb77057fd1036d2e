// Row access in vectors of V consecutive elements, converted to and from
// fp32, and the argument checks shared by the decoder operators (embedding,
// layer norm, cross attention).
#pragma once
#include "common.cuh"
#include "internal.h"
#include "ptcg_b200.h"

#define OP_REQ(cond, code, ...) do { if (!(cond)) { set_err(__VA_ARGS__); return code; } } while (0)
#define OP_CK(x) do { cudaError_t _e = (x); if (_e != cudaSuccess) { \
    set_err("%s failed: %s (%s:%d)", #x, cudaGetErrorString(_e), __FILE__, __LINE__); \
    return PTCG_ECUDA; } } while (0)
#define OP_CKL() OP_CK(cudaGetLastError())

template <typename T, int V> struct VecIO;
template <> struct VecIO<float, 1> {
    static PTCG_DEV void ld(float (&v)[1], const float* p) { v[0] = *p; }
    static PTCG_DEV void st(float* p, const float (&v)[1]) { *p = v[0]; }
};
template <> struct VecIO<bf16, 1> {
    static PTCG_DEV void ld(float (&v)[1], const bf16* p) { v[0] = __bfloat162float(*p); }
    static PTCG_DEV void st(bf16* p, const float (&v)[1]) { *p = __float2bfloat16_rn(v[0]); }
};
template <> struct VecIO<float, 4> {
    static PTCG_DEV void ld(float (&v)[4], const float* p) {
        const float4 a = *reinterpret_cast<const float4*>(p);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    }
    static PTCG_DEV void st(float* p, const float (&v)[4]) {
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    }
};
PTCG_DEV void unpack_bf2(uint32_t u, float& a, float& b) {
    a = __uint_as_float(u << 16);
    b = __uint_as_float(u & 0xffff0000u);
}
PTCG_DEV uint32_t pack_bf2(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <> struct VecIO<bf16, 4> {
    static PTCG_DEV void ld(float (&v)[4], const bf16* p) {
        const uint2 u = *reinterpret_cast<const uint2*>(p);
        unpack_bf2(u.x, v[0], v[1]);
        unpack_bf2(u.y, v[2], v[3]);
    }
    static PTCG_DEV void st(bf16* p, const float (&v)[4]) {
        *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]));
    }
};
template <> struct VecIO<float, 8> {
    static PTCG_DEV void ld(float (&v)[8], const float* p) {
        const float4 a = *reinterpret_cast<const float4*>(p);
        const float4 b = *reinterpret_cast<const float4*>(p + 4);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
    static PTCG_DEV void st(float* p, const float (&v)[8]) {
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
    }
};
template <> struct VecIO<bf16, 8> {
    static PTCG_DEV void ld(float (&v)[8], const bf16* p) {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        unpack_bf2(u.x, v[0], v[1]);
        unpack_bf2(u.y, v[2], v[3]);
        unpack_bf2(u.z, v[4], v[5]);
        unpack_bf2(u.w, v[6], v[7]);
    }
    static PTCG_DEV void st(bf16* p, const float (&v)[8]) {
        *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]),
                                                  pack_bf2(v[4], v[5]), pack_bf2(v[6], v[7]));
    }
};

// one 16-byte piece (or one element) as it lies in memory, converted later:
// half the registers of converted bf16 while many loads are in flight
template <typename T, int V> struct Raw;
template <> struct Raw<bf16, 8> {
    uint4 r;
    PTCG_DEV void ld(const bf16* p) { r = *reinterpret_cast<const uint4*>(p); }
    PTCG_DEV void zero() { r = make_uint4(0u, 0u, 0u, 0u); }
    PTCG_DEV void get(float (&v)[8]) const {
        unpack_bf2(r.x, v[0], v[1]);
        unpack_bf2(r.y, v[2], v[3]);
        unpack_bf2(r.z, v[4], v[5]);
        unpack_bf2(r.w, v[6], v[7]);
    }
};
template <> struct Raw<bf16, 4> {
    uint2 r;
    PTCG_DEV void ld(const bf16* p) { r = *reinterpret_cast<const uint2*>(p); }
    PTCG_DEV void zero() { r = make_uint2(0u, 0u); }
    PTCG_DEV void get(float (&v)[4]) const {
        unpack_bf2(r.x, v[0], v[1]);
        unpack_bf2(r.y, v[2], v[3]);
    }
};
template <> struct Raw<float, 4> {
    float4 r;
    PTCG_DEV void ld(const float* p) { r = *reinterpret_cast<const float4*>(p); }
    PTCG_DEV void zero() { r = make_float4(0.f, 0.f, 0.f, 0.f); }
    PTCG_DEV void get(float (&v)[4]) const { v[0] = r.x; v[1] = r.y; v[2] = r.z; v[3] = r.w; }
};
template <typename T> struct Raw<T, 1> {
    T r;
    PTCG_DEV void ld(const T* p) { r = *p; }
    PTCG_DEV void zero() { r = from_f<T>(0.f); }
    PTCG_DEV void get(float (&v)[1]) const { v[0] = to_f<T>(r); }
};

static inline int dt_size(int dtype) { return dtype == PTCG_BF16 ? 2 : 4; }
static inline bool dt_ok(int dtype) { return dtype == PTCG_FP32 || dtype == PTCG_BF16; }
// rows of `ld` elements from p can be read V elements at a time (16-byte
// pieces at most)
static inline bool vec_ok(const void* p, int dtype, long ld, int V) {
    const long piece = V * (long)dt_size(dtype) < 16 ? V * (long)dt_size(dtype) : 16;
    return !p || ((uintptr_t)p % piece == 0 && (ld * dt_size(dtype)) % piece == 0);
}
static inline bool el_ok(const void* p, int dtype) { return (uintptr_t)p % dt_size(dtype) == 0; }
