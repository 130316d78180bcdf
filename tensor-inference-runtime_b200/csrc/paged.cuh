// paged.cuh -- device parts the paged cache kernels share: vectors of eight
// elements of an activation or cache type, and the page lookup.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "paged.h"

namespace tir {

template <Elem E>
struct ElemOf;
template <>
struct ElemOf<Elem::F32> {
    static constexpr int bytes = 4;
};
template <>
struct ElemOf<Elem::F16> {
    static constexpr int bytes = 2;
};
template <>
struct ElemOf<Elem::BF16> {
    static constexpr int bytes = 2;
};
template <>
struct ElemOf<Elem::Q8> {
    static constexpr int bytes = 1;
};

// Eight consecutive elements as they lie in memory (16-byte aligned).
template <Elem E>
struct Raw8 {
    uint4 w[ElemOf<E>::bytes == 4 ? 2 : 1];
};

template <Elem E>
__device__ __forceinline__ Raw8<E> load_raw8(const char* p) {
    Raw8<E> r;
#pragma unroll
    for (int i = 0; i < (ElemOf<E>::bytes == 4 ? 2 : 1); ++i) r.w[i] = reinterpret_cast<const uint4*>(p)[i];
    return r;
}

__device__ __forceinline__ float2 unpack2(uint32_t w, Elem e) {
    if (e == Elem::F16) return __half22float2(*reinterpret_cast<const __half2*>(&w));
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
}

__device__ __forceinline__ uint32_t pack2(float a, float b, Elem e) {
    if (e == Elem::F16) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

template <Elem E>
__device__ __forceinline__ void expand8(const Raw8<E>& r, float* f) {
    const uint32_t* w = &r.w[0].x;
    if constexpr (E == Elem::F32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = __uint_as_float((&r.w[i >> 2].x)[i & 3]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 p = unpack2(w[i], E);
            f[2 * i] = p.x;
            f[2 * i + 1] = p.y;
        }
    }
}

// Rounds (to nearest even) and stores eight elements.
template <Elem E>
__device__ __forceinline__ void store8_as(char* p, const float* f) {
    if constexpr (E == Elem::F32) {
        reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
    } else {
        uint4 w;
        w.x = pack2(f[0], f[1], E);
        w.y = pack2(f[2], f[3], E);
        w.z = pack2(f[4], f[5], E);
        w.w = pack2(f[6], f[7], E);
        *reinterpret_cast<uint4*>(p) = w;
    }
}

// Two f32 operations in one instruction.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("mul.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<uint64_t&>(r))
        : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<uint64_t&>(r))
        : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
    return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<uint64_t&>(r))
        : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
    return r;
}
__device__ __forceinline__ float2 sub2(float2 a, float2 b) { return fma2(b, make_float2(-1.f, -1.f), a); }
__device__ __forceinline__ float2 pair(const float* f, int i) { return make_float2(f[2 * i], f[2 * i + 1]); }
__device__ __forceinline__ void set_pair(float* f, int i, float2 p) { f[2 * i] = p.x, f[2 * i + 1] = p.y; }

// Four int8 quants of a word, times their block's step (exact in f32).  Each quant + 128
// becomes the low byte of 2^23: integer-to-float conversions issue at a quarter of the rate.
__device__ __forceinline__ void expand_q8x4(uint32_t w, float step, float* f) {
    const uint32_t u = w ^ 0x80808080u;
    const float2 less = make_float2(-8388736.f, -8388736.f), by = make_float2(step, step);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float2 n = make_float2(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7540 + 2 * i)),
                                     __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7541 + 2 * i)));
        set_pair(f, i, mul2(add2(n, less), by));
    }
}

// Page lookup shared by the kernels: the id the table holds for `pos` of row
// `row`, and whether it lies in the pool (else the error bit is set).
__device__ __forceinline__ int32_t page_id(const PagesView& v, int64_t row, int32_t pos) {
    const int32_t i = v.page_shift >= 0 ? pos >> v.page_shift : pos / v.page_size;
    return v.table[row * v.table_stride + i];
}

__device__ __forceinline__ bool page_ok(const PagesView& v, int32_t id) {
    if (static_cast<uint32_t>(id) < static_cast<uint32_t>(v.n_pages)) return true;
    atomicOr(v.err, kBadPage);
    return false;
}

__device__ __forceinline__ int32_t page_of(const PagesView& v, int64_t row, int32_t pos) {
    const int32_t id = page_id(v, row, pos);
    return page_ok(v, id) ? id : -1;
}

// Element offset of `pos` in page `id` (head 0).
__device__ __forceinline__ int64_t slot_of(const PagesView& v, int32_t id, int32_t pos) {
    const int32_t in = v.page_shift >= 0 ? pos & (v.page_size - 1) : pos % v.page_size;
    return id * v.page_stride + in * v.pos_stride;
}

// The same in 16-byte units (a pool spans at most 2^32 of them).
__device__ __forceinline__ uint32_t slot16_of(const PagesView& v, int32_t id, int32_t pos) {
    const uint32_t in = v.page_shift >= 0 ? pos & (v.page_size - 1) : pos % v.page_size;
    return id * v.page16 + in * v.pos16;
}

}  // namespace tir
