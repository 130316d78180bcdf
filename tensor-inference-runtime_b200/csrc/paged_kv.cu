// paged_kv.cu -- the operators that fill and read back a paged key-value
// cache: per-head RMS norm and position rotation of queries and keys, the
// conversion or Q8_0 quantisation of keys and values as they are written to
// their pages, and the read-back of cached positions as rows.
//
// Every head vector of dim = 64, 128 or 256 elements is held by dim / 8 lanes
// of one warp, eight elements (one or two accesses) each, so the norm's sum and a
// block's maximum are shuffles, the rotation's partners lie in one lane and every
// element crosses memory once in and once out: the kernels are bound by memory, and
// by issue in 16-bit types.
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <mutex>
#include <string>
#include <vector>

#include "launch.cuh"
#include "paged.cuh"
#include "paged.h"
#include "ptx.cuh"

namespace tir {

static __device__ uint32_t g_paged_err;
static __device__ uint32_t g_paged_taken;

namespace {

// One step: a bit that another stream sets meanwhile is either taken or stays.
__global__ void take_error_kernel() { g_paged_taken = atomicExch(&g_paged_err, 0u); }

constexpr uint32_t FULL = 0xffffffffu;
constexpr int kRowThreads = 128;
constexpr int kMaxDevices = 64;

std::mutex g_err_mu, g_take_mu;
uint32_t* g_err_ptr[kMaxDevices];

struct RowArgs {
    const char *q, *k, *v;
    char *q_out, *k_out;
    int64_t q_stride, k_stride, v_stride, q_out_stride, k_out_stride;  // bytes between tokens
    const int32_t *seqs, *positions;
    int64_t tokens;
    int32_t q_heads, kv_heads;
    int32_t kinds;  // of key-value heads: keys, or keys and values
    int32_t q_chunks, kv_chunks;  // chunks of a token's query and key heads
    const float *q_w, *k_w, *rope;
    int64_t rope_positions;
    int32_t rope_dim, pairs;
    float eps;
    uint32_t* err;
};

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// Eight elements in two runs of four (8-byte aligned in 16-bit types).
template <Elem E>
__device__ __forceinline__ Raw8<E> load_raw4x2(const char* p0, const char* p1) {
    Raw8<E> r;
    if constexpr (E == Elem::F32) {
        r.w[0] = *reinterpret_cast<const uint4*>(p0);
        r.w[1] = *reinterpret_cast<const uint4*>(p1);
    } else {
        const uint2 x = *reinterpret_cast<const uint2*>(p0), y = *reinterpret_cast<const uint2*>(p1);
        r.w[0] = make_uint4(x.x, x.y, y.x, y.y);
    }
    return r;
}

// Rounds and stores them at elements e0 and e1 of p; APART: else e1 = e0 + 4.
template <Elem E, bool APART>
__device__ __forceinline__ void store4x2_as(char* p, int e0, int e1, const float* f) {
    constexpr int B = ElemOf<E>::bytes;
    if constexpr (!APART) {
        store8_as<E>(p + e0 * B, f);
    } else if constexpr (E == Elem::F32) {
        *reinterpret_cast<float4*>(p + e0 * B) = make_float4(f[0], f[1], f[2], f[3]);
        *reinterpret_cast<float4*>(p + e1 * B) = make_float4(f[4], f[5], f[6], f[7]);
    } else {
        *reinterpret_cast<uint2*>(p + e0 * B) = make_uint2(pack2(f[0], f[1], E), pack2(f[2], f[3], E));
        *reinterpret_cast<uint2*>(p + e1 * B) = make_uint2(pack2(f[4], f[5], E), pack2(f[6], f[7], E));
    }
}

__device__ __forceinline__ float rcp_approx(float x) {  // within one ulp
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

__device__ __forceinline__ float rsqrt_approx(float x) {
    float r;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// One Q8_0 block's rule (activated_q8, src/kernels.rs:8-31) over the four lanes
// that hold its 32 values: step d = the last of the elements of largest |x| / 127,
// quants = round half away (x / d), saturated, NaN -> 0.  The quotient uses the
// step before it is rounded to f16, as there, and the quants equal
// tir_activated_q8's bit for bit:
// * the largest and the smallest value give the step's sign, unless both reach
//   the largest magnitude; then the elements' order decides (a zero block, too);
// * y = x * (1 / d) is within 127 * 2^-22 < 2^-14 of the quotient, so where it is
//   further than that from a half its nearest integer is the quotient's;
// * nearer, with h the half above floor(|y|): the quotient rounded to f32 reaches h
//   where |x| / |d| >= h - half of f32's step below h, and |x| - h |d| is exact in
//   one fma (x and h d agree in their leading 13 bits, h d has eight more than d).
//   Values of 16 bits meet such halves often: x = max / 2 gives 63.5 (dividing there
//   takes 20.3 us for 8192 x 16 heads of 128 in bf16, this 16.9);
// * steps too small or too large for either, and NaN, are divided by.
__device__ __forceinline__ void quantise8(const float* f, int lane4, uint2* quants, float* step) {
    float hi = max3_nan(max3_nan(f[0], f[1], f[2]), max3_nan(f[3], f[4], f[5]), max_nan(f[6], f[7]));
    float lo = max3_nan(max3_nan(-f[0], -f[1], -f[2]), max3_nan(-f[3], -f[4], -f[5]), max_nan(-f[6], -f[7]));
#pragma unroll
    for (int w = 1; w <= 2; w <<= 1) {
        hi = max_nan(hi, __shfl_xor_sync(FULL, hi, w));
        lo = max_nan(lo, __shfl_xor_sync(FULL, lo, w));
    }
    float top = hi > lo ? hi : -lo;  // NaN: -lo, NaN as well
    if (__any_sync(FULL, hi == lo)) {
        uint32_t last = 0u;  // 2 (index + 1) + sign of the last element of magnitude hi
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (fabsf(f[i]) == hi) last = 2u * (lane4 * 8 + i + 1) + (__float_as_uint(f[i]) >> 31);
        last = max(last, __shfl_xor_sync(FULL, last, 1));
        last = max(last, __shfl_xor_sync(FULL, last, 2));
        if (hi == lo) top = last & 1u ? -hi : hi;
    }
    const float d = __fdiv_rn(top, 127.0f);
    const float inv = rcp_approx(d);
    uint32_t b[8];
    float far = 0.f;
    constexpr float kRound = 12582912.0f;  // 1.5 * 2^23: a sum with it has the nearest integer in its low bits
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 y = mul2(pair(f, i), make_float2(inv, inv)), n = add2(y, make_float2(kRound, kRound));
        b[2 * i] = __float_as_uint(n.x);
        b[2 * i + 1] = __float_as_uint(n.y);
        const float2 off = fma2(add2(n, make_float2(-kRound, -kRound)), make_float2(-1.f, -1.f), y);
        far = fmaxf(far, fmaxf(fabsf(off.x), fabsf(off.y)));
    }
    if (!(far < 0.5f - 1.0f / 16384.0f)) {
        const float da = fabsf(d), tiny = da * (1.0f / 16777216.0f);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float n = __fadd_rd(fabsf(__fmul_rn(f[i], inv)), 8388608.0f);  // 2^23 + floor
            const float h = n - 8388607.5f;
            // half a step below h, times |d|: the step is that of the value just below (h = 1/2 is a power of two)
            const float half = __uint_as_float((__float_as_uint(h) - 1u) & 0x7f800000u) * tiny;
            const float m = h + (fmaf(-h, da, fabsf(f[i])) >= -half ? 0.5f : -0.5f);
            b[i] = __float_as_uint(copysignf(m, __uint_as_float(__float_as_uint(f[i]) ^ __float_as_uint(d))) + kRound);
        }
    }
    if (!(fabsf(d) >= 1e-30f && fabsf(d) <= 1e30f)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float r = roundf(__fdiv_rn(f[i], d));
            b[i] = r != r ? 0u : static_cast<uint32_t>(static_cast<int>(fminf(fmaxf(r, -128.f), 127.f)));
        }
    }
    quants->x = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    quants->y = __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410);
    *step = d;
}

// The cached slot of token t; false (and the error bit) outside the table or
// on a bad page.
__device__ __forceinline__ bool find_slot(const RowArgs& a, const PagesView& kv, int64_t row, int32_t pos, bool tell, int64_t* at) {
    if (row < 0 || row >= kv.table_rows || pos >= static_cast<int64_t>(kv.max_pages) * kv.page_size) {
        if (tell) atomicOr(a.err, kBadPosition);
        return false;
    }
    const int32_t id = page_of(kv, row, pos);
    if (id < 0) return false;
    *at = slot_of(kv, id, pos);
    return true;
}

enum class Mode { Rows, Fused, FusedQ8, Append, AppendQ8 };

// Blocks an SM holds: eight of 64 registers a thread where a lane's four heads fit
// them (4109 tokens of 48 heads of 128 in f16: 20.8 us, with six 22.0; 8 x 1024 tokens
// of 16 heads of 128 in bf16 to Q8_0 and back: 25.2 and 25.8); where they would spill,
// six of 80 (norm and rotation of halves only, 8192 tokens of 40 heads of 128 in bf16:
// 32.1 us, with eight 37.4; into Q8_0, 48 heads: 52.7 and 55.3).
template <Elem A, Mode M, int HPG, bool H>
constexpr int kMinBlocks = HPG == 4 && (A == Elem::F32 || M == Mode::FusedQ8 || (M == Mode::Rows && H)) ? 6 : 8;

// A group of D / 8 lanes takes HPG heads of one kind (queries, keys or values) of
// a token, a block the same heads of 128 / (D / 8) tokens.  With many tokens
// HPG = 4: their loads are in flight together, and the token's position, slot,
// angles and weights are read once for four heads; with few, HPG = 1 spreads
// them.  The heads' data are asked for before the slot is looked up.  M says what
// a launch does and H that halves are paired in the rotation, so that each keeps
// only the registers it needs (more warps: the kernel is bound by issue and memory
// alike).  With paired halves a lane of the rotated part holds four elements of
// either half, so that it turns pairs of its own with half the angles (instead of eight
// consecutive ones and the partners by shuffles; together with the packed arithmetic and
// the grid by head and token that took 4109 tokens of 48 heads of 128 in f16 from 25.9 to
// 21.3 us, 64 in bf16 from 3.0 to 2.5); a block to be quantised then goes back to
// consecutive lanes by as many shuffles.  8192 tokens of 36 heads of 64 in f32 take 24.2 us
// (6.2 TB/s), the 4109 in f16 20.8 (4.9 TB/s).
template <Elem A, int D, Mode M, int HPG, bool H>
__global__ void __launch_bounds__(kRowThreads, kMinBlocks<A, M, HPG, H>) rows_kernel(const RowArgs a, const PagesView kv, const Elem cache) {
    constexpr int G = D / 8;
    constexpr int AB = ElemOf<A>::bytes;
    constexpr bool kAppend = M != Mode::Rows, kTurn = M == Mode::Rows || M == Mode::Fused || M == Mode::FusedQ8;
    constexpr bool kQ8 = M == Mode::FusedQ8 || M == Mode::AppendQ8;
    const int gl = threadIdx.x % G;
    // a block has one kind of head: what depends on it is the same for all its warps
    int chunk = static_cast<int>(blockIdx.x);
    const uint32_t t = (blockIdx.y + blockIdx.z * gridDim.y) * (kRowThreads / G) + threadIdx.x / G;
    const bool is_q = kTurn && chunk < a.q_chunks;
    if (!is_q) chunk -= a.q_chunks;
    const bool is_v = kAppend && !is_q && chunk >= a.kv_chunks;
    if (is_v) chunk -= a.kv_chunks;
    const int h0 = chunk * HPG, n = t < a.tokens ? min((is_q ? a.q_heads : a.kv_heads) - h0, HPG) : 0;
    griddep_wait();
    const int32_t pos = n > 0 && a.positions ? a.positions[t] : 0;
    const int32_t seq = kAppend && n > 0 && a.seqs ? a.seqs[t] : static_cast<int32_t>(t);
    const bool split = H && !is_v && gl < a.rope_dim / 8;
    const int e0 = split ? gl * 4 : gl * 8, e1 = split ? a.rope_dim / 2 + gl * 4 : gl * 8 + 4;
    const char* src = (is_q ? a.q + t * a.q_stride : is_v ? a.v + t * a.v_stride : a.k + t * a.k_stride) + h0 * D * AB;
    Raw8<A> raw[HPG];
#pragma unroll
    for (int x = 0; x < HPG; ++x) {
        raw[x] = Raw8<A>{};
        if (x < n) raw[x] = H ? load_raw4x2<A>(src + (x * D + e0) * AB, src + (x * D + e1) * AB) : load_raw8<A>(src + (x * D + e0) * AB);
    }
    const float* w_of = !kTurn ? nullptr : is_q ? a.q_w : is_v ? nullptr : a.k_w;
    float4 w[2];
    if (w_of) {
        w[0] = *reinterpret_cast<const float4*>(w_of + e0);
        w[1] = *reinterpret_cast<const float4*>(w_of + e1);
    }
    bool live = n > 0 && pos >= 0;
    if (kTurn && live && a.rope && pos >= a.rope_positions) {
        if (gl == 0) atomicOr(a.err, kBadPosition);
        live = false;
    }
    const bool turns = kTurn && live && !is_v && gl < a.rope_dim / 8;
    float4 cs[2];  // of this lane's four pairs
    if (turns) {
        const float* p = a.rope + static_cast<int64_t>(pos) * a.rope_dim + gl * 8;
        cs[0] = reinterpret_cast<const float4*>(p)[0];
        cs[1] = reinterpret_cast<const float4*>(p)[1];
    }
    // where it goes
    const bool to_cache = kAppend && !is_q;
    int64_t at = 0;
    if (to_cache && live) {
        live = find_slot(a, kv, seq, pos, gl == 0, &at);
        at += static_cast<int64_t>(h0) * kv.head_stride;
    }
    char* pool = is_v ? kv.v : kv.k;
    uint16_t* steps = is_v ? kv.vs : kv.ks;
    char* dst = (is_q ? a.q_out + t * a.q_out_stride : a.k_out + t * a.k_out_stride) + h0 * D * AB;
    const bool quantises = kQ8 && to_cache && __any_sync(FULL, live);
    const bool normed = kTurn && (a.q_w || a.k_w);
#pragma unroll
    for (int x = 0; x < HPG; ++x) {
        float f[8];
        expand8<A>(raw[x], f);
        if (normed) {  // for the whole launch: the shuffles stay outside what depends on the head
            float2 s2 = make_float2(0.f, 0.f);
#pragma unroll
            for (int i = 0; i < 4; ++i) s2 = fma2(pair(f, i), pair(f, i), s2);
            float ss = s2.x + s2.y;
#pragma unroll
            for (int o = G / 2; o; o >>= 1) ss += __shfl_xor_sync(FULL, ss, o);
            if (w_of) {
                // one step of Newton's iteration takes rsqrtf's two ulps to one rounding
                const float v = fmaf(ss, 1.0f / D, a.eps);
                float inv = rsqrt_approx(v);
                inv = fmaf(0.5f * inv, fmaf(-v * inv, inv, 1.0f), inv);
                if (!(v >= 1e-30f && v <= 1e30f)) inv = rsqrtf(v);
#pragma unroll
                for (int i = 0; i < 4; ++i) set_pair(f, i, mul2(mul2(pair(f, i), pair(&w[i >> 1].x, i & 1)), make_float2(inv, inv)));
            }
        }
        if (turns) {
            if constexpr (H) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float c = i & 1 ? cs[i >> 1].z : cs[i >> 1].x, s = i & 1 ? cs[i >> 1].w : cs[i >> 1].y;
                    const float u = f[i], v = f[i + 4];
                    f[i] = fmaf(c, u, __fmul_rn(-s, v));
                    f[i + 4] = fmaf(c, v, __fmul_rn(s, u));
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float c = i & 1 ? cs[i >> 1].z : cs[i >> 1].x, s = i & 1 ? cs[i >> 1].w : cs[i >> 1].y;
                    const float u = f[2 * i], v = f[2 * i + 1];
                    f[2 * i] = __fadd_rn(__fmul_rn(c, u), __fmul_rn(-s, v));
                    f[2 * i + 1] = __fadd_rn(__fmul_rn(s, u), __fmul_rn(c, v));
                }
            }
        }
        const bool write = live && x < n;
        if (quantises) {
            uint2 q;
            float step;
            if (H && !is_v) {  // a block's values back to consecutive lanes
                const bool odd = gl & 1, upper = gl >= a.rope_dim / 16;
                const int from = 2 * (upper ? gl - a.rope_dim / 16 : gl);
                const bool swap = split ? upper : odd;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    // even lanes send the first half's, then the second's; odd lanes the other way round
                    const float y = __shfl_sync(FULL, odd ? f[i + 4] : f[i], split ? from + upper : gl, G);
                    const float z = __shfl_sync(FULL, odd ? f[i] : f[i + 4], split ? from + !upper : gl, G);
                    f[i] = swap ? z : y;
                    f[i + 4] = swap ? y : z;
                }
            }
            quantise8(f, gl & 3, &q, &step);
            if (write && to_cache) {
                const int64_t here = at + x * kv.head_stride + gl * 8;
                *reinterpret_cast<uint2*>(pool + here) = q;
                if ((gl & 3) == 0) steps[here >> 5] = __half_as_ushort(__float2half_rn(step));
            }
        }
        if (!write) continue;
        if (!to_cache) {
            store4x2_as<A, H>(dst + x * D * AB, e0, e1, f);
        } else if (!kQ8) {
            const int64_t here = at + x * kv.head_stride;
            if (cache == Elem::F32)
                store4x2_as<Elem::F32, H>(pool + here * 4, e0, e1, f);
            else if (cache == Elem::F16)
                store4x2_as<Elem::F16, H>(pool + here * 2, e0, e1, f);
            else
                store4x2_as<Elem::BF16, H>(pool + here * 2, e0, e1, f);
        }
    }
}

// Cache -> rows: a group of D / 8 lanes takes HPG of a token's keys and values
// (HPG = 4 with many tokens: the three lookups before the data are then paid once
// for four loads in flight).
template <Elem A, int D, int HPG>
__global__ void __launch_bounds__(kRowThreads) gather_kernel(const RowArgs a, const PagesView kv, const Elem cache) {
    constexpr int G = D / 8;
    constexpr int AB = ElemOf<A>::bytes;
    const int gl = threadIdx.x % G;
    int chunk = static_cast<int>(blockIdx.x);
    const uint32_t t = (blockIdx.y + blockIdx.z * gridDim.y) * (kRowThreads / G) + threadIdx.x / G;
    griddep_wait();
    if (t >= a.tokens) return;
    const bool is_v = chunk >= a.kv_chunks;
    if (is_v) chunk -= a.kv_chunks;
    const int h0 = chunk * HPG, n = min(a.kv_heads - h0, HPG);
    const int32_t pos = a.positions[t];
    const int32_t seq = a.seqs ? a.seqs[t] : static_cast<int32_t>(t);
    int64_t at;
    if (pos < 0 || !find_slot(a, kv, seq, pos, gl == 0, &at)) return;
    at += static_cast<int64_t>(h0) * kv.head_stride + gl * 8;
    const char* pool = is_v ? kv.v : kv.k;
    const uint16_t* steps = is_v ? kv.vs : kv.ks;
    Raw8<Elem::F32> raw[HPG];
    float step[HPG];
#pragma unroll
    for (int x = 0; x < HPG; ++x) {
        if (x >= n) break;
        const int64_t here = at + x * kv.head_stride;
        if (cache == Elem::Q8) {
            const uint2 q = *reinterpret_cast<const uint2*>(pool + here);
            raw[x].w[0].x = q.x, raw[x].w[0].y = q.y;
            step[x] = __half2float(__ushort_as_half(steps[here >> 5]));
        } else if (cache == Elem::F32) {
            raw[x] = load_raw8<Elem::F32>(pool + here * 4);
        } else {
            raw[x].w[0] = *reinterpret_cast<const uint4*>(pool + here * 2);
        }
    }
    char* dst = (is_v ? a.k_out + t * a.k_out_stride : a.q_out + t * a.q_out_stride) + (h0 * D + gl * 8) * AB;
#pragma unroll
    for (int x = 0; x < HPG; ++x) {
        if (x >= n) break;
        float f[8];
        if (cache == Elem::Q8) {
            expand_q8x4(raw[x].w[0].x, step[x], f);
            expand_q8x4(raw[x].w[0].y, step[x], f + 4);
        } else if (cache == Elem::F32) {
            expand8<Elem::F32>(raw[x], f);
        } else if (cache == Elem::F16) {
            expand8<Elem::F16>(Raw8<Elem::F16>{{raw[x].w[0]}}, f);
        } else {
            expand8<Elem::BF16>(Raw8<Elem::BF16>{{raw[x].w[0]}}, f);
        }
        store8_as<A>(dst + x * D * AB, f);
    }
}

template <typename F>
cudaError_t by_type(Elem e, int32_t dim, F&& f) {
    using std::integral_constant;
    auto dims = [&](auto el) {
        if (dim == 64) return f(el, integral_constant<int, 64>{});
        if (dim == 128) return f(el, integral_constant<int, 128>{});
        return f(el, integral_constant<int, 256>{});
    };
    if (e == Elem::F32) return dims(integral_constant<Elem, Elem::F32>{});
    if (e == Elem::F16) return dims(integral_constant<Elem, Elem::F16>{});
    return dims(integral_constant<Elem, Elem::BF16>{});
}

// Heads a group of lanes takes, and the grid: four once one each would give every
// SM two blocks or more for each of its four schedulers (8192 tokens of 36 heads of
// 64 in f32: 27.4 us with one, 24.2 with four; with cache write 512 tokens of 48 heads of
// 128 in bf16: 6.5 and 5.4, 256 3.7 both), one below that (64 tokens: 2.3 and 3.1 us;
// read-back of 2047 positions of 4 heads of 64 in f32 2.6 and 2.9, of 65536 47.9 and 44.5).
struct RowShape {
    bool four;
    dim3 grid;  // chunks of one kind of head, blocks of tokens
};

bool row_shape(RowArgs* a, int32_t dim, RowShape* s) {
    if (a->tokens > INT32_MAX) return false;
    const int64_t per = kRowThreads / (dim / 8);
    s->four = a->tokens * (a->q_heads + static_cast<int64_t>(a->kinds) * a->kv_heads) > 4 * per * 148 * 2;
    const int64_t hpg = s->four ? 4 : 1;
    a->q_chunks = static_cast<int32_t>((a->q_heads + hpg - 1) / hpg);
    a->kv_chunks = static_cast<int32_t>((a->kv_heads + hpg - 1) / hpg);
    const int64_t chunks = a->q_chunks + a->kinds * static_cast<int64_t>(a->kv_chunks), blocks = (a->tokens + per - 1) / per;
    constexpr int64_t kGridY = 32768;  // the grid's second and third dimension end at 65535
    s->grid = dim3(static_cast<unsigned>(chunks), static_cast<unsigned>(blocks < kGridY ? blocks : kGridY),
                   static_cast<unsigned>((blocks + kGridY - 1) / kGridY));
    return chunks * blocks <= INT32_MAX;
}

// Both kernels and the attention are launched to take over as soon as the work before them
// is over (64 tokens with cache write: 2.3 us instead of 2.5; attention of one row of 144,
// called back to back: 6.1 instead of 8.2), but none lets the next one in before its own
// end: blocks that start while others still run gather on the SMs that come free first (64
// tokens' write, then attention over 64 x 2048 in Q8_0: 33.8 us so, 27.0 without).
template <Mode M>
cudaError_t launch_mode(const RowArgs& a, const PagesView& kv, Elem act, Elem cache, int32_t dim, const RowShape& s, cudaStream_t stream) {
    return by_type(act, dim, [&](auto el, auto d) {
        constexpr bool kTurn = M == Mode::Rows || M == Mode::Fused || M == Mode::FusedQ8;
        auto* kernel = s.four ? rows_kernel<decltype(el)::value, decltype(d)::value, M, 4, false>
                              : rows_kernel<decltype(el)::value, decltype(d)::value, M, 1, false>;
        if constexpr (kTurn)
            if (a.rope && a.pairs == TIR_PAIRS_HALVES)
                kernel = s.four ? rows_kernel<decltype(el)::value, decltype(d)::value, M, 4, true>
                                : rows_kernel<decltype(el)::value, decltype(d)::value, M, 1, true>;
        return launch_kernel(kernel, s.grid, dim3(kRowThreads), 0, stream, true, a, kv, cache);
    });
}

// `turned`: norm or rotation on the way (q_heads may be 0).
tir_status launch_rows(RowArgs a, const PagesView& kv, Elem act, Elem cache, int32_t dim, bool append, bool turned, void* stream,
                       const char* entry) {
    RowShape s;
    if (!row_shape(&a, dim, &s)) return fail(TIR_ERR_UNSUPPORTED_SHAPE, std::string(entry) + ": too many tokens");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool q8 = cache == Elem::Q8;
    cudaError_t e;
    if (!append)
        e = launch_mode<Mode::Rows>(a, kv, act, cache, dim, s, st);
    else if (turned)
        e = q8 ? launch_mode<Mode::FusedQ8>(a, kv, act, cache, dim, s, st) : launch_mode<Mode::Fused>(a, kv, act, cache, dim, s, st);
    else
        e = q8 ? launch_mode<Mode::AppendQ8>(a, kv, act, cache, dim, s, st) : launch_mode<Mode::Append>(a, kv, act, cache, dim, s, st);
    return e == cudaSuccess ? TIR_OK : paged_fail(e, entry);
}

tir_status check_norm(const tir_qk_norm* n, const int32_t* positions, int32_t dim, const char* entry) {
    const std::string who = entry;
    if (!n) return fail(TIR_ERR_INVALID_ARG, who + ": null norm description");
    if (n->rope) {
        if (n->rope_dim <= 0 || n->rope_dim % 16 || n->rope_dim > dim)
            return fail(TIR_ERR_UNSUPPORTED_SHAPE, who + ": rope_dim must be a positive multiple of 16 up to the head size");
        if (n->pairs != TIR_PAIRS_ADJACENT && n->pairs != TIR_PAIRS_HALVES)
            return fail(TIR_ERR_INVALID_ARG, who + ": unknown pairing of the rotation");
        if (n->rope_positions <= 0) return fail(TIR_ERR_INVALID_ARG, who + ": empty rotation table");
        if (!positions) return fail(TIR_ERR_INVALID_ARG, who + ": a rotation needs positions");
    }
    if ((reinterpret_cast<uintptr_t>(n->q_weight) | reinterpret_cast<uintptr_t>(n->k_weight) | reinterpret_cast<uintptr_t>(n->rope)) % 16)
        return fail(TIR_ERR_INVALID_ARG, who + ": weights and rotation table must be 16-byte aligned");
    if ((n->q_weight || n->k_weight) && !(n->eps >= 0.f))
        return fail(TIR_ERR_INVALID_ARG, who + ": eps must not be negative");
    return TIR_OK;
}

void set_norm(RowArgs* a, const tir_qk_norm* n) {
    a->q_w = n->q_weight;
    a->k_w = n->k_weight;
    a->rope = n->rope;
    a->rope_positions = n->rope_positions;
    a->rope_dim = n->rope ? n->rope_dim : 0;
    a->pairs = n->pairs;
    a->eps = n->eps;
}

tir_status check_dim(int32_t dim, const char* entry) {
    if (dim != 64 && dim != 128 && dim != 256)
        return fail(TIR_ERR_UNSUPPORTED_SHAPE, std::string(entry) + ": the head size must be 64, 128 or 256");
    return TIR_OK;
}

}  // namespace

bool act_elem(int32_t dtype, Elem* out) {
    switch (dtype) {
        case TIR_DTYPE_F32: *out = Elem::F32; return true;
        case TIR_DTYPE_F16: *out = Elem::F16; return true;
        case TIR_DTYPE_BF16: *out = Elem::BF16; return true;
        default: return false;
    }
}

tir_status paged_fail(cudaError_t e, const char* what) {
    return fail(e == cudaErrorMemoryAllocation ? TIR_ERR_OOM : TIR_ERR_CUDA,
                std::string(what) + ": " + cudaGetErrorName(e) + " (" + cudaGetErrorString(e) + ")");
}

static int elem_bytes(Elem e) { return e == Elem::F32 ? 4 : e == Elem::Q8 ? 1 : 2; }

tir_status pages_view(const tir_kv_pages* kv, const char* entry, PagesView* v, Elem* type) {
    const std::string who = entry;
    if (!kv) return fail(TIR_ERR_INVALID_ARG, who + ": null cache description");
    if (kv->dtype == TIR_DTYPE_Q8_0)
        *type = Elem::Q8;
    else if (!act_elem(kv->dtype, type))
        return fail(TIR_ERR_UNSUPPORTED_DTYPE, who + ": cache type " + std::to_string(kv->dtype) + " is not F32, F16, BF16 or Q8_0");
    const tir_status rc = check_dim(kv->dim, entry);
    if (rc != TIR_OK) return rc;
    const bool q8 = *type == Elem::Q8;
    if (!kv->k || !kv->v || !kv->table || (q8 && (!kv->k_scale || !kv->v_scale)))
        return fail(TIR_ERR_INVALID_ARG, who + ": null pool, scale or table pointer");
    if (kv->kv_heads <= 0 || kv->page_size <= 0 || kv->max_pages <= 0 || kv->table_rows < 0 ||
        kv->table_stride < kv->max_pages || kv->n_pages <= 0 || kv->n_pages > INT32_MAX)
        return fail(TIR_ERR_INVALID_ARG, who + ": bad cache sizes");
    if (static_cast<int64_t>(kv->max_pages) * kv->page_size > (1 << 30))
        return fail(TIR_ERR_UNSUPPORTED_SHAPE, who + ": a table row holds more than 2^30 positions");
    const int64_t unit = q8 ? kv->dim : 16 / elem_bytes(*type);
    const int64_t strides[3] = {kv->page_stride, kv->pos_stride, kv->head_stride};
    for (int64_t s : strides)
        if (s < 0 || s % unit)
            return fail(TIR_ERR_INVALID_ARG, who + ": cache strides must be multiples of " + std::to_string(unit) + " elements");
    if ((reinterpret_cast<uintptr_t>(kv->k) | reinterpret_cast<uintptr_t>(kv->v) |
         (q8 ? reinterpret_cast<uintptr_t>(kv->k_scale) | reinterpret_cast<uintptr_t>(kv->v_scale) : 0)) % 16)
        return fail(TIR_ERR_INVALID_ARG, who + ": pools must be 16-byte aligned");
    const int es = elem_bytes(*type);
    const double span = (static_cast<double>(kv->n_pages) * kv->page_stride + static_cast<double>(kv->page_size) * kv->pos_stride +
                         static_cast<double>(kv->kv_heads) * kv->head_stride) * es / 16;
    if (span >= 4294967295.0) return fail(TIR_ERR_UNSUPPORTED_SHAPE, who + ": a pool spans 64 GB or more");
    v->page16 = static_cast<uint32_t>(kv->page_stride * es / 16);
    v->pos16 = static_cast<uint32_t>(kv->pos_stride * es / 16);
    v->head16 = static_cast<uint32_t>(kv->head_stride * es / 16);
    v->k = static_cast<char*>(kv->k);
    v->v = static_cast<char*>(kv->v);
    v->ks = kv->k_scale;
    v->vs = kv->v_scale;
    v->table = kv->table;
    v->table_rows = kv->table_rows;
    v->table_stride = kv->table_stride;
    v->n_pages = kv->n_pages;
    v->page_stride = kv->page_stride;
    v->pos_stride = kv->pos_stride;
    v->head_stride = kv->head_stride;
    v->max_pages = kv->max_pages;
    v->page_size = kv->page_size;
    v->page_shift = -1;
    for (int s = 0; s < 31; ++s)
        if ((1 << s) == kv->page_size) v->page_shift = s;
    v->kv_heads = kv->kv_heads;
    v->dim = kv->dim;
    v->err = nullptr;
    return TIR_OK;
}

tir_status check_rows(const void* p, int64_t stride, int64_t heads, int64_t dim, Elem e, const char* entry,
                      const char* what) {
    if (!p) return fail(TIR_ERR_INVALID_ARG, std::string(entry) + ": null " + what);
    if (stride < heads * dim)
        return fail(TIR_ERR_INVALID_ARG, std::string(entry) + ": " + what + " stride is shorter than a token's heads");
    if (reinterpret_cast<uintptr_t>(p) % 16 || (stride * elem_bytes(e)) % 16)
        return fail(TIR_ERR_INVALID_ARG, std::string(entry) + ": " + what + " must keep 16-byte alignment");
    return TIR_OK;
}

tir_status paged_error_word(uint32_t** out) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return paged_fail(e, "cudaGetDevice");
    if (dev < 0 || dev >= kMaxDevices) return fail(TIR_ERR_INVALID_ARG, "device index out of range");
    std::lock_guard<std::mutex> lock(g_err_mu);
    if (!g_err_ptr[dev]) {
        void* p = nullptr;
        e = cudaGetSymbolAddress(&p, g_paged_err);
        if (e != cudaSuccess) return paged_fail(e, "cudaGetSymbolAddress");
        g_err_ptr[dev] = static_cast<uint32_t*>(p);
    }
    *out = g_err_ptr[dev];
    return TIR_OK;
}

tir_status paged_take_error(int device, void* stream, uint32_t* bits) {
    *bits = 0u;
    {
        std::lock_guard<std::mutex> lock(g_err_mu);  // not over the wait: launches take it, too
        if (device < 0 || device >= kMaxDevices || !g_err_ptr[device]) return TIR_OK;
    }
    std::lock_guard<std::mutex> lock(g_take_mu);  // until the taken bits are read
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e = launch_kernel(take_error_kernel, dim3(1), dim3(1), 0, st, false);
    if (e == cudaSuccess) e = cudaMemcpyFromSymbolAsync(bits, g_paged_taken, sizeof(uint32_t), 0, cudaMemcpyDeviceToHost, st);
    const cudaError_t done = cudaStreamSynchronize(st);
    if (e == cudaSuccess) e = done;
    return e == cudaSuccess ? TIR_OK : paged_fail(e, "paged cache error word");
}

}  // namespace tir

using namespace tir;

extern "C" {

tir_status tir_rope_table(float base, int64_t dim, int64_t n_pos, float* out_host) {
    clear_error();
    if (dim <= 0 || dim % 2 || n_pos < 0) return fail(TIR_ERR_INVALID_ARG, "rope table: dim must be even and positive, n_pos not negative");
    if (!out_host && n_pos > 0) return fail(TIR_ERR_INVALID_ARG, "rope table: null output");
    // rope_angles (src/math.rs:181-193) and its cosf / sinf, as the engine's own table
    const int64_t half = dim / 2;
    for (int64_t i = 0; i < half; ++i) {
        const float freq = powf(base, (-2.0f * static_cast<float>(i)) / static_cast<float>(dim));
        for (int64_t pos = 0; pos < n_pos; ++pos) {
            const float theta = static_cast<float>(pos) * freq;
            out_host[(pos * half + i) * 2] = cosf(theta);
            out_host[(pos * half + i) * 2 + 1] = sinf(theta);
        }
    }
    return TIR_OK;
}

tir_status tir_qk_norm_rope(const void* q, int64_t q_stride, const void* k, int64_t k_stride, void* q_out,
                            int64_t q_out_stride, void* k_out, int64_t k_out_stride, const int32_t* positions,
                            int64_t tokens, int32_t q_heads, int32_t kv_heads, int32_t dim, int32_t dtype,
                            const tir_qk_norm* norm, void* stream) {
    clear_error();
    const char* who = "tir_qk_norm_rope";
    Elem act;
    if (!act_elem(dtype, &act)) return fail(TIR_ERR_UNSUPPORTED_DTYPE, std::string(who) + ": activations must be F32, F16 or BF16");
    tir_status rc = check_dim(dim, who);
    if (rc != TIR_OK) return rc;
    if (tokens < 0 || q_heads < 0 || kv_heads < 0 || q_heads + static_cast<int64_t>(kv_heads) > (1 << 20))
        return fail(TIR_ERR_INVALID_ARG, std::string(who) + ": bad sizes");
    if (tokens == 0 || q_heads + kv_heads == 0) return TIR_OK;
    rc = check_norm(norm, positions, dim, who);
    if (rc == TIR_OK && q_heads) rc = check_rows(q, q_stride, q_heads, dim, act, who, "q");
    if (rc == TIR_OK && q_heads) rc = check_rows(q_out, q_out_stride, q_heads, dim, act, who, "q_out");
    if (rc == TIR_OK && kv_heads) rc = check_rows(k, k_stride, kv_heads, dim, act, who, "k");
    if (rc == TIR_OK && kv_heads) rc = check_rows(k_out, k_out_stride, kv_heads, dim, act, who, "k_out");
    if (rc != TIR_OK) return rc;
    const int es = elem_bytes(act);
    RowArgs a{};
    a.q = static_cast<const char*>(q);
    a.k = static_cast<const char*>(k);
    a.q_out = static_cast<char*>(q_out);
    a.k_out = static_cast<char*>(k_out);
    a.q_stride = q_stride * es;
    a.k_stride = k_stride * es;
    a.q_out_stride = q_out_stride * es;
    a.k_out_stride = k_out_stride * es;
    a.positions = positions;
    a.tokens = tokens;
    a.q_heads = q_heads;
    a.kv_heads = kv_heads;
    a.kinds = 1;
    set_norm(&a, norm);
    rc = paged_error_word(&a.err);
    if (rc != TIR_OK) return rc;
    return launch_rows(a, PagesView{}, act, Elem::F32, dim, false, true, stream, who);
}

static tir_status append(const char* who, const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v,
                         int64_t v_stride, void* q_out, int64_t q_out_stride, const tir_kv_pages* kv,
                         const int32_t* seqs, const int32_t* positions, int64_t tokens, int32_t q_heads, int32_t dtype,
                         const tir_qk_norm* norm, void* stream) {
    Elem act, cache;
    PagesView view;
    if (!act_elem(dtype, &act)) return fail(TIR_ERR_UNSUPPORTED_DTYPE, std::string(who) + ": activations must be F32, F16 or BF16");
    tir_status rc = pages_view(kv, who, &view, &cache);
    if (rc != TIR_OK) return rc;
    if (tokens < 0 || q_heads < 0 || q_heads + 2ll * kv->kv_heads > (1 << 20))
        return fail(TIR_ERR_INVALID_ARG, std::string(who) + ": bad sizes");
    if (tokens == 0) return TIR_OK;
    if (!positions) return fail(TIR_ERR_INVALID_ARG, std::string(who) + ": null positions");
    if (!seqs && tokens > kv->table_rows)
        return fail(TIR_ERR_INVALID_ARG, std::string(who) + ": more tokens than table rows and no sequence indices");
    if (norm) rc = check_norm(norm, positions, kv->dim, who);
    if (rc == TIR_OK && q_heads) rc = check_rows(q, q_stride, q_heads, kv->dim, act, who, "q");
    if (rc == TIR_OK && q_heads) rc = check_rows(q_out, q_out_stride, q_heads, kv->dim, act, who, "q_out");
    if (rc == TIR_OK) rc = check_rows(k, k_stride, kv->kv_heads, kv->dim, act, who, "k");
    if (rc == TIR_OK) rc = check_rows(v, v_stride, kv->kv_heads, kv->dim, act, who, "v");
    if (rc != TIR_OK) return rc;
    const int es = elem_bytes(act);
    RowArgs a{};
    a.q = static_cast<const char*>(q);
    a.k = static_cast<const char*>(k);
    a.v = static_cast<const char*>(v);
    a.q_out = static_cast<char*>(q_out);
    a.q_stride = q_stride * es;
    a.k_stride = k_stride * es;
    a.v_stride = v_stride * es;
    a.q_out_stride = q_out_stride * es;
    a.seqs = seqs;
    a.positions = positions;
    a.tokens = tokens;
    a.q_heads = q_heads;
    a.kv_heads = kv->kv_heads;
    a.kinds = 2;
    if (norm) set_norm(&a, norm);
    rc = paged_error_word(&a.err);
    if (rc != TIR_OK) return rc;
    view.err = a.err;
    return launch_rows(a, view, act, cache, kv->dim, true, norm != nullptr, stream, who);
}

tir_status tir_qk_norm_rope_append(const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v,
                                   int64_t v_stride, void* q_out, int64_t q_out_stride, const tir_kv_pages* kv,
                                   const int32_t* seqs, const int32_t* positions, int64_t tokens, int32_t q_heads,
                                   int32_t dtype, const tir_qk_norm* norm, void* stream) {
    clear_error();
    if (!norm) return fail(TIR_ERR_INVALID_ARG, "tir_qk_norm_rope_append: null norm description");
    return append("tir_qk_norm_rope_append", q, q_stride, k, k_stride, v, v_stride, q_out, q_out_stride, kv, seqs,
                  positions, tokens, q_heads, dtype, norm, stream);
}

tir_status tir_kv_append(const tir_kv_pages* kv, const void* k, int64_t k_stride, const void* v, int64_t v_stride,
                         const int32_t* seqs, const int32_t* positions, int64_t tokens, int32_t dtype, void* stream) {
    clear_error();
    return append("tir_kv_append", nullptr, 0, k, k_stride, v, v_stride, nullptr, 0, kv, seqs, positions, tokens, 0, dtype,
                  nullptr, stream);
}

tir_status tir_kv_gather(const tir_kv_pages* kv, void* k_out, int64_t k_out_stride, void* v_out, int64_t v_out_stride,
                         const int32_t* seqs, const int32_t* positions, int64_t tokens, int32_t dtype, void* stream) {
    clear_error();
    const char* who = "tir_kv_gather";
    Elem act, cache;
    PagesView view;
    if (!act_elem(dtype, &act)) return fail(TIR_ERR_UNSUPPORTED_DTYPE, std::string(who) + ": rows must be F32, F16 or BF16");
    tir_status rc = pages_view(kv, who, &view, &cache);
    if (rc != TIR_OK) return rc;
    if (tokens < 0 || kv->kv_heads > (1 << 19)) return fail(TIR_ERR_INVALID_ARG, std::string(who) + ": bad sizes");
    if (tokens == 0) return TIR_OK;
    if (!positions) return fail(TIR_ERR_INVALID_ARG, std::string(who) + ": null positions");
    if (!seqs && tokens > kv->table_rows)
        return fail(TIR_ERR_INVALID_ARG, std::string(who) + ": more tokens than table rows and no sequence indices");
    rc = check_rows(k_out, k_out_stride, kv->kv_heads, kv->dim, act, who, "k_out");
    if (rc == TIR_OK) rc = check_rows(v_out, v_out_stride, kv->kv_heads, kv->dim, act, who, "v_out");
    if (rc != TIR_OK) return rc;
    const int es = elem_bytes(act);
    RowArgs a{};
    a.q_out = static_cast<char*>(k_out);
    a.k_out = static_cast<char*>(v_out);
    a.q_out_stride = k_out_stride * es;
    a.k_out_stride = v_out_stride * es;
    a.seqs = seqs;
    a.positions = positions;
    a.tokens = tokens;
    a.kv_heads = kv->kv_heads;
    a.kinds = 2;
    rc = paged_error_word(&a.err);
    if (rc != TIR_OK) return rc;
    view.err = a.err;
    RowShape s;
    if (!row_shape(&a, kv->dim, &s)) return fail(TIR_ERR_UNSUPPORTED_SHAPE, std::string(who) + ": too many tokens");
    const cudaError_t e = by_type(act, kv->dim, [&](auto el, auto d) {
        auto* kernel = s.four ? gather_kernel<decltype(el)::value, decltype(d)::value, 4>
                              : gather_kernel<decltype(el)::value, decltype(d)::value, 1>;
        return launch_kernel(kernel, s.grid, dim3(kRowThreads), 0, static_cast<cudaStream_t>(stream), true, a, view, cache);
    });
    return e == cudaSuccess ? TIR_OK : paged_fail(e, who);
}

}  // extern "C"
