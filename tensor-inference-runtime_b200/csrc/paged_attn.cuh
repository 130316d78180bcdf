// paged_attn.cuh -- decode attention over a paged cache: one query token per
// sequence, a group of query heads per key-value head.
//
//   t_j = c (q . k_j),  c = scale log2 e;   o = sum_j 2^(t_j - m) v_j / sum_j 2^(t_j - m)
//
// It is bound by the bytes of the cache, read once: a key-value head's query
// heads share every key and value.  A CTA takes one (row, key-value head, tile of
// 8 NT query heads) over a part of the row's positions; its warps take tiles of 16
// or 32 positions in turn, each with a ring of cp.async half tiles (keys, values,
// keys, ...) and a softmax (m, l, o) of its own, so the loop has no CTA barrier.
// The warps' parts meet in shared memory, those of different CTAs in
// paged_attn_join.  64 rows of 2048 positions take 84 to 87 us in bf16 with 8 heads of
// 128 (6.3 TB/s: bound by memory), 49.5 in f32 with 4 heads of 64 (5.4 TB/s) and 24 in
// Q8_0 (3.0 TB/s).  The last two are bound by latency: 256 CTAs leave a scheduler 1.7
// warps, each of which issues every 3.4 to 3.8 cycles (most of them the fixed latency of
// the instruction before: two tf32 parts of every value, the conversions of every quant),
// so that a scheduler issues in half of its cycles and no pipe is busy for above 46 %.
//
// Products on the tensor cores (mma.sync: with 8 query heads a tile is M = 16
// positions or dimensions by N = 8 heads, far below the smallest tcgen05 tile,
// and the pipe is not the bound), transposed so that heads are the N columns and
// no row of a tile is padding:
//   S' (16 positions x 8 heads)  = K (16 x dim) . Q' (dim x 8)
//   O' (dim x 8 heads)          += V' (dim x 16) . P' (16 x 8)
// S' comes out with positions along the lanes' rows; movmatrix turns its 8 x 8
// blocks into the operand layout of P'.
//
// Operand types.  K and V enter as they are stored: f16 / bf16 directly, Q8_0
// quants as exact f16 integers with the block steps applied outside, f32 split
// into two tf32 parts.  q and the weights p are split into as many parts as they
// need: 16-bit queries are exact in one (bf16 ones scaled by a power of two for
// f16), f32 queries take two f16 (22 bits under a per-head power of two), three
// bf16 or two tf32 parts.  p has two bf16 parts (16 bits, below the rounding of a
// 16-bit output; three under f32 queries), two tf32 parts or two f16 ones, the
// second kept above its place so that f16's range does not cut small weights off.
// Scores, m, l and o are f32 throughout.
#pragma once
#include <cuda_runtime.h>

#include <atomic>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "launch.cuh"
#include "paged.cuh"
#include "ptx.cuh"

namespace tir {

struct AttnArgs {
    const char* q;
    char* out;
    int64_t q_stride, out_stride;  // elements
    const int32_t* lens;
    int32_t q_heads, group, head_tiles;  // head_tiles: tiles of 8 NT query heads per key-value head
    int32_t window;                      // INT32_MAX: none
    int32_t splits, min_units;
    float scale_log2;
    Elem act;
    float *part_o, *part_ml;  // [rows][q_heads][splits][dim], [..][splits][2]
};

// The part of a row's positions that split `i` of `splits` takes, in units of
// `unit` positions: as even as whole units allow, none below `min_units` units.
// `used` splits have any.
struct AttnRange {
    int32_t first, k0, k1, used;
};

__device__ __forceinline__ AttnRange attn_range(int32_t len, int32_t window, int32_t splits, int32_t min_units,
                                                int32_t unit, int32_t i) {
    AttnRange r;
    r.first = len > window ? len - window : 0;
    const int32_t units = (len - r.first + unit - 1) / unit;
    const int32_t per = max((units + splits - 1) / splits, min_units);
    r.used = (units + per - 1) / per;
    const int64_t k0 = r.first + static_cast<int64_t>(i) * per * unit;
    r.k0 = static_cast<int32_t>(min(k0, static_cast<int64_t>(len)));
    r.k1 = static_cast<int32_t>(min(k0 + static_cast<int64_t>(per) * unit, static_cast<int64_t>(len)));
    return r;
}

__device__ __forceinline__ int32_t row_length(const AttnArgs& a, const PagesView& kv, int64_t row) {
    const int32_t len = a.lens[row];
    const int64_t cap = static_cast<int64_t>(kv.max_pages) * kv.page_size;
    if (len >= 0 && len <= cap) return len;
    if (threadIdx.x == 0) atomicOr(kv.err, kBadLength);
    return len < 0 ? 0 : static_cast<int32_t>(cap);
}

// ---- instruction wrappers ----------------------------------------------------
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// Copies 16 bytes, or (size 0) writes zeros and reads nothing.
__device__ __forceinline__ void cp_async16_sized(uint32_t dst, const void* src, int size) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(size) : "memory");
}

template <int B>
__device__ __forceinline__ void cp_async_small_or_zero(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(B), "r"(live ? B : 0)
                 : "memory");
}

__device__ __forceinline__ void ldsm4(uint32_t* r, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

__device__ __forceinline__ void ldsm4_t(uint32_t* r, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// d (16 x 8, f32) += a (16 x 16) b (16 x 8)
template <bool BF>
__device__ __forceinline__ void mma16(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    if constexpr (BF)
        asm(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// d (16 x 8, f32) += a (16 x 8) b (8 x 8), tf32 operands
__device__ __forceinline__ void mma8(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t to_tf32(float x) {
    uint32_t y;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(y) : "f"(x));
    return y;
}

// x = hi + lo to 22 bits, both tf32.
__device__ __forceinline__ void split_tf32(float x, uint32_t* hi, uint32_t* lo) {
    *hi = to_tf32(x);
    *lo = to_tf32(x - __uint_as_float(*hi));
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Parts (m, l, o) of a row count 2^(m - top) times.  One without a position on a page of the
// pool has m = -inf, and a row of such parts gets zeros; one whose scores are all -inf has
// kNoWeight, below every other, and a row of such parts 0 / 0.
constexpr float kNoWeight = -3.402823466e38f;
__device__ __forceinline__ float part_factor(float m, float top) { return m == -INFINITY ? 0.f : exp2_fast(m - top); }
__device__ __forceinline__ float part_sum(float sum, float top) { return top == -INFINITY ? 1.f : sum; }

// Four int8 as exact f16 integers: bytes 0 and 2 in *even, 1 and 3 in *odd.  The
// byte 128 + n under the exponent of 1024 reads 1152 + n.  (Leaving the 128 in, as f16's
// denormals (128 + n) 2^-24, and taking 128 sum q off the keys' products spares two of five
// operations, but such a sum has f32's steps at 128 sum q: with quants below 4 beside one of
// 127 outputs were off by 3e-5, without the 128 by 3e-7.)
__device__ __forceinline__ void q8_pairs(uint32_t w, uint32_t* even, uint32_t* odd) {
    const uint32_t a = (w & 0x00ff00ffu) ^ 0x64806480u, b = ((w >> 8) & 0x00ff00ffu) ^ 0x64806480u;
    const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
    const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), bias), y = __hsub2(*reinterpret_cast<const __half2*>(&b), bias);
    *even = *reinterpret_cast<const uint32_t*>(&x);
    *odd = *reinterpret_cast<const uint32_t*>(&y);
}

// The Q8_0 steps of one position's head: D / 32 halves in one load.
template <int D>
struct Steps {
    uint32_t w[D / 64];
    __device__ __forceinline__ void load(const uint8_t* p, int key) {
        if constexpr (D == 64) {
            w[0] = reinterpret_cast<const uint32_t*>(p)[key];
        } else if constexpr (D == 128) {
            const uint2 x = reinterpret_cast<const uint2*>(p)[key];
            w[0] = x.x, w[1] = x.y;
        } else {
            const uint4 x = reinterpret_cast<const uint4*>(p)[key];
            w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
        }
    }
    __device__ __forceinline__ float get(int b) const {
        return __half2float(__ushort_as_half(static_cast<uint16_t>(b & 1 ? w[b / 2] >> 16 : w[b / 2] & 0xffffu)));
    }
    // the larger magnitudes of the even and the odd blocks, as two 16-bit patterns
    __device__ __forceinline__ uint32_t top() const {
        uint32_t m = w[0] & 0x7fff7fffu;
#pragma unroll
        for (int i = 1; i < D / 64; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
        return m;
    }
};

// ---- configuration -----------------------------------------------------------
// C: cache type; D: head size; NT: tiles of 8 query heads a CTA takes; F32Q: f32
// queries (else 16-bit ones).
template <Elem C, int D, int NT, bool F32Q>
struct AttnCfg {
    static constexpr bool tf32 = C == Elem::F32, f16 = C == Elem::F16, bf = C == Elem::BF16, q8 = C == Elem::Q8;
    static constexpr int ES = ElemOf<C>::bytes;
    static constexpr int NQ = tf32 ? 2 : !F32Q ? 1 : bf ? 3 : 2;  // parts of q
    static constexpr int NP = tf32 ? 2 : bf && F32Q ? 3 : 2;      // parts of p
    // f16 operands hold q under a per-head power of two, but for f16 queries of f16 caches (exact as they are)
    static constexpr bool scaled = q8 || (C == Elem::F16 && F32Q);
    // f32 queries take the scores' factor in before they are split; unscaled ones
    // leave nothing to multiply a score by
    static constexpr bool plain = F32Q && !scaled;
    static constexpr int ROW = D * ES;
    // positions of a warp's tile: 32 where rows are short, so that the work around a
    // tile (pages, copies, votes) is shared by more of them
    static constexpr int TILE = ROW <= 128 ? 32 : 16;
    static constexpr int MT = TILE / 16;
    static constexpr int PITCH = ROW + 16;  // an odd number of 16-byte units: ldmatrix rows fall on different banks
    static constexpr int STEPS = q8 ? D / 32 * 2 : 0;  // bytes of a position's Q8_0 steps
    static constexpr int STEPS_AT = TILE * PITCH;
    static constexpr int HALF = STEPS_AT + TILE * STEPS;  // the keys or the values of a tile
    static constexpr int KSTEPS = tf32 ? D / 8 : D / 16;  // q operand steps
    static constexpr int QBYTES = KSTEPS * NT * NQ * 256;
    static constexpr int HEADS = 8 * NT;
    static constexpr int WARPS = HALF > 16 * 1024 && NT == 2 ? 2 : 4;  // two where q takes the room
    static constexpr int THREADS = WARPS * 32;
    static constexpr int UNIT = WARPS * TILE;
    static constexpr int FIXED = QBYTES + HEADS * 4 + WARPS * HEADS * 8;
    // a warp's ring: SLOTS half tiles (keys, values, keys, ...), an odd number, so that
    // a step on keys asks for keys.  Three CTAs an SM for heads of 64 (64 x 2048 in f32:
    // 49.5 us, 51.1 with two; 64 x 256 10.3 and 10.6), two for wider ones where three slots
    // fit (64 x 2048 in bf16 with heads of 128: 86 us, 98 with three).
    static constexpr int fits(int ctas) { return (227 * 1024 / ctas - 1024 - FIXED) / (WARPS * HALF); }
    static constexpr int PER_SM = fits(3) >= 3 && D == 64 && NT == 1 ? 3 : fits(2) >= 3 ? 2 : 1;
    static constexpr int SLOTS = fits(PER_SM) >= 7 ? 7 : fits(PER_SM) >= 5 ? 5 : 3;
    static constexpr int AHEAD = (SLOTS - 1) / 2;  // tiles asked for before they are used
    static constexpr int RING = WARPS * SLOTS * HALF;
    static constexpr int SMEM = RING + FIXED;
    // q operands in registers where they are few
    static constexpr bool q_in_regs = KSTEPS * NT * NQ * 2 <= 64;
    static_assert(fits(PER_SM) >= 3, "the ring needs three slots");
    static_assert(SLOTS * HALF >= HEADS * (D + 4) * 4, "a warp's output fits its ring");
    static_assert(HALF % 16 == 0 && RING % 16 == 0 && QBYTES % 16 == 0, "16-byte copies");
};

template <Elem C, int D, int NT, bool F32Q>
__global__ void __launch_bounds__(AttnCfg<C, D, NT, F32Q>::THREADS, AttnCfg<C, D, NT, F32Q>::PER_SM)
    paged_attn_kernel(const AttnArgs a, const PagesView kv) {
    using X = AttnCfg<C, D, NT, F32Q>;
    constexpr uint32_t FULL = 0xffffffffu;
    constexpr int CH = X::ROW / 16;        // 16-byte pieces of a cached row
    constexpr int LPR = CH < 8 ? CH : 8;  // lanes that copy a row
    // Weights are 2^kLift above their logarithm's reference, which may lag the maximum by
    // kLag: those in f16 parts fill its range from the top (2^15).  Their second part is
    // kept kRest above its place, in a sum of its own: in its place its digits would end
    // with f16's range, from weights of 2^-12 of the reference's on (a key that leads the
    // row by 8), and a long row sums 10^5 of those.  So 20 bits remain down to 2^-28 (19),
    // 12 to 2^-36 (25); in Q8_0 of weights times steps, beside the largest step.
    constexpr bool kSmall = X::f16 || X::q8;
    constexpr float kLift = kSmall ? 11.f : 0.f;
    constexpr float kLag = kSmall ? 4.f : 8.f;
    constexpr float kRest = 4096.f;
    extern __shared__ __align__(16) uint8_t smem[];
    uint8_t* ring = smem;
    uint32_t* qf = reinterpret_cast<uint32_t*>(smem + X::RING);
    float* cs = reinterpret_cast<float*>(smem + X::RING + X::QBYTES);
    float* ml = cs + X::HEADS;  // [WARPS][HEADS][2]

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int tiles = kv.kv_heads * a.head_tiles;
    // the heads of a row's part are neighbours: their rows lie side by side in the
    // pages, and are read at about the same time
    const int tile = static_cast<int>(blockIdx.x % tiles);
    const int split = static_cast<int>(blockIdx.x / tiles % a.splits);
    const int64_t row = blockIdx.x / tiles / a.splits;
    const int hk = tile / a.head_tiles, j0 = tile % a.head_tiles * X::HEADS;  // key-value head, first head of its group
    const int nh = min(a.group - j0, X::HEADS);
    const int h0 = hk * a.group + j0;
    griddep_wait();
    // what depends on no length is asked for along with it: this warp's query heads
    // (element i * 32 + lane) and, where the row is not divided, its first pages
    float xq[X::HEADS / X::WARPS][D / 32];
#pragma unroll
    for (int y = 0; y < X::HEADS / X::WARPS; ++y)
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            const int j = y * X::WARPS + warp;
            const int64_t at = row * a.q_stride + static_cast<int64_t>(h0 + j) * D + i * 32 + lane;
            xq[y][i] = j >= nh                 ? 0.f
                       : a.act == Elem::F32   ? reinterpret_cast<const float*>(a.q)[at]
                       : a.act == Elem::F16 ? __half2float(reinterpret_cast<const __half*>(a.q)[at])
                                            : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(a.q)[at]);
        }
    const bool undivided = a.splits == 1 && a.window == INT32_MAX;
    int32_t pages[X::AHEAD + 1];
    if (undivided) {
        const int32_t cap = kv.max_pages * kv.page_size;
#pragma unroll
        for (int i = 0; i <= X::AHEAD; ++i) {
            const int32_t pos = (i * X::WARPS + warp) * X::TILE + (lane & (X::TILE - 1));
            pages[i] = pos < cap ? page_id(kv, row, pos) : -1;
        }
    }
    const int32_t len = row_length(a, kv, row);
    const AttnRange range = attn_range(len, a.window, a.splits, a.min_units, X::UNIT, split);
    if (range.used == 0) {  // nothing to look at: zeros
        if (split == 0)
            for (int i = threadIdx.x; i < nh * (D / 8); i += X::THREADS) {
                const float z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                const int64_t at = row * a.out_stride + static_cast<int64_t>(h0) * D + i * 8;
                if (a.act == Elem::F32)
                    store8_as<Elem::F32>(a.out + at * 4, z);
                else
                    store8_as<Elem::F16>(a.out + at * 2, z);
            }
        return;
    }
    if (range.k0 >= range.k1) return;

    // ---- the ring ----
    const int n_tiles = (range.k1 - range.k0 + X::TILE - 1) / X::TILE;
    const int my_tiles = n_tiles > warp ? (n_tiles - warp + X::WARPS - 1) / X::WARPS : 0;
    uint8_t* my_ring = ring + warp * X::SLOTS * X::HALF;
    const uint32_t ring_addr = smem_u32(my_ring);
    // this lane's position (lane % TILE) of the warp's tile i, and the page it is on:
    // asked for one tile before its copies are issued, checked only then
    auto position = [&](int i) -> int32_t { return range.k0 + (i * X::WARPS + warp) * X::TILE + (lane & (X::TILE - 1)); };
    auto lookup = [&](int i) -> int32_t {
        const int32_t pos = position(i);
        return pos < range.k1 ? page_id(kv, row, pos) : -1;
    };
    // where this lane's position of tile i lies, in 16-byte units; kNowhere past the
    // end or on a bad page: zeros are copied instead, and its score is -inf
    constexpr uint32_t kNowhere = 0xffffffffu;
    const uint32_t head_at = hk * kv.head16;
    auto place = [&](int i, int32_t page) -> uint32_t {
        const int32_t pos = position(i);
        return pos < range.k1 && page_ok(kv, page) ? slot16_of(kv, page, pos) + head_at : kNowhere;
    };
    // copies the keys or values of a tile into a slot, a 128-byte line (or a whole
    // shorter row) at a time
    auto issue = [&](int slot, uint32_t mine, bool full, const char* pool, const uint16_t* steps) {
        const uint32_t dst = ring_addr + slot * X::HALF;
        if constexpr (X::q8) {
            if (X::TILE == 32 || lane < 16)
                cp_async_small_or_zero<X::STEPS>(dst + X::STEPS_AT + lane * X::STEPS, steps + (mine == kNowhere ? 0 : mine >> 1), mine != kNowhere);
        }
        const char* from = pool + (lane % LPR) * 16;
        const uint32_t to = dst + (lane / LPR) * X::PITCH + (lane % LPR) * 16;
        if (full) {
#pragma unroll
            for (int u = 0; u < X::TILE * LPR / 32; ++u) {
                const uint32_t at = __shfl_sync(FULL, mine, u * (32 / LPR) + lane / LPR);
                const char* row_from = from + static_cast<uint64_t>(at) * 16;
#pragma unroll
                for (int ch = 0; ch < CH; ch += LPR) cp_async16(to + u * (32 / LPR) * X::PITCH + ch * 16, row_from + ch * 16);
            }
        } else {
#pragma unroll
            for (int u = 0; u < X::TILE * LPR / 32; ++u) {
                const uint32_t at = __shfl_sync(FULL, mine, u * (32 / LPR) + lane / LPR);
                const char* row_from = from + (at == kNowhere ? 0 : static_cast<uint64_t>(at) * 16);
#pragma unroll
                for (int ch = 0; ch < CH; ch += LPR)
                    cp_async16_sized(to + u * (32 / LPR) * X::PITCH + ch * 16, row_from + ch * 16, at == kNowhere ? 0 : 16);
            }
        }
    };
    if (!undivided) {  // all asked for before the first is waited for
#pragma unroll
        for (int i = 0; i <= X::AHEAD; ++i) pages[i] = lookup(i);
    }
    uint32_t live[X::AHEAD];  // of the tiles asked for, in order: bit p (TILE 16: p + 16, too) for position p
#pragma unroll
    for (int i = 0; i < X::AHEAD; ++i) {
        const uint32_t at = place(i, pages[i]);
        live[i] = __ballot_sync(FULL, at != kNowhere);
        if (i < my_tiles) issue(2 * i, at, live[i] == FULL, kv.k, kv.ks);
        cp_async_commit();
        if (i < my_tiles) issue(2 * i + 1, at, live[i] == FULL, kv.v, kv.vs);
        cp_async_commit();
    }
    uint32_t any_live = 0u;
    int32_t next_page = pages[X::AHEAD];

    // ---- q operands, while the first tiles are on their way ----
#pragma unroll
    for (int y = 0; y < X::HEADS / X::WARPS; ++y) {
        const int j = y * X::WARPS + warp;
        float* x = xq[y];
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            if constexpr (F32Q) x[i] *= a.scale_log2;
            top = fmaxf(top, fabsf(x[i]));
        }
        float c = F32Q ? 1.f : a.scale_log2;
        if constexpr (X::scaled) {
#pragma unroll
            for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(FULL, top, o));
            const int e = static_cast<int>(__float_as_uint(top) >> 23);  // biased exponent
            if (e > 0 && e < 255) {                                      // top * 2^s in [2^9, 2^10)
                const int s = min(136 - e, 60);  // below 2^-51 every score rounds to 0 whatever its digits
                const float up = __uint_as_float(static_cast<uint32_t>(127 + s) << 23);
                c *= __uint_as_float(static_cast<uint32_t>(127 - s) << 23);
#pragma unroll
                for (int i = 0; i < D / 32; ++i) x[i] *= up;
            }
        }
        if (lane == 0) cs[j] = fmaxf(c, 1.2e-38f);  // never 0: a masked score is c * -inf
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            const int e = i * 32 + lane;  // element of the head
            if constexpr (X::tf32) {
                const int kk = e / 8, r = e % 8, at = ((kk * NT + j / 8) * 2) * 64 + ((j % 8) * 4 + r % 4) * 2 + r / 4;
                split_tf32(x[i], &qf[at], &qf[at + 64]);
            } else {
                // operand element k = 2 t' + {0, 1} (+ 8 in the second register); Q8_0 words
                // hold elements 4 t' .. 4 t' + 3 and give bytes 0, 2 and 1, 3: there the order is theirs
                const int kk = e / 16, r = e % 16;
                const int tt = X::q8 ? r / 4 : r % 8 / 2, reg = X::q8 ? r & 1 : r / 8;
                float rem = x[i];
#pragma unroll
                for (int s = 0; s < X::NQ; ++s) {
                    const int at = (((kk * NT + j / 8) * X::NQ + s) * 32 + (j % 8) * 4 + tt) * 2 + reg;
                    uint16_t* p = reinterpret_cast<uint16_t*>(qf + at) + (X::q8 ? r % 4 / 2 : r & 1);
                    if constexpr (X::bf) {
                        const __nv_bfloat16 b = __float2bfloat16_rn(rem);
                        *p = __bfloat16_as_ushort(b);
                        rem -= __bfloat162float(b);
                    } else {
                        const __half b = __float2half_rn(rem);
                        *p = __half_as_ushort(b);
                        rem -= __half2float(b);
                    }
                }
            }
        }
    }
    __syncthreads();
    uint32_t qr[X::q_in_regs ? X::KSTEPS * NT * X::NQ * 2 : 1];
    if constexpr (X::q_in_regs) {
#pragma unroll
        for (int i = 0; i < X::KSTEPS * NT * X::NQ; ++i) {
            const uint2 w = reinterpret_cast<const uint2*>(qf)[i * 32 + lane];
            qr[2 * i] = w.x;
            qr[2 * i + 1] = w.y;
        }
    }
    auto q_op = [&](int kk, int nt, int s) -> uint2 {
        const int i = (kk * NT + nt) * X::NQ + s;
        if constexpr (X::q_in_regs) return make_uint2(qr[2 * i], qr[2 * i + 1]);
        else return reinterpret_cast<const uint2*>(qf)[i * 32 + lane];
    };
    float c[NT][2], m[NT][2], base[NT][2], l[NT][2], o[D / 16][NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            c[n][e] = cs[n * 8 + 2 * t + e];
            m[n][e] = -INFINITY;
            base[n][e] = -kLift;
            l[n][e] = 0.f;
        }
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][n][e] = 0.f;
    int v_exp = 0;  // Q8_0: o is kept over 2^(v_exp - 14), the power of two above the steps seen so far

    // c s - base.  The product is rounded (or exact: c is a power of two under f32
    // queries) before the difference is taken, as the maximum's was: equal scores
    // stay equal whatever their size.
    auto above = [&](float2 s, int n) -> float2 {
        const float2 less = make_float2(-base[n][0], -base[n][1]);
        if constexpr (X::plain) return add2(s, less);
        else if constexpr (F32Q) return fma2(s, pair(c[n], 0), less);
        else return add2(mul2(s, pair(c[n], 0)), less);
    };

    // ---- the loop over this warp's tiles ----
    int slot = 0, free_slot = X::SLOTS - 1;
    auto advance = [&]() {
        free_slot = slot;
        slot = slot + 1 == X::SLOTS ? 0 : slot + 1;
    };
    for (int it = 0; it < my_tiles; ++it) {
        cp_async_wait<X::SLOTS - 2>();
        __syncwarp();
        const bool more = it + X::AHEAD < my_tiles;
        const uint32_t ahead = place(it + X::AHEAD, next_page);
        const uint32_t now = live[0];
        any_live |= now;
#pragma unroll
        for (int i = 0; i + 1 < X::AHEAD; ++i) live[i] = live[i + 1];
        live[X::AHEAD - 1] = __ballot_sync(FULL, ahead != kNowhere);
        const bool full = live[X::AHEAD - 1] == FULL;
        if (more) issue(free_slot, ahead, full, kv.k, kv.ks);
        cp_async_commit();
        next_page = lookup(it + X::AHEAD + 1);
        const uint8_t* st = my_ring + slot * X::HALF;
        const uint32_t row_addr = ring_addr + slot * X::HALF + (lane & 15) * X::PITCH + (lane >> 4) * 16;
        advance();

        // S' = K Q'
        float s[X::MT][NT][4];
#pragma unroll
        for (int mt = 0; mt < X::MT; ++mt) {
            const uint32_t k_addr = row_addr + mt * 16 * X::PITCH;
            // several sums at once: a product waits for the one before it in its chain
            constexpr int CHAINS = X::q8 ? 1 : X::tf32 ? 6 : 2 * X::NQ;
            float acc[CHAINS][NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[mt][n][e] = 0.f;
#pragma unroll
                    for (int x = 0; x < CHAINS; ++x) acc[x][n][e] = 0.f;
                }
            if constexpr (X::q8) {
                Steps<D> k_steps[2];
                k_steps[0].load(st + X::STEPS_AT, mt * 16 + g);
                k_steps[1].load(st + X::STEPS_AT, mt * 16 + g + 8);
#pragma unroll
                for (int b = 0; b < D / 32; ++b) {
                    uint32_t w[4], x0[4], x1[4];
                    ldsm4(w, k_addr + b * 32);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t* x = i < 2 ? x0 : x1;
                        q8_pairs(w[i], &x[i & 1], &x[2 + (i & 1)]);
                    }
                    const float d0 = k_steps[0].get(b), d1 = k_steps[1].get(b);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int p = X::NQ - 1; p >= 0; --p) {
                            const uint2 q0 = q_op(2 * b, n, p), q1 = q_op(2 * b + 1, n, p);
                            mma16<false>(sum, x0, q0.x, q0.y);
                            mma16<false>(sum, x1, q1.x, q1.y);
                        }
                        s[mt][n][0] = fmaf(sum[0], d0, s[mt][n][0]);
                        s[mt][n][1] = fmaf(sum[1], d0, s[mt][n][1]);
                        s[mt][n][2] = fmaf(sum[2], d1, s[mt][n][2]);
                        s[mt][n][3] = fmaf(sum[3], d1, s[mt][n][3]);
                    }
                }
            } else if constexpr (X::tf32) {
#pragma unroll
                for (int kk = 0; kk < D / 8; ++kk) {
                    uint32_t w[4], hi[4], lo[4];
                    ldsm4(w, k_addr + kk * 32);
#pragma unroll
                    for (int e = 0; e < 4; ++e) split_tf32(__uint_as_float(w[e]), &hi[e], &lo[e]);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const uint2 qh = q_op(kk, n, 0), ql = q_op(kk, n, 1);
                        mma8(acc[kk & 1][n], lo, qh.x, qh.y);
                        mma8(acc[2 + (kk & 1)][n], hi, ql.x, ql.y);
                        mma8(acc[4 + (kk & 1)][n], hi, qh.x, qh.y);
                    }
                }
            } else {
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                    uint32_t w[4];
                    ldsm4(w, k_addr + kk * 32);
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int p = X::NQ - 1; p >= 0; --p) {
                            const uint2 qv = q_op(kk, n, p);
                            mma16<X::bf>(acc[2 * (X::NQ - 1 - p) + (kk & 1)][n], w, qv.x, qv.y);
                        }
                }
            }
            if constexpr (!X::q8) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        // smallest parts first
                        float2 sum = pair(acc[0][n], y);
#pragma unroll
                        for (int x = 1; x < CHAINS; ++x) sum = add2(sum, pair(acc[x][n], y));
                        set_pair(s[mt][n], y, sum);
                    }
            }
        }

        // weights: p = 2^(t - m + lift), with m moved only when a score passes it by
        // more than kLag (rare after the first tiles): no reduction in the usual tile
        if (now != FULL) {
#pragma unroll
            for (int mt = 0; mt < X::MT; ++mt)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!(now >> (mt * 16 + g + (e >> 1) * 8) & 1u)) s[mt][n][e] = -INFINITY;
        }
        bool moves = false;
        float top[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                top[n][e] = fmaxf(s[0][n][e], s[0][n][e + 2]);
#pragma unroll
                for (int mt = 1; mt < X::MT; ++mt) top[n][e] = fmaxf(top[n][e], fmaxf(s[mt][n][e], s[mt][n][e + 2]));
                if constexpr (!X::plain) top[n][e] *= c[n][e];
                moves |= top[n][e] > m[n][e] + kLag;
            }
        // the values' turn
        cp_async_wait<X::SLOTS - 2>();
        __syncwarp();
        if (more) issue(free_slot, ahead, full, kv.v, kv.vs);
        cp_async_commit();
        const uint8_t* sv = my_ring + slot * X::HALF;
        const uint32_t v_base = ring_addr + slot * X::HALF;
        advance();
        Steps<X::q8 ? D : 64> v_steps[X::MT][2];
        uint32_t v_top = 0u;
        if constexpr (X::q8) {
#pragma unroll
            for (int mt = 0; mt < X::MT; ++mt)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    v_steps[mt][half].load(sv + X::STEPS_AT, mt * 16 + g + 8 * half);
                    v_top = __vmaxu2(v_top, v_steps[mt][half].top());
                }
            v_top = max(v_top & 0xffffu, v_top >> 16) >> 10;
            moves |= static_cast<int>(v_top) > v_exp;
        }
        if (__any_sync(FULL, moves)) {
            float shrink = 1.f;
            if constexpr (X::q8) {
                v_top = __reduce_max_sync(FULL, v_top);
                const int up = max(static_cast<int>(v_top) - v_exp, 0);
                shrink = __uint_as_float(static_cast<uint32_t>(127 - up) << 23);
                v_exp += up;
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float f[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
#pragma unroll
                    for (int w = 4; w < 32; w <<= 1) top[n][e] = fmaxf(top[n][e], __shfl_xor_sync(FULL, top[n][e], w));
                    const float mn = fmaxf(m[n][e], top[n][e]);
                    const float corr = m[n][e] == mn ? 1.f : exp2_fast(m[n][e] - mn);
                    m[n][e] = mn;
                    base[n][e] = (mn == -INFINITY ? 0.f : mn) - kLift;
                    l[n][e] *= corr;
                    f[e] = corr * shrink;
                }
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                    o[i][n][0] *= f[0];
                    o[i][n][1] *= f[1];
                    o[i][n][2] *= f[0];
                    o[i][n][3] *= f[1];
                }
            }
        }
#pragma unroll
        for (int mt = 0; mt < X::MT; ++mt)
#pragma unroll
            for (int n = 0; n < NT; ++n)
            {
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const float2 z = above(pair(s[mt][n], y), n);
                    set_pair(s[mt][n], y, make_float2(exp2_fast(z.x), exp2_fast(z.y)));
                }
                set_pair(l[n], 0, add2(pair(l[n], 0), add2(pair(s[mt][n], 0), pair(s[mt][n], 1))));
            }

        // O' += V' P'.  The tensor core's f32 sums are cut off, not rounded: under f32
        // queries a tile's products are summed from zero and then added, so that a
        // long row's error does not grow with its length.
        auto begin = [&](float* acc, const float* sum) {
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] = F32Q ? 0.f : sum[e];
        };
        auto finish = [&](float* sum, const float* acc) {
#pragma unroll
            for (int e = 0; e < 2; ++e) set_pair(sum, e, F32Q ? add2(pair(sum, e), pair(acc, e)) : pair(acc, e));
        };
        auto add_rest = [&](float* acc, const float* rest) {
#pragma unroll
            for (int e = 0; e < 2; ++e) set_pair(acc, e, fma2(pair(rest, e), make_float2(1.f / kRest, 1.f / kRest), pair(acc, e)));
        };
        if constexpr (X::q8) {
            const float inv = __uint_as_float(static_cast<uint32_t>(127 + 14 - v_exp) << 23);
            const uint32_t v_addr = v_base + (lane & 15) * X::PITCH + (lane >> 4) * 16;
#pragma unroll
            for (int b = 0; b < D / 32; ++b) {
                float acc[2][NT][4], rest[2][NT][4];
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        begin(acc[i][n], o[2 * b + i][n]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) rest[i][n][e] = 0.f;
                    }
#pragma unroll
                for (int mt = 0; mt < X::MT; ++mt) {
                    const float d0 = v_steps[mt][0].get(b) * inv, d1 = v_steps[mt][1].get(b) * inv;
                    uint32_t p0[NT][2], p1[NT][2];
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const float2 wa = mul2(pair(s[mt][n], 0), make_float2(d0, d0)), wb = mul2(pair(s[mt][n], 1), make_float2(d1, d1));
                        const __half2 ha = __float22half2_rn(wa), hb = __float22half2_rn(wb);
                        const float2 up = make_float2(kRest, kRest);
                        const float2 ra = mul2(sub2(wa, __half22float2(ha)), up), rb = mul2(sub2(wb, __half22float2(hb)), up);
                        p0[n][0] = transpose8x8(*reinterpret_cast<const uint32_t*>(&ha));
                        p0[n][1] = transpose8x8(*reinterpret_cast<const uint32_t*>(&hb));
                        p1[n][0] = transpose8x8(pack2(ra.x, ra.y, Elem::F16));
                        p1[n][1] = transpose8x8(pack2(rb.x, rb.y, Elem::F16));
                    }
                    uint32_t w[4], x[2][4];
                    ldsm4_t(w, v_addr + mt * 16 * X::PITCH + b * 32);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        q8_pairs(w[2 * i], &x[i][0], &x[i][1]);
                        q8_pairs(w[2 * i + 1], &x[i][2], &x[i][3]);
#pragma unroll
                        for (int n = 0; n < NT; ++n) mma16<false>(rest[i][n], x[i], p1[n][0], p1[n][1]);
                    }
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int n = 0; n < NT; ++n) mma16<false>(acc[i][n], x[i], p0[n][0], p0[n][1]);
                }
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        add_rest(acc[i][n], rest[i][n]);
                        finish(o[2 * b + i][n], acc[i][n]);
                    }
            }
        } else if constexpr (X::tf32) {
            uint32_t ph[X::MT][2][NT][2], pl[X::MT][2][NT][2];
#pragma unroll
            for (int mt = 0; mt < X::MT; ++mt)
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const uint32_t x = __float_as_uint(s[mt][n][2 * kb]), y = __float_as_uint(s[mt][n][2 * kb + 1]);
                        const uint32_t up = transpose8x8(__byte_perm(x, y, 0x7632)), dn = transpose8x8(__byte_perm(x, y, 0x5410));
                        split_tf32(__uint_as_float(__byte_perm(dn, up, 0x5410)), &ph[mt][kb][n][0], &pl[mt][kb][n][0]);
                        split_tf32(__uint_as_float(__byte_perm(dn, up, 0x7632)), &ph[mt][kb][n][1], &pl[mt][kb][n][1]);
                    }
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                float acc[NT][4];
#pragma unroll
                for (int n = 0; n < NT; ++n) begin(acc[n], o[i][n]);
#pragma unroll
                for (int mt = 0; mt < X::MT; ++mt)
#pragma unroll
                    for (int kb = 0; kb < 2; ++kb) {
                        const uint8_t* v = sv + (mt * 16 + 8 * kb + 2 * t) * X::PITCH + g * 8 + i * 64;
                        const float2 va = *reinterpret_cast<const float2*>(v);
                        const float2 vb = *reinterpret_cast<const float2*>(v + X::PITCH);
                        uint32_t hi[4], lo[4];
                        split_tf32(va.x, &hi[0], &lo[0]);
                        split_tf32(va.y, &hi[1], &lo[1]);
                        split_tf32(vb.x, &hi[2], &lo[2]);
                        split_tf32(vb.y, &hi[3], &lo[3]);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            mma8(acc[n], lo, ph[mt][kb][n][0], ph[mt][kb][n][1]);
                            mma8(acc[n], hi, pl[mt][kb][n][0], pl[mt][kb][n][1]);
                            mma8(acc[n], hi, ph[mt][kb][n][0], ph[mt][kb][n][1]);
                        }
                    }
#pragma unroll
                for (int n = 0; n < NT; ++n) finish(o[i][n], acc[n]);
            }
        } else {
            uint32_t pp[X::MT][NT][X::NP][2];
#pragma unroll
            for (int mt = 0; mt < X::MT; ++mt)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float2 ra = pair(s[mt][n], 0), rb = pair(s[mt][n], 1);
#pragma unroll
                    for (int p = 0; p < X::NP; ++p) {
                        const uint32_t wa = pack2(ra.x, ra.y, C), wb = pack2(rb.x, rb.y, C);
                        pp[mt][n][p][0] = transpose8x8(wa);
                        pp[mt][n][p][1] = transpose8x8(wb);
                        ra = sub2(ra, unpack2(wa, C)), rb = sub2(rb, unpack2(wb, C));
                        if constexpr (kSmall) ra = mul2(ra, make_float2(kRest, kRest)), rb = mul2(rb, make_float2(kRest, kRest));
                    }
                }
            const uint32_t v_addr = v_base + ((lane & 7) + (lane >> 4) * 8) * X::PITCH + ((lane >> 3) & 1) * 16;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                float acc[NT][4], rest[NT][4];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    begin(acc[n], o[i][n]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) rest[n][e] = 0.f;
                }
#pragma unroll
                for (int mt = 0; mt < X::MT; ++mt) {
                    uint32_t w[4];
                    ldsm4_t(w, v_addr + mt * 16 * X::PITCH + i * 32);
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int p = X::NP - 1; p >= 0; --p)
                            mma16<X::bf>(kSmall && p == 1 ? rest[n] : acc[n], w, pp[mt][n][p][0], pp[mt][n][p][1]);
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    if constexpr (kSmall) add_rest(acc[n], rest[n]);
                    finish(o[i][n], acc[n]);
                }
            }
        }
    }
    cp_async_wait_all();
    if (a.splits > 1) griddep_launch_dependents();  // the join
    __syncwarp();

    // ---- the warps' parts joined ----
    if constexpr (X::q8) {
        const float f = __uint_as_float(static_cast<uint32_t>(127 + v_exp - 14) << 23);
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][n][e] *= f;
    }
    float* mine = reinterpret_cast<float*>(my_ring);  // [HEADS][D + 4]
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int j = n * 8 + 2 * t + e;
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) l[n][e] += __shfl_xor_sync(FULL, l[n][e], w);
            if (g == 0) {
                ml[(warp * X::HEADS + j) * 2] = any_live ? fmaxf(m[n][e], kNoWeight) : m[n][e];
                ml[(warp * X::HEADS + j) * 2 + 1] = l[n][e];
            }
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                float* at = mine + j * (D + 4) + i * 16;
                if constexpr (X::q8 || X::tf32) {  // rows g, g + 8 of a 16-dimension tile are dimensions 2 g, 2 g + 1
                    *reinterpret_cast<float2*>(at + 2 * g) = make_float2(o[i][n][e], o[i][n][e + 2]);
                } else {
                    at[g] = o[i][n][e];
                    at[g + 8] = o[i][n][e + 2];
                }
            }
        }
    __syncthreads();
    for (int i = threadIdx.x; i < nh * (D / 8); i += X::THREADS) {
        const int j = i / (D / 8), d = i % (D / 8) * 8;
        float top = -INFINITY, sum = 0.f, y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < X::WARPS; ++w) top = fmaxf(top, ml[(w * X::HEADS + j) * 2]);
#pragma unroll
        for (int w = 0; w < X::WARPS; ++w) {
            const float f = part_factor(ml[(w * X::HEADS + j) * 2], top);
            const float lw = ml[(w * X::HEADS + j) * 2 + 1];
            sum += f * lw;
            const float* part = reinterpret_cast<const float*>(ring + w * X::SLOTS * X::HALF) + j * (D + 4) + d;
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = fmaf(f, part[e], y[e]);
        }
        if (range.used == 1) {
            sum = part_sum(sum, top);
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = y[e] / sum;
            const int64_t at = row * a.out_stride + static_cast<int64_t>(h0 + j) * D + d;
            if (a.act == Elem::F32)
                store8_as<Elem::F32>(a.out + at * 4, y);
            else if (a.act == Elem::F16)
                store8_as<Elem::F16>(a.out + at * 2, y);
            else
                store8_as<Elem::BF16>(a.out + at * 2, y);
        } else {
            const int64_t at = (row * a.q_heads + h0 + j) * a.splits + split;
            store8_as<Elem::F32>(reinterpret_cast<char*>(a.part_o + at * D + d), y);
            if (d == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(top, sum);
        }
    }
}

template <Elem C, int D, int NT, bool F32Q>
cudaError_t launch_attn_as(const AttnArgs& a, const PagesView& kv, int64_t rows, cudaStream_t stream) {
    using X = AttnCfg<C, D, NT, F32Q>;
    // the shared-memory opt-in, once on each device
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    const uint64_t bit = uint64_t{1} << (dev & 63);
    if (e == cudaSuccess && !(done.load(std::memory_order_relaxed) & bit)) {
        e = cudaFuncSetAttribute(paged_attn_kernel<C, D, NT, F32Q>, cudaFuncAttributeMaxDynamicSharedMemorySize, X::SMEM);
        if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    }
    if (e != cudaSuccess) return e;
    const unsigned grid = static_cast<unsigned>(rows * kv.kv_heads * a.head_tiles * a.splits);
    return launch_kernel(paged_attn_kernel<C, D, NT, F32Q>, dim3(grid), dim3(X::THREADS), X::SMEM, stream, true, a, kv);
}

// What the split's estimate knows of the kernel that a cache type, head size and
// query type get: CTAs an SM holds, the positions of a unit, the bytes an element
// weighs in an SM that holds several (Q8_0: half as much again, its
// instructions take longer than its bytes), and the time of a unit in a CTA that has an SM to itself
// (measured on B200: f32 0.95 us with heads of 64 and 1.5 with 128, 16-bit types 0.60
// with 128 and 0.83 with 256, Q8_0 0.88 with 64 and 1.27 with 128).
struct AttnShape {
    int per_sm, unit;
    float bytes, lone;
};

template <Elem C, int D, bool F32Q>
AttnShape attn_shape_as(int nt) {
    const float bytes = C == Elem::Q8 ? 1.5f * 34 / 32 : ElemOf<C>::bytes;
    const float each = C == Elem::F32 ? 82e-6f : C == Elem::Q8 ? 32e-6f : 24.5e-6f;  // us an element
    auto of = [&](auto x) -> AttnShape { return {x.PER_SM, x.UNIT, bytes, 0.25f + each * x.UNIT * 2 * D}; };
    return nt == 1 ? of(AttnCfg<C, D, 1, F32Q>{}) : of(AttnCfg<C, D, 2, F32Q>{});
}

// One function per cache type (paged_attn_<type>.cu): the launch, or with `shape`
// given only the geometry.
template <Elem C, bool F32Q>
cudaError_t attn_of_type(const AttnArgs* a, const PagesView& kv, int nt, int64_t rows, cudaStream_t st, AttnShape* shape) {
    auto go = [&](auto d) {
        constexpr int D = decltype(d)::value;
        if (shape) {
            *shape = attn_shape_as<C, D, F32Q>(nt);
            return cudaSuccess;
        }
        return nt == 1 ? launch_attn_as<C, D, 1, F32Q>(*a, kv, rows, st) : launch_attn_as<C, D, 2, F32Q>(*a, kv, rows, st);
    };
    if (kv.dim == 64) return go(std::integral_constant<int, 64>{});
    if (kv.dim == 128) return go(std::integral_constant<int, 128>{});
    return go(std::integral_constant<int, 256>{});
}

cudaError_t attn_f32(const AttnArgs* a, const PagesView& kv, int nt, int64_t rows, cudaStream_t st, AttnShape* shape);
cudaError_t attn_f16(const AttnArgs* a, const PagesView& kv, bool f32q, int nt, int64_t rows, cudaStream_t st, AttnShape* shape);
cudaError_t attn_bf16(const AttnArgs* a, const PagesView& kv, bool f32q, int nt, int64_t rows, cudaStream_t st, AttnShape* shape);
cudaError_t attn_q8(const AttnArgs* a, const PagesView& kv, bool f32q, int nt, int64_t rows, cudaStream_t st, AttnShape* shape);

}  // namespace tir
