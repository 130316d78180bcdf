// paged_kv.cu -- the operators that fill and read back a paged key-value
// cache: per-head RMS norm and position rotation of queries and keys, the
// conversion or Q8_0 quantisation of keys and values as they are written to
// their pages, and the read-back of cached positions as rows.
//
// Every head vector of dim = 64, 128 or 256 elements is held by dim / 8 lanes
// of one warp, eight elements (one or two 16-byte accesses) each, so the norm's
// sum, the rotation's partner and a block's maximum are shuffles and every
// element crosses memory once in and once out: the kernels are bound by memory.
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <mutex>
#include <string>
#include <vector>

#include "paged.cuh"
#include "paged.h"
#include "ptx.cuh"

namespace tir {

static __device__ uint32_t g_paged_err;

namespace {

constexpr uint32_t FULL = 0xffffffffu;
constexpr int kRowThreads = 256;
constexpr int kMaxDevices = 64;

std::mutex g_err_mu;
uint32_t* g_err_ptr[kMaxDevices];

struct RowArgs {
    const char *q, *k, *v;
    char *q_out, *k_out;
    int64_t q_stride, k_stride, v_stride, q_out_stride, k_out_stride;  // bytes between tokens
    const int32_t *seqs, *positions;
    int64_t tokens;
    int32_t q_heads, kv_heads;
    int32_t heads;  // of a token: q_heads + kv_heads (+ kv_heads values, when appending)
    const float *q_w, *k_w, *rope;
    int64_t rope_positions;
    int32_t rope_dim, pairs;
    float eps;
    uint32_t* err;
};

// One Q8_0 block's rule (activated_q8, src/kernels.rs:8-31) over the four lanes
// that hold its 32 values: step = the last of the elements of largest |x| / 127,
// quants = round half away (x / step), saturated, NaN -> 0.  The quotient uses
// the step before it is rounded to f16, as there.  IEEE divisions keep the
// quants equal to tir_activated_q8's.
__device__ __forceinline__ void quantise8(const float* f, int lane4, uint2* quants, float* step) {
    uint32_t top = 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(f[i]) & 0x7fffffffu);
    top = max(top, __shfl_xor_sync(FULL, top, 1));
    top = max(top, __shfl_xor_sync(FULL, top, 2));
    uint32_t last = 0u;  // 2 (index + 1) + sign of the last element of magnitude `top`
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if ((__float_as_uint(f[i]) & 0x7fffffffu) == top) last = 2u * (lane4 * 8 + i + 1) + (__float_as_uint(f[i]) >> 31);
    last = max(last, __shfl_xor_sync(FULL, last, 1));
    last = max(last, __shfl_xor_sync(FULL, last, 2));
    const float d = __fdiv_rn(__uint_as_float(top | (last << 31)), 127.0f);
    uint32_t b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float r = roundf(__fdiv_rn(f[i], d));
        const int n = r != r ? 0 : static_cast<int>(fminf(fmaxf(r, -128.f), 127.f));
        b[i] = static_cast<uint32_t>(n) & 0xffu;
    }
    quants->x = b[0] | (b[1] << 8) | (b[2] << 16) | (b[3] << 24);
    quants->y = b[4] | (b[5] << 8) | (b[6] << 16) | (b[7] << 24);
    *step = d;
}

// Writes this lane's eight elements of a head to element offset `at` of a pool.
// Every lane of the warp calls it (the block maxima are shuffles).
__device__ __forceinline__ void store_cache8(const float* f, bool live, Elem type, char* pool, uint16_t* scales,
                                             int64_t at, int gl) {
    if (type == Elem::Q8) {
        uint2 w;
        float step;
        quantise8(f, gl & 3, &w, &step);
        if (live) {
            *reinterpret_cast<uint2*>(pool + at) = w;
            if ((gl & 3) == 0) scales[at >> 5] = __half_as_ushort(__float2half_rn(step));
        }
    } else if (live) {
        if (type == Elem::F32)
            store8_as<Elem::F32>(pool + at * 4, f);
        else if (type == Elem::F16)
            store8_as<Elem::F16>(pool + at * 2, f);
        else
            store8_as<Elem::BF16>(pool + at * 2, f);
    }
}

// Group of D / 8 lanes per (token, head).  kAppend: keys and values go to the
// cache, else keys go to rows and there are no values.
template <Elem A, int D, bool kAppend>
__global__ void __launch_bounds__(kRowThreads) rows_kernel(const RowArgs a, const PagesView kv, const Elem cache) {
    constexpr int G = D / 8;
    constexpr int AB = ElemOf<A>::bytes;
    const int gl = threadIdx.x % G;
    const int64_t item = (blockIdx.x * static_cast<int64_t>(kRowThreads) + threadIdx.x) / G;
    const int64_t t = item / a.heads;
    const int h = static_cast<int>(item % a.heads);
    bool live = t < a.tokens;
    const int32_t pos = live && a.positions ? a.positions[t] : 0;
    if (pos < 0) live = false;
    const bool is_q = h < a.q_heads, is_k = !is_q && h < a.q_heads + a.kv_heads;
    const int hk = is_q ? h : is_k ? h - a.q_heads : h - a.q_heads - a.kv_heads;
    const bool turns = a.rope && (is_q || is_k);
    if (live && a.rope && pos >= a.rope_positions) {
        if (gl == 0) atomicOr(a.err, kBadPosition);
        live = false;
    }
    // where it goes
    int64_t at = 0;
    if (kAppend && live && !is_q) {
        const int64_t row = a.seqs ? a.seqs[t] : t;
        const int64_t cap = static_cast<int64_t>(kv.max_pages) * kv.page_size;
        if (row < 0 || row >= kv.table_rows || pos >= cap) {
            if (gl == 0) atomicOr(a.err, kBadPosition);
            live = false;
        } else {
            const int32_t id = page_of(kv, row, pos);
            live = id >= 0;
            at = slot_of(kv, id, pos) + hk * kv.head_stride + gl * 8;
        }
    }
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = 0.f;
    if (live) {
        const char* src = is_q ? a.q + t * a.q_stride : is_k ? a.k + t * a.k_stride : a.v + t * a.v_stride;
        expand8<A>(load_raw8<A>(src + (static_cast<int64_t>(hk) * D + gl * 8) * AB), f);
    }
    const float* w = is_q ? a.q_w : is_k ? a.k_w : nullptr;
    // the lanes of a group share the branch; the shuffles stay outside it, a
    // warp may hold groups of either kind
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(f[i], f[i], ss);
#pragma unroll
    for (int o = G / 2; o; o >>= 1) ss += __shfl_xor_sync(FULL, ss, o);
    if (w) {
        const float rms = __fsqrt_rn(__fadd_rn(__fdiv_rn(ss, static_cast<float>(D)), a.eps));
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = __fdiv_rn(__fmul_rn(f[i], w[gl * 8 + i]), rms);
    }
    const int half8 = a.rope_dim / 16;  // lanes of one half of the rotated elements
    const int mate = a.pairs == TIR_PAIRS_HALVES && gl < 2 * half8 ? (gl < half8 ? gl + half8 : gl - half8) : gl;
    float g[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) g[i] = __shfl_sync(FULL, f[i], mate, G);
    if (live && turns && gl < 2 * half8) {
        const float* cs = a.rope + static_cast<int64_t>(pos) * a.rope_dim;
        if (a.pairs == TIR_PAIRS_ADJACENT) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float c = cs[gl * 8 + 2 * i], s = cs[gl * 8 + 2 * i + 1];
                const float x = f[2 * i], y = f[2 * i + 1];
                f[2 * i] = __fadd_rn(__fmul_rn(c, x), __fmul_rn(-s, y));
                f[2 * i + 1] = __fadd_rn(__fmul_rn(s, x), __fmul_rn(c, y));
            }
        } else {
            const bool upper = gl >= half8;
            const float* cp = cs + (upper ? gl - half8 : gl) * 16;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float c = cp[2 * i], s = upper ? cp[2 * i + 1] : -cp[2 * i + 1];
                f[i] = __fadd_rn(__fmul_rn(c, f[i]), __fmul_rn(s, g[i]));
            }
        }
    }
    if (kAppend) {
        const bool write = live && !is_q;
        store_cache8(f, write, cache, is_k ? kv.k : kv.v, is_k ? kv.ks : kv.vs, at, gl);
    }
    if (live && (is_q || !kAppend)) {
        char* dst = is_q ? a.q_out + t * a.q_out_stride : a.k_out + t * a.k_out_stride;
        store8_as<A>(dst + (static_cast<int64_t>(hk) * D + gl * 8) * AB, f);
    }
}

// Group of D / 8 lanes per (token, key or value, head): cache -> rows.
template <Elem A, int D>
__global__ void __launch_bounds__(kRowThreads) gather_kernel(const RowArgs a, const PagesView kv, const Elem cache) {
    constexpr int G = D / 8;
    constexpr int AB = ElemOf<A>::bytes;
    const int gl = threadIdx.x % G;
    const int64_t item = (blockIdx.x * static_cast<int64_t>(kRowThreads) + threadIdx.x) / G;
    const int64_t t = item / a.heads;
    if (t >= a.tokens) return;
    const int h = static_cast<int>(item % a.heads);
    const bool is_k = h < a.kv_heads;
    const int hk = is_k ? h : h - a.kv_heads;
    const int32_t pos = a.positions[t];
    if (pos < 0) return;
    const int64_t row = a.seqs ? a.seqs[t] : t;
    const int64_t cap = static_cast<int64_t>(kv.max_pages) * kv.page_size;
    if (row < 0 || row >= kv.table_rows || pos >= cap) {
        if (gl == 0) atomicOr(a.err, kBadPosition);
        return;
    }
    const int32_t id = page_of(kv, row, pos);
    if (id < 0) return;
    const int64_t at = slot_of(kv, id, pos) + hk * kv.head_stride + gl * 8;
    const char* pool = is_k ? kv.k : kv.v;
    float f[8];
    if (cache == Elem::Q8) {
        const uint2 w = *reinterpret_cast<const uint2*>(pool + at);
        const float step = __half2float(__ushort_as_half((is_k ? kv.ks : kv.vs)[at >> 5]));
        expand_q8x4(w.x, step, f);
        expand_q8x4(w.y, step, f + 4);
    } else if (cache == Elem::F32) {
        expand8<Elem::F32>(load_raw8<Elem::F32>(pool + at * 4), f);
    } else if (cache == Elem::F16) {
        expand8<Elem::F16>(load_raw8<Elem::F16>(pool + at * 2), f);
    } else {
        expand8<Elem::BF16>(load_raw8<Elem::BF16>(pool + at * 2), f);
    }
    char* dst = is_k ? a.q_out + t * a.q_out_stride : a.k_out + t * a.k_out_stride;
    store8_as<A>(dst + (static_cast<int64_t>(hk) * D + gl * 8) * AB, f);
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

bool grid_of(const RowArgs& a, int32_t dim, unsigned* grid) {
    const int64_t per = kRowThreads / (dim / 8);
    const int64_t n = (a.tokens * a.heads + per - 1) / per;
    *grid = static_cast<unsigned>(n);
    return n <= INT32_MAX;
}

template <bool kAppend>
tir_status launch_rows(const RowArgs& a, const PagesView& kv, Elem act, Elem cache, int32_t dim, void* stream,
                       const char* entry) {
    unsigned grid;
    if (!grid_of(a, dim, &grid)) return fail(TIR_ERR_UNSUPPORTED_SHAPE, std::string(entry) + ": too many tokens");
    const cudaError_t e = by_type(act, dim, [&](auto el, auto d) {
        rows_kernel<decltype(el)::value, decltype(d)::value, kAppend>
            <<<grid, kRowThreads, 0, static_cast<cudaStream_t>(stream)>>>(a, kv, cache);
        return cudaGetLastError();
    });
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

tir_status paged_take_error(int device, uint32_t* bits) {
    *bits = 0u;
    uint32_t* p = nullptr;
    {
        std::lock_guard<std::mutex> lock(g_err_mu);
        if (device >= 0 && device < kMaxDevices) p = g_err_ptr[device];
    }
    if (!p) return TIR_OK;
    cudaError_t e = cudaMemcpy(bits, p, sizeof(uint32_t), cudaMemcpyDeviceToHost);
    if (e == cudaSuccess && *bits) e = cudaMemset(p, 0, sizeof(uint32_t));
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
    a.heads = q_heads + kv_heads;
    set_norm(&a, norm);
    rc = paged_error_word(&a.err);
    if (rc != TIR_OK) return rc;
    return launch_rows<false>(a, PagesView{}, act, Elem::F32, dim, stream, who);
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
    a.heads = q_heads + 2 * kv->kv_heads;
    if (norm) set_norm(&a, norm);
    rc = paged_error_word(&a.err);
    if (rc != TIR_OK) return rc;
    view.err = a.err;
    return launch_rows<true>(a, view, act, cache, kv->dim, stream, who);
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
    a.heads = 2 * kv->kv_heads;
    rc = paged_error_word(&a.err);
    if (rc != TIR_OK) return rc;
    view.err = a.err;
    unsigned grid;
    if (!grid_of(a, kv->dim, &grid)) return fail(TIR_ERR_UNSUPPORTED_SHAPE, std::string(who) + ": too many tokens");
    const cudaError_t e = by_type(act, kv->dim, [&](auto el, auto d) {
        gather_kernel<decltype(el)::value, decltype(d)::value>
            <<<grid, kRowThreads, 0, static_cast<cudaStream_t>(stream)>>>(a, view, cache);
        return cudaGetLastError();
    });
    return e == cudaSuccess ? TIR_OK : paged_fail(e, who);
}

}  // extern "C"
