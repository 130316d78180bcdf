// paged_attn.cu -- attention of one query token per sequence over its pages.
//
// One warp per (row, query head): every lane holds dim / 32 neighbouring
// elements of the query and the running output; the scores of a position are a
// warp sum, the softmax keeps a running maximum and sum (base 2) in f32.
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <string>

#include "paged.cuh"
#include "paged.h"

namespace tir {

namespace {

constexpr uint32_t FULL = 0xffffffffu;

struct AttnArgs {
    const char* q;
    char* out;
    int64_t q_stride, out_stride;  // elements
    const int32_t* lens;
    int64_t rows;
    int32_t q_heads, group;
    int32_t window;  // INT32_MAX: none
    float scale_log2;
    Elem act, cache;
};

__device__ __forceinline__ float load_elem(const char* p, int64_t i, Elem e) {
    if (e == Elem::F32) return reinterpret_cast<const float*>(p)[i];
    if (e == Elem::F16) return __half2float(reinterpret_cast<const __half*>(p)[i]);
    return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
}

__device__ __forceinline__ float load_cached(const char* pool, const uint16_t* steps, int64_t i, Elem e) {
    if (e == Elem::Q8)
        return __fmul_rn(static_cast<float>(reinterpret_cast<const int8_t*>(pool)[i]),
                         __half2float(__ushort_as_half(steps[i >> 5])));
    return load_elem(pool, i, e);
}

template <int D>
__global__ void __launch_bounds__(32) attn_kernel(const AttnArgs a, const PagesView kv) {
    constexpr int N = D / 32;
    const int64_t row = blockIdx.x / a.q_heads;
    const int h = static_cast<int>(blockIdx.x % a.q_heads);
    const int g = h / a.group, lane = threadIdx.x;
    const int64_t cap = static_cast<int64_t>(kv.max_pages) * kv.page_size;
    int32_t len = a.lens[row];
    if (len < 0 || len > cap) {
        if (lane == 0) atomicOr(kv.err, kBadLength);
        len = len < 0 ? 0 : static_cast<int32_t>(cap);
    }
    float q[N], o[N], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        q[i] = load_elem(a.q, row * a.q_stride + h * D + lane * N + i, a.act) * a.scale_log2;
        o[i] = 0.f;
    }
    for (int32_t pos = len > a.window ? len - a.window : 0; pos < len; ++pos) {
        const int32_t id = page_of(kv, row, pos);
        if (id < 0) continue;
        const int64_t at = slot_of(kv, id, pos) + g * kv.head_stride + lane * N;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) s = fmaf(q[i], load_cached(kv.k, kv.ks, at + i, a.cache), s);
#pragma unroll
        for (int w = 16; w; w >>= 1) s += __shfl_xor_sync(FULL, s, w);
        const float mn = fmaxf(m, s), safe = mn == -INFINITY ? 0.f : mn;
        const float corr = exp2f(m - safe), p = exp2f(s - safe);
        l = l * corr + p;
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] = fmaf(p, load_cached(kv.v, kv.vs, at + i, a.cache), o[i] * corr);
        m = mn;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float r = len == 0 ? 0.f : o[i] / l;
        const int64_t at = row * a.out_stride + h * D + lane * N + i;
        if (a.act == Elem::F32)
            reinterpret_cast<float*>(a.out)[at] = r;
        else if (a.act == Elem::F16)
            reinterpret_cast<__half*>(a.out)[at] = __float2half_rn(r);
        else
            reinterpret_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(r);
    }
}

}  // namespace
}  // namespace tir

using namespace tir;

static tir_status check_sizes(const tir_kv_pages* kv, int64_t rows, int32_t q_heads, int64_t max_len, int64_t window,
                              PagesView* view, Elem* cache) {
    const char* who = "tir_paged_attention";
    const tir_status rc = pages_view(kv, who, view, cache);
    if (rc != TIR_OK) return rc;
    if (rows < 0 || rows > kv->table_rows || q_heads <= 0 || q_heads > (1 << 20) || q_heads % kv->kv_heads || max_len < 0 ||
        window < 0)
        return fail(TIR_ERR_INVALID_ARG, std::string(who) + ": bad sizes");
    if (rows * q_heads > INT32_MAX) return fail(TIR_ERR_UNSUPPORTED_SHAPE, std::string(who) + ": too many rows");
    return TIR_OK;
}

extern "C" {

int64_t tir_paged_attention_workspace(const tir_kv_pages* kv, int64_t rows, int32_t q_heads, int64_t max_len,
                                      int64_t window) {
    clear_error();
    Elem cache;
    PagesView view;
    if (check_sizes(kv, rows, q_heads, max_len, window, &view, &cache) != TIR_OK) return -1;
    return 0;
}

tir_status tir_paged_attention(const void* q, int64_t q_stride, const tir_kv_pages* kv, const int32_t* seq_lens,
                               void* out, int64_t out_stride, int64_t rows, int32_t q_heads, int32_t dtype,
                               float scale, int64_t max_len, int64_t window, void* workspace, int64_t workspace_bytes,
                               void* stream) {
    clear_error();
    (void)workspace;
    (void)workspace_bytes;
    const char* who = "tir_paged_attention";
    Elem act, cache;
    PagesView view;
    if (!act_elem(dtype, &act)) return fail(TIR_ERR_UNSUPPORTED_DTYPE, std::string(who) + ": activations must be F32, F16 or BF16");
    tir_status rc = check_sizes(kv, rows, q_heads, max_len, window, &view, &cache);
    if (rc != TIR_OK) return rc;
    if (act != Elem::F32 && cache != act && cache != Elem::Q8)
        return fail(TIR_ERR_UNSUPPORTED_DTYPE, std::string(who) + ": 16-bit queries need a cache of their type or Q8_0");
    if (!(scale >= 0.f) || std::isinf(scale)) return fail(TIR_ERR_INVALID_ARG, std::string(who) + ": bad scale");
    if (rows == 0) return TIR_OK;
    if (!seq_lens) return fail(TIR_ERR_INVALID_ARG, std::string(who) + ": null lengths");
    rc = check_rows(q, q_stride, q_heads, kv->dim, act, who, "q");
    if (rc == TIR_OK) rc = check_rows(out, out_stride, q_heads, kv->dim, act, who, "out");
    if (rc != TIR_OK) return rc;
    rc = paged_error_word(&view.err);
    if (rc != TIR_OK) return rc;
    AttnArgs a{};
    a.q = static_cast<const char*>(q);
    a.out = static_cast<char*>(out);
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.lens = seq_lens;
    a.rows = rows;
    a.q_heads = q_heads;
    a.group = q_heads / kv->kv_heads;
    a.window = window > 0 && window < INT32_MAX ? static_cast<int32_t>(window) : INT32_MAX;
    const float sc = scale == 0.f ? 1.0f / std::sqrt(static_cast<float>(kv->dim)) : scale;
    a.scale_log2 = sc * 1.44269504088896340736f;
    a.act = act;
    a.cache = cache;
    const unsigned grid = static_cast<unsigned>(rows * q_heads);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (kv->dim == 64)
        attn_kernel<64><<<grid, 32, 0, st>>>(a, view);
    else if (kv->dim == 128)
        attn_kernel<128><<<grid, 32, 0, st>>>(a, view);
    else
        attn_kernel<256><<<grid, 32, 0, st>>>(a, view);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? TIR_OK : paged_fail(e, who);
}

}  // extern "C"
