// paged_attn.cu -- tir_paged_attention: the choice of kernel and split, and the
// kernel that joins the parts of rows shared by several CTAs.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>

#include "launch.cuh"
#include "paged_attn.cuh"

namespace tir {

namespace {

constexpr int kJoinWarps = 4;

// o = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i over the parts of one (row,
// head).  A CTA per head; warp w takes parts w, w + 4, ..., lanes the dimensions.
// Reads what the split wrote (L2), a few percent of the cache's bytes at most.
template <int D>
__global__ void __launch_bounds__(kJoinWarps * 32) paged_attn_join(const AttnArgs a, const PagesView kv, int32_t unit) {
    constexpr int N = D / 32;
    __shared__ float part[kJoinWarps][D];
    __shared__ float sums[kJoinWarps];
    griddep_wait();
    const int64_t row = blockIdx.x / a.q_heads;
    const int h = static_cast<int>(blockIdx.x % a.q_heads);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const AttnRange range = attn_range(row_length(a, kv, row), a.window, a.splits, a.min_units, unit, 0);
    if (range.used <= 1) return;  // written by the split itself
    const float* ml = a.part_ml + (row * a.q_heads + h) * a.splits * 2;
    const float* po = a.part_o + (row * a.q_heads + h) * a.splits * D + lane * N;
    float top = -INFINITY;
    for (int i = lane; i < range.used; i += 32) top = fmaxf(top, ml[2 * i]);
#pragma unroll
    for (int w = 16; w; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
    float o[N], l = 0.f;
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] = 0.f;
#pragma unroll 4
    for (int i = warp; i < range.used; i += kJoinWarps) {
        const float2 x = *reinterpret_cast<const float2*>(ml + 2 * i);
        const float f = part_factor(x.x, top);
        l = fmaf(f, x.y, l);
#pragma unroll
        for (int e = 0; e < N; e += 2) {
            const float2 v = *reinterpret_cast<const float2*>(po + static_cast<int64_t>(i) * D + e);
            o[e] = fmaf(f, v.x, o[e]);
            o[e + 1] = fmaf(f, v.y, o[e + 1]);
        }
    }
#pragma unroll
    for (int e = 0; e < N; ++e) part[warp][lane * N + e] = o[e];
    if (lane == 0) sums[warp] = l;
    __syncthreads();
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) sum += sums[w];
    sum = part_sum(sum, top);
    for (int d = threadIdx.x; d < D; d += kJoinWarps * 32) {
        float y = 0.f;
#pragma unroll
        for (int w = 0; w < kJoinWarps; ++w) y += part[w][d];
        y /= sum;
        const int64_t at = row * a.out_stride + static_cast<int64_t>(h) * D + d;
        if (a.act == Elem::F32)
            reinterpret_cast<float*>(a.out)[at] = y;
        else if (a.act == Elem::F16)
            reinterpret_cast<__half*>(a.out)[at] = __float2half_rn(y);
        else
            reinterpret_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(y);
    }
}

cudaError_t attn(const AttnArgs* a, const PagesView& kv, Elem cache, bool f32q, int nt, int64_t rows, cudaStream_t st,
                 AttnShape* shape) {
    switch (cache) {
        case Elem::F32: return attn_f32(a, kv, nt, rows, st, shape);
        case Elem::F16: return attn_f16(a, kv, f32q, nt, rows, st, shape);
        case Elem::BF16: return attn_bf16(a, kv, f32q, nt, rows, st, shape);
        default: return attn_q8(a, kv, f32q, nt, rows, st, shape);
    }
}

int multiprocessors() {
    static thread_local int dev_of = -1, n_of = 0;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 0;
    if (dev != dev_of) {
        int n = 0;
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
        dev_of = dev;
        n_of = n;
    }
    return n_of;
}

struct Plan {
    int nt, head_tiles, sms;
    AttnShape shape;
    int64_t units, slots;  // of the longest row; CTAs the GPU holds
    int32_t splits, min_units;
};

// What the sizes alone give.
tir_status make_shape(const PagesView& kv, Elem cache, bool f32q, int64_t rows, int32_t q_heads, int64_t max_len,
                      int64_t window, Plan* p) {
    const int group = q_heads / kv.kv_heads;
    p->nt = group <= 8 ? 1 : 2;
    p->head_tiles = (group + 8 * p->nt - 1) / (8 * p->nt);
    attn(nullptr, kv, cache, f32q, p->nt, rows, nullptr, &p->shape);
    p->sms = multiprocessors();
    if (p->sms <= 0) return fail(TIR_ERR_CUDA, "tir_paged_attention: no multiprocessor count for the current device");
    int64_t n = static_cast<int64_t>(kv.max_pages) * kv.page_size;
    if (max_len > 0) n = std::min(n, max_len);
    if (window > 0) n = std::min(n, window);
    p->units = (n + p->shape.unit - 1) / p->shape.unit;
    p->slots = static_cast<int64_t>(p->sms) * p->shape.per_sm;
    return TIR_OK;
}

// Parts beyond the first that a call may be divided into, in CTAs the GPU holds.
constexpr int64_t kMostParts = 8;

// Bytes that hold the parts of any call of these sizes or smaller ones.  The count of parts
// that suits a call best goes up and down with its rows, so this takes what make_plan
// looks at: rows * heads * (s - 1) <= kMostParts * slots, s <= units.
int64_t workspace_of(const Plan& p, const PagesView& kv, int64_t rows, int32_t q_heads) {
    if (p.units <= 1) return 0;
    const int64_t most = kMostParts * p.slots / (kv.kv_heads * p.head_tiles), r = std::min(rows, most);
    return std::min(most + r, r * p.units) * q_heads * (kv.dim + 2) * 4;
}

// How many CTAs share a row's head (s).  The time of a call is estimated twice,
// for rows that are all of the longest length (waves of a start and a part's units)
// and for rows spread evenly below it (all units over the GPU, starts, half a
// longest part), and the s with the least sum of the two, each over its least, is
// taken: the lengths are on the device, and a count that suits both costs either
// little.  Measured on B200, the choice first: 64 rows x 4 heads x 2048 positions in f32
// take 49 us with s = 1, 56 with 3, 62 with 4; 64 rows x 8 heads up to 8192 in bf16 174 with
// 4, 198 with 1, 190 with 12; one row of 16000 beside 63 of 300 45 with 5, 176 with 1, 40 with
// 6; one row of 131071 87 with 18, 1303 with 1, 94 with 37.
constexpr float kStart = 2.0f, kJoin = 2.3f, kJoinRow = 1.0f / 1200.0f;  // us
constexpr float kBytesPerUs = 6.2e6f;

struct SplitTime {
    float even, ragged;
};

SplitTime split_time(int64_t items, int64_t units, int64_t s, int64_t slots, float unit_sm, float lone, int sms, int64_t heads) {
    const int64_t per = (units + s - 1) / s, parts = (units + per - 1) / per, n = items * parts;
    auto wave = [&](int64_t ctas) { return kStart + per * std::max(lone, unit_sm * static_cast<float>(ctas) / sms); };
    const float join = parts > 1 ? kJoin + kJoinRow * heads : 0.f;
    SplitTime t;
    t.even = static_cast<float>(n / slots) * wave(slots) + (n % slots ? wave(n % slots) : 0.f) + join;
    const float all = 0.5f * items * units * unit_sm / sms, longest = kStart + per * lone;
    t.ragged = std::max(all + 0.5f * per * lone, longest) + kStart * 0.35f * items * (parts + 1) / slots + join;
    return t;
}

tir_status make_plan(const PagesView& kv, Elem cache, bool f32q, int64_t rows, int32_t q_heads, int64_t max_len,
                     int64_t window, Plan* p) {
    const tir_status rc = make_shape(kv, cache, f32q, rows, q_heads, max_len, window, p);
    if (rc != TIR_OK) return rc;
    const int sms = p->sms;
    const int64_t units = p->units, slots = p->slots;
    const int64_t items = std::max<int64_t>(rows * kv.kv_heads * p->head_tiles, 1);
    const float unit_sm = static_cast<float>(p->shape.unit * kv.dim * 2 * p->shape.bytes * sms / kBytesPerUs);
    int64_t tries[48];
    SplitTime times[48];
    int n_tries = 0;
    float even = 1e30f, ragged = 1e30f;
    auto consider = [&](int64_t s) {
        if (n_tries == 48) return;
        const SplitTime t = split_time(items, units, s, slots, unit_sm, p->shape.lone, sms, rows * q_heads);
        even = std::min(even, t.even);
        ragged = std::min(ragged, t.ragged);
        times[n_tries] = t;
        tries[n_tries++] = s;
    };
    for (int64_t w = 1; w <= 3; ++w)  // parts that fill whole waves
        if (const int64_t s = w * slots / items; s > 1 && s <= units) consider(s);
    for (int64_t s = 1; s <= units && (s - 1) * items <= kMostParts * slots; s += 1 + s / 6) consider(s);
    int64_t best = 1;
    float least = 1e30f;
    for (int i = 0; i < n_tries; ++i) {
        const float cost = times[i].even / even + (rows > 1 ? times[i].ragged / ragged : 0.f);
        if (cost < least || (cost == least && tries[i] < best)) {
            least = cost;
            best = tries[i];
        }
    }
    if (items * best > INT32_MAX) return fail(TIR_ERR_UNSUPPORTED_SHAPE, "tir_paged_attention: too many rows");
    p->splits = static_cast<int32_t>(best);
    // shorter rows get fewer parts, down to half the length of the longest row's
    p->min_units = static_cast<int32_t>(std::max<int64_t>((units + best - 1) / best / 2, 1));
    return TIR_OK;
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
    // the query type may change the kernel's geometry: what either would need
    int64_t most = 0;
    for (const bool f32q : {false, true}) {
        Plan p;
        if (make_shape(view, cache, f32q, rows, q_heads, max_len, window, &p) != TIR_OK) return -1;
        most = std::max(most, workspace_of(p, view, rows, q_heads));
    }
    return most;
}

tir_status tir_paged_attention(const void* q, int64_t q_stride, const tir_kv_pages* kv, const int32_t* seq_lens,
                               void* out, int64_t out_stride, int64_t rows, int32_t q_heads, int32_t dtype,
                               float scale, int64_t max_len, int64_t window, void* workspace, int64_t workspace_bytes,
                               void* stream) {
    clear_error();
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
    Plan p;
    rc = make_plan(view, cache, act == Elem::F32, rows, q_heads, max_len, window, &p);
    if (rc != TIR_OK) return rc;
    const int64_t need = p.splits > 1 ? workspace_of(p, view, rows, q_heads) : 0;
    if (need > 0 && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16))
        return fail(TIR_ERR_INVALID_ARG, std::string(who) + ": needs a 16-byte aligned workspace of " + std::to_string(need) + " bytes");
    AttnArgs a{};
    a.q = static_cast<const char*>(q);
    a.out = static_cast<char*>(out);
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.lens = seq_lens;
    a.q_heads = q_heads;
    a.group = q_heads / kv->kv_heads;
    a.head_tiles = p.head_tiles;
    a.window = window > 0 && window < INT32_MAX ? static_cast<int32_t>(window) : INT32_MAX;
    a.splits = p.splits;
    a.min_units = p.min_units;
    const float sc = scale == 0.f ? 1.0f / std::sqrt(static_cast<float>(kv->dim)) : scale;
    a.scale_log2 = sc * 1.44269504088896340736f;
    a.act = act;
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = a.part_o + (need > 0 ? rows * q_heads * p.splits * kv->dim : 0);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e = attn(&a, view, cache, act == Elem::F32, p.nt, rows, st, nullptr);
    if (e == cudaSuccess && p.splits > 1) {
        const dim3 grid(static_cast<unsigned>(rows * q_heads)), block(kJoinWarps * 32);
        auto* join = kv->dim == 64 ? paged_attn_join<64> : kv->dim == 128 ? paged_attn_join<128> : paged_attn_join<256>;
        e = launch_kernel(join, grid, block, 0, st, true, a, view, static_cast<int32_t>(p.shape.unit));
    }
    return e == cudaSuccess ? TIR_OK : paged_fail(e, who);
}

}  // extern "C"
