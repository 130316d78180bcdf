// paged_attn_f16.cu -- the decode attention kernels of f16 caches.
#include "paged_attn.cuh"

namespace tir {

cudaError_t attn_f16(const AttnArgs* a, const PagesView& kv, bool f32q, int nt, int64_t rows, cudaStream_t st,
                   AttnShape* shape) {
    return f32q ? attn_of_type<Elem::F16, true>(a, kv, nt, rows, st, shape)
                : attn_of_type<Elem::F16, false>(a, kv, nt, rows, st, shape);
}

}  // namespace tir
