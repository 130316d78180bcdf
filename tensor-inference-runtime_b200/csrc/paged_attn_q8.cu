// paged_attn_q8.cu -- the decode attention kernels of Q8_0 caches.
#include "paged_attn.cuh"

namespace tir {

cudaError_t attn_q8(const AttnArgs* a, const PagesView& kv, bool f32q, int nt, int64_t rows, cudaStream_t st,
                   AttnShape* shape) {
    return f32q ? attn_of_type<Elem::Q8, true>(a, kv, nt, rows, st, shape)
                : attn_of_type<Elem::Q8, false>(a, kv, nt, rows, st, shape);
}

}  // namespace tir
