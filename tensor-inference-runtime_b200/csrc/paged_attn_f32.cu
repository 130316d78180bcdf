// paged_attn_f32.cu -- the decode attention kernels of f32 caches.
#include "paged_attn.cuh"

namespace tir {

cudaError_t attn_f32(const AttnArgs* a, const PagesView& kv, int nt, int64_t rows, cudaStream_t st, AttnShape* shape) {
    return attn_of_type<Elem::F32, true>(a, kv, nt, rows, st, shape);
}

}  // namespace tir
