// paged.h -- internals shared by the paged key-value cache operators
// (paged_kv.cu: per-head norm and rotation, cache write, read-back;
// paged_attn*.cu: decode attention).
#pragma once
#include <cuda_runtime.h>

#include <cstdint>
#include <string>

#include "host.h"

namespace tir {

// Element types as the kernels see them.
enum class Elem : int32_t { F32 = 0, F16 = 1, BF16 = 2, Q8 = 3 };

// A tir_kv_pages as the kernels take it.  Offsets are in elements and 64-bit:
// a pool may hold more than 2^32 of them.
struct PagesView {
    char *k, *v;
    uint16_t *ks, *vs;  // Q8: f16 step of 32 elements at (element offset) / 32
    const int32_t* table;
    int64_t table_rows, table_stride, n_pages;
    int64_t page_stride, pos_stride, head_stride;
    int32_t max_pages, page_size, page_shift;  // shift: log2(page_size), -1 where it is no power of two
    int32_t kv_heads, dim;
    uint32_t page16, pos16, head16;  // the strides of the pools in 16-byte units
    uint32_t* err;  // sticky bits, kBad*
};

// What a kernel found in device memory that no host check can see; the access
// is skipped and the bit kept until tir_ops_check reports it.
constexpr uint32_t kBadPosition = 1u;  // a position or sequence outside the table
constexpr uint32_t kBadPage = 2u;      // a page id outside the pool
constexpr uint32_t kBadLength = 4u;    // a length above what the table can hold

// Activation types (F32, F16, BF16) and cache types of the C interface; false
// for any other code.
bool act_elem(int32_t dtype, Elem* out);
// Checks a cache description and fills the kernels' view of it.  `entry` names
// the caller in the message.
tir_status pages_view(const tir_kv_pages* kv, const char* entry, PagesView* view, Elem* type);
// `p` and `stride` (elements between tokens) must keep 16-byte alignment.
tir_status check_rows(const void* p, int64_t stride, int64_t heads, int64_t dim, Elem e, const char* entry,
                      const char* what);
// The error word of the current device (looked up on its first use there).
tir_status paged_error_word(uint32_t** out);
// Takes the error word of `device`, the current one, on `stream` and waits; 0 where no
// paged operator ran on it.
tir_status paged_take_error(int device, void* stream, uint32_t* bits);
tir_status paged_fail(cudaError_t e, const char* what);

}  // namespace tir
