// Shared by the paged-cache kernels: index types, argument checks, page lookups.
//
// A pool holds num_pages pages per plane; a page is page_size cache rows of
// num_kv_heads * head_dim fp16 values.  Row b of a page table (max_pages int32
// entries) names the pages of sequence b in order: its cache row t lies in page
// table[b][t / page_size], row t % page_size.
#pragma once

#include "attn_internal.hpp"

namespace attn {

inline bool paged_u31(size_t v) { return v <= 0x7fffffffull; }

// a * b where it stays below 2^63 (sizes of buffers), else 0x8000000000000000
inline uint64_t paged_mul(uint64_t a, uint64_t b) {
    const unsigned __int128 p = (unsigned __int128)a * b;
    return p >> 63 ? 1ull << 63 : (uint64_t)p;
}

// Sizes every paged entry point takes: tables of num_seqs x max_pages entries over
// num_pages pages of page_size rows.  Row numbers of a pool and positions of a
// sequence stay within 31 bits; offsets in elements are 64-bit.
inline bool paged_sizes_ok(size_t num_seqs, size_t max_pages, size_t num_pages,
                           size_t page_size) {
    return paged_u31(num_seqs) && paged_u31(max_pages) && paged_u31(num_pages) && page_size > 0 &&
           paged_u31(page_size) && paged_mul(num_pages, page_size) <= 0x7fffffffull &&
           paged_mul(max_pages, page_size) <= 0x7fffffffull;
}

// pages that hold n rows (n >= 0)
__host__ __device__ __forceinline__ uint32_t pages_for(uint32_t n, uint32_t page_size) {
    return n == 0 ? 0u : (n - 1u) / page_size + 1u;
}

// a length read from device memory, held within what a table row can name
__device__ __forceinline__ uint32_t clamp_len(int32_t n, uint32_t max_pages, uint32_t page_size) {
    return n <= 0 ? 0u : min((uint32_t)n, max_pages * page_size);
}

}  // namespace attn
