// C++ launchers of the paged-cache and 4-bit entry points (attn_mi355x.h), beside the
// launchers of kernels.hpp: the same argument order and __half pointers, strides of 0 for
// packed rows, a trailing stream.  They have no counterpart in the reference.  A call that
// the library rejects, or a launch that fails, throws std::runtime_error naming the
// launcher and the HIP error; sizes of zero launch nothing.
#pragma once
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>
#include <stdexcept>
#include <string>

#include "../attn_mi355x.h"

namespace paged_detail {
inline attn_f16_t* bits(__half* p) { return reinterpret_cast<attn_f16_t*>(p); }
inline const attn_f16_t* bits(const __half* p) { return reinterpret_cast<const attn_f16_t*>(p); }
inline void report(int rc, const char* launcher) {
    if (rc != 0)
        throw std::runtime_error(std::string("attn_mi355x: ") + launcher + " failed: " +
                                 hipGetErrorString((hipError_t)rc) + " (" + std::to_string(rc) +
                                 ")");
}
}  // namespace paged_detail

// attn_paged_rope_store_kv: new tokens' queries and keys rotated, keys and values into pages
inline void launch_paged_rope_and_store_kv(
    __half* d_q, const __half* d_k, const __half* d_v, __half* d_q_out, __half* d_k_pages,
    __half* d_v_pages, const __half* d_cos, const __half* d_sin, const int32_t* d_page_table,
    const int32_t* d_seq_ids, const int32_t* d_positions, size_t num_tokens, size_t num_seqs,
    size_t max_pages, size_t num_pages, size_t page_size, size_t max_seq_len, size_t num_heads,
    size_t num_kv_heads, size_t head_dim, size_t q_stride, size_t k_stride, bool apply_rotation,
    hipStream_t stream = nullptr) {
    using paged_detail::bits;
    paged_detail::report(
        attn_paged_rope_store_kv(bits(d_q), bits(d_k), bits(d_v), bits(d_q_out), bits(d_k_pages),
                                 bits(d_v_pages), bits(d_cos), bits(d_sin), d_page_table,
                                 d_seq_ids, d_positions, num_tokens, num_seqs, max_pages,
                                 num_pages, page_size, max_seq_len, num_heads, num_kv_heads,
                                 head_dim, q_stride, k_stride, apply_rotation ? 1 : 0, stream),
        "launch_paged_rope_and_store_kv");
}

// attn_paged_decode: one new token per sequence over its pages
inline void launch_paged_attention_decode(
    const __half* d_q, const __half* d_k_pages, const __half* d_v_pages, __half* d_out,
    const int32_t* d_page_table, const int32_t* d_kv_lens, size_t num_seqs, size_t max_pages,
    size_t num_pages, size_t page_size, size_t num_heads, size_t num_kv_heads, size_t head_dim,
    size_t q_stride, void* d_workspace, hipStream_t stream = nullptr) {
    using paged_detail::bits;
    paged_detail::report(
        attn_paged_decode(bits(d_q), bits(d_k_pages), bits(d_v_pages), bits(d_out), d_page_table,
                          d_kv_lens, num_seqs, max_pages, num_pages, page_size, num_heads,
                          num_kv_heads, head_dim, q_stride, d_workspace, stream),
        "launch_paged_attention_decode");
}

// attn_w4_pack: fp16 weights to 4-bit codes and group scales
inline void launch_w4_pack(const __half* d_weights, void* d_packed, __half* d_scales,
                           size_t out_dim, size_t in_dim, size_t group_size,
                           hipStream_t stream = nullptr) {
    using paged_detail::bits;
    paged_detail::report(attn_w4_pack(bits(d_weights), d_packed, bits(d_scales), out_dim, in_dim,
                                      group_size, stream),
                         "launch_w4_pack");
}

// attn_w4_matvec: y = W x (+ residual) on 4-bit weights for one token or a batch
inline void launch_w4_matvec(const __half* d_x, __half* d_y, const void* d_packed,
                             const __half* d_scales, const __half* d_residual, size_t num_tokens,
                             size_t in_dim, size_t out_dim, size_t group_size, size_t x_stride = 0,
                             size_t y_stride = 0, hipStream_t stream = nullptr) {
    using paged_detail::bits;
    paged_detail::report(attn_w4_matvec(bits(d_x), bits(d_y), d_packed, bits(d_scales),
                                        bits(d_residual), num_tokens, in_dim, out_dim, group_size,
                                        x_stride, y_stride, stream),
                         "launch_w4_matvec");
}
