// Paged KV cache of a batch of sequences: the pool of all layers, the page table, lengths
// and reference counts, all in device memory.  The pool has KVCache's layout (kv_cache.hpp)
// with max_seq_len = num_pages * page_size rows per layer.  Calls on one cache must be
// ordered (one stream); sequences are the rows 0 .. max_seqs - 1, and arguments with an
// entry per sequence are device arrays of max_seqs int32.
#pragma once
#include <cstddef>
#include <cstdint>

#include "gpu_utils.hpp"
#include "kernels/paged_kernels.hpp"

class PagedKVCache {
    size_t num_layers_, num_pages_, page_size_, num_kv_heads_, head_dim_, max_seqs_, max_pages_;
    __half* pool_ = nullptr;
    int32_t* state_ = nullptr;  // table, lengths, counts, status (2), pages in use (1)
    void* pages_ws_ = nullptr;
    void* decode_ws_ = nullptr;
    size_t decode_heads_;

    size_t page_elems() const { return page_size_ * num_kv_heads_ * head_dim_; }
    size_t plane_elems() const { return num_pages_ * page_elems(); }
    size_t table_entries() const { return max_seqs_ * max_pages_; }

  public:
    // Config: num_layers, num_heads, num_kv_heads and head_dim, as KVCache takes it
    template <typename Config>
    PagedKVCache(const Config& config, size_t num_pages, size_t page_size, size_t max_seqs,
                 size_t max_pages)
        : num_layers_(config.num_layers),
          num_pages_(num_pages),
          page_size_(page_size),
          num_kv_heads_(config.num_kv_heads),
          head_dim_(config.head_dim),
          max_seqs_(max_seqs),
          max_pages_(max_pages),
          decode_heads_(config.num_heads) {
        const size_t words = table_entries() + max_seqs_ + num_pages_ + 3;
        HIP_CHECK(hipMalloc(&pool_, 2 * num_layers_ * plane_elems() * sizeof(__half)));
        HIP_CHECK(hipMalloc(&state_, words * sizeof(int32_t)));
        HIP_CHECK(hipMalloc(&pages_ws_, attn_pages_workspace_bytes(max_seqs_, num_pages_)));
        HIP_CHECK(hipMalloc(&decode_ws_,
                            attn_paged_decode_workspace_bytes(max_seqs_, decode_heads_,
                                                              num_kv_heads_, head_dim_)));
        HIP_CHECK(hipMemset(state_, 0, words * sizeof(int32_t)));
        HIP_CHECK(hipStreamSynchronize(nullptr));  // zero for calls on any stream
    }
    ~PagedKVCache() {
        (void)hipFree(pool_);
        (void)hipFree(state_);
        (void)hipFree(pages_ws_);
        (void)hipFree(decode_ws_);
    }
    PagedKVCache(const PagedKVCache&) = delete;
    PagedKVCache& operator=(const PagedKVCache&) = delete;

    __half* get_layer_k_ptr(size_t layer) const { return pool_ + 2 * layer * plane_elems(); }
    __half* get_layer_v_ptr(size_t layer) const { return pool_ + (2 * layer + 1) * plane_elems(); }
    int32_t* page_table() const { return state_; }
    int32_t* seq_lens() const { return state_ + table_entries(); }
    int32_t* ref_counts() const { return seq_lens() + max_seqs_; }
    // what the last grow found missing: pages of the pool, rows that are too short
    int32_t* status() const { return ref_counts() + num_pages_; }
    int32_t* num_used() const { return status() + 2; }

    void grow(const int32_t* d_tokens, hipStream_t stream = nullptr) {
        paged_detail::report(
            attn_pages_grow(paged_detail::bits(pool_), 2 * num_layers_, 0, page_elems(),
                            page_table(), seq_lens(), d_tokens, ref_counts(), status(), max_seqs_,
                            max_pages_, num_pages_, page_size_, pages_ws_, stream),
            "PagedKVCache::grow");
    }
    // null: every sequence to nothing
    void free(const int32_t* d_keep_lens = nullptr, hipStream_t stream = nullptr) {
        paged_detail::report(attn_pages_free(page_table(), seq_lens(), d_keep_lens, ref_counts(),
                                             max_seqs_, max_pages_, num_pages_, page_size_, stream),
                             "PagedKVCache::free");
    }
    void fork(const int32_t* d_parents, hipStream_t stream = nullptr) {
        paged_detail::report(
            attn_pages_fork(page_table(), seq_lens(), page_table(), seq_lens(), d_parents,
                            ref_counts(), max_seqs_, max_seqs_, max_pages_, num_pages_, page_size_,
                            stream),
            "PagedKVCache::fork");
    }
    void compact(hipStream_t stream = nullptr) {
        paged_detail::report(
            attn_pages_compact(paged_detail::bits(pool_), 2 * num_layers_, 0, page_elems(),
                               page_table(), seq_lens(), ref_counts(), page_table(), ref_counts(),
                               num_used(), max_seqs_, max_pages_, num_pages_, page_size_,
                               pages_ws_, stream),
            "PagedKVCache::compact");
    }
    void append(size_t layer, __half* d_q, const __half* d_k, const __half* d_v, __half* d_q_out,
                const __half* d_cos, const __half* d_sin, const int32_t* d_seq_ids,
                const int32_t* d_positions, size_t num_tokens, size_t max_seq_len, size_t q_stride,
                size_t k_stride, bool apply_rotation, hipStream_t stream = nullptr) {
        launch_paged_rope_and_store_kv(d_q, d_k, d_v, d_q_out, get_layer_k_ptr(layer),
                                       get_layer_v_ptr(layer), d_cos, d_sin, page_table(),
                                       d_seq_ids, d_positions, num_tokens, max_seqs_, max_pages_,
                                       num_pages_, page_size_, max_seq_len, decode_heads_,
                                       num_kv_heads_, head_dim_, q_stride, k_stride,
                                       apply_rotation, stream);
    }
    void decode(size_t layer, const __half* d_q, __half* d_out, size_t q_stride = 0,
                hipStream_t stream = nullptr) {
        launch_paged_attention_decode(d_q, get_layer_k_ptr(layer), get_layer_v_ptr(layer), d_out,
                                      page_table(), seq_lens(), max_seqs_, max_pages_, num_pages_,
                                      page_size_, decode_heads_, num_kv_heads_, head_dim_,
                                      q_stride, decode_ws_, stream);
    }
};
