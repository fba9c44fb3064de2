// RoPE + KV append into pages: the paged form of rope_store_kv.hip for any set of
// new tokens (one per sequence of a decode batch, or chunks of prompts).
//
// Token t belongs to sequence seq_ids[t] (t itself without the list) at position
// positions[t] = p: K heads rotated by table row p and V heads copied to row p %
// page_size of page table[seq][p / page_size]; Q heads rotated in place, or to
// q_out packed [tokens][Hq][D] (copied there when apply == 0).  The rotation is
// rope_pair's: fp32 products each rounded, one rounding to fp16, so every value
// equals what rope_store_kv writes for that position, bit for bit.
//
// A token that names no cache row (a negative position, one past the rotation
// tables or the page table's row, a sequence or page number out of range) is left
// alone: its q, q_out row and all pages keep their values.  Batches padded to a
// fixed size mark their unused tokens so.
//
// Bound by HBM, and for small batches by the chain position -> page -> row.  One lane
// owns 8 rotation pairs of a head (two 16-byte loads and stores), as in
// rope_store_kv_vec; every lane looks its token's page up by itself (the loads of a
// token's lanes hit one cache line), which needs no barrier.  Measured (16/4 heads of
// 128, traced): 2000 tokens 6.4 us for 25.1 MB (3.9 TB/s, one round of loads), 64 tokens
// 2.9 us.
#include "paged_internal.hpp"
#include "../../include/attn_mi355x.h"

namespace attn {
namespace {

struct PagedRopeArgs {
    f16* q;                 // rows q_stride apart
    f16* q_out;             // packed [tokens][Hq][D], or nullptr: q in place
    const f16* k;           // rows k_stride apart
    const f16* v;           // rows k_stride apart
    f16* kp;                // K pages [num_pages][page_size][Hkv*D]
    f16* vp;
    const f16* cos_t;       // [max_seq_len][D/2]
    const f16* sin_t;
    const int32_t* table;   // [num_seqs][max_pages]
    const int32_t* seq_ids; // [tokens] or nullptr
    const int32_t* pos;     // [tokens]
    uint64_t q_stride;
    uint64_t k_stride;
    uint32_t tokens;
    uint32_t num_seqs;
    uint32_t max_pages;
    uint32_t num_pages;
    uint32_t page_size;
    uint32_t max_seq_len;
    uint32_t num_heads;
    uint32_t num_kv_heads;
    uint32_t head_dim;
    uint32_t apply;
};

// the pool row of token t and its position; false: the token names none
__device__ __forceinline__ bool paged_row(const PagedRopeArgs& a, uint32_t t, uint32_t& p,
                                          uint64_t& row) {
    const uint32_t seq = a.seq_ids ? (uint32_t)a.seq_ids[t] : t;
    p = (uint32_t)a.pos[t];  // negative: past every limit
    if (seq >= a.num_seqs || p >= a.max_seq_len) return false;
    const uint32_t j = p / a.page_size;
    if (j >= a.max_pages) return false;
    const uint32_t page = (uint32_t)a.table[(uint64_t)seq * a.max_pages + j];
    if (page >= a.num_pages) return false;
    row = (uint64_t)page * a.page_size + (p - j * a.page_size);
    return true;
}

// W values of each half of a head per thread: 8 (16-byte loads) or 1
template <int W>
__global__ __launch_bounds__(256) void paged_rope_store_kv(PagedRopeArgs a) {
    const uint32_t D = a.head_dim, half = D >> 1;
    const uint32_t lanes = half / W;
    const uint32_t slots = a.num_heads + 2u * a.num_kv_heads;
    const uint64_t gid = (uint64_t)blockIdx.x * 256u + threadIdx.x;
    const uint64_t per_token = (uint64_t)slots * lanes;
    const uint64_t t = gid / per_token;
    if (t >= a.tokens) return;
    const uint32_t rem = (uint32_t)(gid - t * per_token);
    const uint32_t slot = rem / lanes;
    const uint32_t off = (rem - slot * lanes) * W;
    uint32_t p;
    uint64_t row;
    if (!paged_row(a, (uint32_t)t, p, row)) return;
    const bool is_q = slot < a.num_heads;
    const bool is_v = slot >= a.num_heads + a.num_kv_heads;
    const bool turn = a.apply && !is_v;
    const f16* src;
    f16* dst;
    if (is_q) {
        f16* const x = a.q + t * a.q_stride + (uint64_t)slot * D;
        if (!a.apply && !a.q_out) return;
        src = x;
        dst = a.q_out ? a.q_out + (t * a.num_heads + slot) * D : x;
    } else {
        const uint32_t h = slot - a.num_heads - (is_v ? a.num_kv_heads : 0u);
        src = (is_v ? a.v : a.k) + t * a.k_stride + (uint64_t)h * D;
        dst = (is_v ? a.vp : a.kp) + (row * a.num_kv_heads + h) * D;
    }
    const uint64_t turn_at = (uint64_t)p * half + off;
    if constexpr (W == 8) {
        f16x8 x0 = ld16(src + off), x1 = ld16(src + half + off);
        if (turn) rope_rotate8(x0, x1, ld16(a.cos_t + turn_at), ld16(a.sin_t + turn_at), x0, x1);
        st16(dst + off, x0);
        st16(dst + half + off, x1);
    } else {
        f16 x0 = src[off], x1 = src[half + off];
        if (turn) rope_pair(x0, x1, a.cos_t[turn_at], a.sin_t[turn_at], x0, x1);
        dst[off] = x0;
        dst[half + off] = x1;
    }
}

}  // namespace
}  // namespace attn

using namespace attn;

extern "C" int attn_paged_rope_store_kv(
    attn_f16_t* q, const attn_f16_t* k, const attn_f16_t* v, attn_f16_t* q_out,
    attn_f16_t* k_pages, attn_f16_t* v_pages, const attn_f16_t* cos_table,
    const attn_f16_t* sin_table, const int32_t* page_table, const int32_t* seq_ids,
    const int32_t* positions, size_t num_tokens, size_t num_seqs, size_t max_pages,
    size_t num_pages, size_t page_size, size_t max_seq_len, size_t num_heads, size_t num_kv_heads,
    size_t head_dim, size_t q_stride, size_t k_stride, int apply_rotation, hipStream_t stream) {
    if (num_tokens == 0) return 0;
    if (!paged_sizes_ok(num_seqs, max_pages, num_pages, page_size) || !paged_u31(num_tokens) ||
        !paged_u31(max_seq_len) || num_heads > 65535 || num_kv_heads > 65535 || head_dim > 65535 ||
        head_dim == 0 || (head_dim & 1u))
        return (int)hipErrorInvalidValue;
    if (num_heads + num_kv_heads == 0) return 0;
    if (num_heads && !q) return (int)hipErrorInvalidValue;
    if (num_kv_heads && (!k || !v || !k_pages || !v_pages)) return (int)hipErrorInvalidValue;
    if (!page_table || !positions || (apply_rotation && (!cos_table || !sin_table)))
        return (int)hipErrorInvalidValue;
    if (!seq_ids && num_tokens > num_seqs) return (int)hipErrorInvalidValue;
    PagedRopeArgs a{};
    a.q = reinterpret_cast<f16*>(q);
    a.q_out = reinterpret_cast<f16*>(q_out);
    a.k = reinterpret_cast<const f16*>(k);
    a.v = reinterpret_cast<const f16*>(v);
    a.kp = reinterpret_cast<f16*>(k_pages);
    a.vp = reinterpret_cast<f16*>(v_pages);
    a.cos_t = reinterpret_cast<const f16*>(cos_table);
    a.sin_t = reinterpret_cast<const f16*>(sin_table);
    a.table = page_table;
    a.seq_ids = seq_ids;
    a.pos = positions;
    a.q_stride = q_stride ? q_stride : num_heads * head_dim;
    a.k_stride = k_stride ? k_stride : num_kv_heads * head_dim;
    a.tokens = (uint32_t)num_tokens;
    a.num_seqs = (uint32_t)num_seqs;
    a.max_pages = (uint32_t)max_pages;
    a.num_pages = (uint32_t)num_pages;
    a.page_size = (uint32_t)page_size;
    a.max_seq_len = (uint32_t)max_seq_len;
    a.num_heads = (uint32_t)num_heads;
    a.num_kv_heads = (uint32_t)num_kv_heads;
    a.head_dim = (uint32_t)head_dim;
    a.apply = apply_rotation ? 1u : 0u;
    const bool vec = head_dim % 16 == 0 && a.q_stride % 8 == 0 && a.k_stride % 8 == 0 &&
                     aligned16(q) && aligned16(q_out) && aligned16(k) && aligned16(v) &&
                     aligned16(k_pages) && aligned16(v_pages) &&
                     (!apply_rotation || (aligned16(cos_table) && aligned16(sin_table)));
    const uint64_t lanes = head_dim / 2 / (vec ? 8 : 1);
    const uint64_t slots = num_heads + 2 * num_kv_heads;
    const uint64_t blocks = (num_tokens * slots * lanes + 255) / 256;
    if (slots * lanes > 0x7fffffffull || blocks > 0x7fffffffull) return (int)hipErrorInvalidValue;
    if (vec)
        hipLaunchKernelGGL(paged_rope_store_kv<8>, dim3((uint32_t)blocks), dim3(256), 0, stream, a);
    else
        hipLaunchKernelGGL(paged_rope_store_kv<1>, dim3((uint32_t)blocks), dim3(256), 0, stream, a);
    return (int)hipGetLastError();
}
