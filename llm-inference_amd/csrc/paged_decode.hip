// Decode attention over a paged KV cache: one new token for each of a batch of
// sequences, out[b][h] = sum_j softmax_j(q[b][h] . k_j / sqrt(D)) v_j over the
// kv_lens[b] cached rows of sequence b, whose pages row b of the page table names.
//
// A sequence of length 0 (a row of a padded batch) leaves its output as it was.  A
// page number out of range makes its sequence's output NaN: nothing is read for it.
#include "paged_internal.hpp"
#include "../../include/attn_mi355x.h"

#include <cmath>

namespace attn {
namespace {

struct PagedDecodeArgs {
    const f16* q;           // rows q_stride apart, Hq heads of D
    const f16* kp;          // K pages [num_pages][page_size][Hkv*D]
    const f16* vp;
    f16* out;               // packed [num_seqs][Hq][D]
    const int32_t* table;   // [num_seqs][max_pages]
    const int32_t* lens;    // [num_seqs]
    uint64_t q_stride;
    uint32_t num_seqs;
    uint32_t max_pages;
    uint32_t num_pages;
    uint32_t page_size;
    uint32_t num_heads;
    uint32_t num_kv_heads;
    uint32_t group;
    uint32_t head_dim;
    float scale_log2;
    uint32_t pad_;
};

// Any head_dim up to 256, page size, alignment and grouping: one workgroup per
// sequence and query head, tiles of 256 keys, one score per thread, then a dim per
// thread; fp32 throughout.
constexpr int kTile = 256;

__global__ __launch_bounds__(kTile) void paged_decode_generic(PagedDecodeArgs a) {
    __shared__ float s_q[256], s_p[kTile], s_red[2][kTile / 64];
    __shared__ uint64_t s_row[kTile];
    const uint32_t b = blockIdx.y, h = blockIdx.x, tid = threadIdx.x;
    const uint32_t D = a.head_dim, wave = tid >> 6;
    const uint32_t len = clamp_len(a.lens[b], a.max_pages, a.page_size);
    if (len == 0) return;
    if (tid < D) s_q[tid] = (float)a.q[b * a.q_stride + (uint64_t)h * D + tid];
    const uint64_t stride = (uint64_t)a.num_kv_heads * D;
    const f16* const kb = a.kp + (uint64_t)(h / a.group) * D;
    const f16* const vb = a.vp + (uint64_t)(h / a.group) * D;
    const int32_t* const row = a.table + (uint64_t)b * a.max_pages;
    float m_run = -1.0e30f, l_run = 0.f, acc = 0.f;
    for (uint32_t j0 = 0; j0 < len; j0 += kTile) {
        __syncthreads();  // the last tile's rows and weights are read, q is written
        const uint32_t j = j0 + tid;
        float s = -INFINITY;
        if (j < len) {
            const uint32_t page = (uint32_t)row[j / a.page_size];
            const bool ok = page < a.num_pages;
            s_row[tid] = ok ? (uint64_t)page * a.page_size + j % a.page_size : 0u;
            float dot = __builtin_nanf("");
            if (ok) {
                const f16* const kr = kb + s_row[tid] * stride;
                dot = 0.f;
                for (uint32_t d = 0; d < D; ++d) dot += s_q[d] * (float)kr[d];
            }
            s = dot * a.scale_log2;
        }
        const float wm = wave_max(s);
        if ((tid & 63u) == 0) s_red[0][wave] = wm;
        __syncthreads();
        const float m_new = fmaxf(fmaxf(fmaxf(s_red[0][0], s_red[0][1]),
                                        fmaxf(s_red[0][2], s_red[0][3])), m_run);
        const float p = j < len ? fast_exp2(s - m_new) : 0.f;
        s_p[tid] = p;
        const float wl = wave_sum(p);
        if ((tid & 63u) == 0) s_red[1][wave] = wl;
        __syncthreads();
        const float alpha = fast_exp2(m_run - m_new);
        l_run = l_run * alpha + ((s_red[1][0] + s_red[1][1]) + (s_red[1][2] + s_red[1][3]));
        m_run = m_new;
        if (tid < D) {
            const uint32_t n = min(len - j0, (uint32_t)kTile);
            float part = 0.f;
            // rows of pages out of range are row 0 with a weight of NaN
            if (a.num_pages)
                for (uint32_t i = 0; i < n; ++i)
                    part = __builtin_fmaf(s_p[i], (float)vb[s_row[i] * stride + tid], part);
            acc = acc * alpha + part;
        }
    }
    if (tid < D) a.out[((uint64_t)b * a.num_heads + h) * D + tid] = (f16)(acc / l_run);
}

}  // namespace
}  // namespace attn

using namespace attn;

extern "C" {

size_t attn_paged_decode_workspace_bytes(size_t num_seqs, size_t num_heads, size_t num_kv_heads,
                                         size_t head_dim) {
    (void)num_seqs; (void)num_heads; (void)num_kv_heads; (void)head_dim;
    return 256;
}

int attn_paged_decode(const attn_f16_t* q, const attn_f16_t* k_pages, const attn_f16_t* v_pages,
                      attn_f16_t* out, const int32_t* page_table, const int32_t* kv_lens,
                      size_t num_seqs, size_t max_pages, size_t num_pages, size_t page_size,
                      size_t num_heads, size_t num_kv_heads, size_t head_dim, size_t q_stride,
                      void* workspace, hipStream_t stream) {
    if (num_seqs == 0 || max_pages == 0 || num_heads == 0) return 0;
    if (!paged_sizes_ok(num_seqs, max_pages, num_pages, page_size) || num_kv_heads == 0 ||
        num_heads % num_kv_heads != 0 || num_heads > 65535 || num_seqs > 65535 || head_dim == 0 ||
        head_dim > 256 || !q || !k_pages || !v_pages || !out || !page_table || !kv_lens ||
        !workspace)
        return (int)hipErrorInvalidValue;
    PagedDecodeArgs a{};
    a.q = reinterpret_cast<const f16*>(q);
    a.kp = reinterpret_cast<const f16*>(k_pages);
    a.vp = reinterpret_cast<const f16*>(v_pages);
    a.out = reinterpret_cast<f16*>(out);
    a.table = page_table;
    a.lens = kv_lens;
    a.q_stride = q_stride ? q_stride : num_heads * head_dim;
    a.num_seqs = (uint32_t)num_seqs;
    a.max_pages = (uint32_t)max_pages;
    a.num_pages = (uint32_t)num_pages;
    a.page_size = (uint32_t)page_size;
    a.num_heads = (uint32_t)num_heads;
    a.num_kv_heads = (uint32_t)num_kv_heads;
    a.group = (uint32_t)(num_heads / num_kv_heads);
    a.head_dim = (uint32_t)head_dim;
    a.scale_log2 = (float)(1.4426950408889634 / std::sqrt((double)head_dim));
    hipLaunchKernelGGL(paged_decode_generic, dim3(a.num_heads, a.num_seqs), dim3(kTile), 0, stream,
                       a);
    return (int)hipGetLastError();
}

}  // extern "C"
