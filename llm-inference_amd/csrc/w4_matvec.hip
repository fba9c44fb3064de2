// Matrix-vector products with 4-bit weights and group scales, and the packer that
// makes them from fp16 weights.
//
//   y[t][n] = sum_k (c[n][k] - 8) s[n][k / G] x[t][k]  (+ residual[t][n])
//
// Packed form.  Codes lie in tiles of 16 rows and 128 columns, 1 KiB each, tiles of a
// row block in column order: 16 bytes for each of 64 lanes, lane 16 a + r holding row
// r's columns 32 s + 8 a + 0..7 in its word s (s = 0..3): a wave reads a tile in one
// contiguous 16-byte load per lane, and word s of the 64 lanes is the A operand of one
// 16x16x32 MFMA, which takes 8 consecutive columns per lane.  Within a word column 2 i
// is in bits 4 i and column 2 i + 1 in bits 16 + 4 i, so that one mask leaves two
// neighbouring columns in the two halves of a register.  Rows past the matrix and
// columns past it hold code 8 (zero).  Scales are fp16 [ceil(K / G)][N rounded up to 16],
// zero in rows past the matrix.
#include "attn_internal.hpp"
#include "../../include/attn_mi355x.h"

namespace attn {
namespace {

struct W4Args {
    const f16* x;          // rows x_stride apart
    f16* y;                // rows y_stride apart
    const f16* residual;   // rows y_stride apart, or nullptr
    const uint32_t* w;
    const f16* scales;
    uint64_t x_stride;
    uint64_t y_stride;
    uint32_t tokens;
    uint32_t rows;
    uint32_t cols;
    uint32_t group;
    uint32_t row_tiles;    // ceil(rows / 16)
    uint32_t col_tiles;    // ceil(cols / 128)
};

__device__ __forceinline__ int w4_code(uint32_t word, int e) {
    return (int)((word >> (4 * (e >> 1) + 16 * (e & 1))) & 15u);
}

// One wave per row and token.
__global__ __launch_bounds__(256) void w4_matvec_simple(W4Args a) {
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t row = blockIdx.x * 4u + (threadIdx.x >> 6), t = blockIdx.y;
    if (row >= a.rows) return;
    const uint32_t words = a.col_tiles * 16u;  // of a row
    const f16* const x = a.x + t * a.x_stride;
    float sum = 0.f;
    for (uint32_t i = lane; i < words; i += 64u) {
        const uint32_t c = i >> 4, s = (i >> 2) & 3u, q = i & 3u;
        const uint32_t k = 128u * c + 32u * s + 8u * q;
        if (k >= a.cols) continue;
        const uint32_t word =
            a.w[(((uint64_t)(row >> 4) * a.col_tiles + c) * 64u + 16u * q + (row & 15u)) * 4u + s];
        const float scale = (float)a.scales[(uint64_t)(k / a.group) * a.row_tiles * 16u + row];
        float part = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (k + e < a.cols) part += (float)(w4_code(word, e) - 8) * (float)x[k + e];
        sum = __builtin_fmaf(scale, part, sum);
    }
    sum = wave_sum(sum);
    if (lane != 0) return;
    if (a.residual) sum += (float)a.residual[t * a.y_stride + row];
    a.y[t * a.y_stride + row] = (f16)sum;
}

struct W4PackArgs {
    const f16* w;     // [rows][cols]
    uint32_t* out;
    f16* scales;
    uint32_t rows, cols, group, row_tiles, col_tiles;
};

// One wave per scale: the largest magnitude of a row's group over 7, rounded to fp16
// (7 of the 8 steps each way, so that the codes are symmetric).  An infinity gives an
// infinite scale and a NaN a NaN, which the products then hold.
__global__ __launch_bounds__(256) void w4_scales(W4PackArgs a) {
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t row = blockIdx.x * 4u + (threadIdx.x >> 6);
    const uint32_t g = blockIdx.y;
    if (row >= a.row_tiles * 16u) return;
    float most = 0.f;
    bool nan = false;
    if (row < a.rows) {
        const f16* const w = a.w + (uint64_t)row * a.cols;
        const uint32_t end = min((uint64_t)a.cols, (uint64_t)(g + 1u) * a.group);
        for (uint64_t k = (uint64_t)g * a.group + lane; k < end; k += 64u) {
            const float v = (float)w[k];
            nan |= v != v;
            most = fmaxf(most, fabsf(v));
        }
    }
    most = wave_max(most);
    if (__ballot(nan)) most = __builtin_nanf("");
    if (lane == 0) a.scales[(uint64_t)g * a.row_tiles * 16u + row] = (f16)(most / 7.0f);
}

// One thread per word: code = round(w / scale) + 8, ties to even, within 0..15; zero
// scales and values that are no number give 8.
__global__ __launch_bounds__(256) void w4_codes(W4PackArgs a) {
    const uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x;
    if (i >= (uint64_t)a.row_tiles * a.col_tiles * 256u) return;
    const uint32_t s = i & 3u, r = (i >> 2) & 15u, q = (i >> 6) & 3u;
    const uint64_t tile = i >> 8;
    const uint32_t rt = (uint32_t)(tile / a.col_tiles), c = (uint32_t)(tile - (uint64_t)rt * a.col_tiles);
    const uint32_t row = rt * 16u + r, k = 128u * c + 32u * s + 8u * q;
    uint32_t word = 0x88888888u;
    if (row < a.rows && k < a.cols) {
        const float scale = (float)a.scales[(uint64_t)(k / a.group) * a.row_tiles * 16u + row];
        if (scale > 0.f) {
            word = 0;
            for (int e = 0; e < 8; ++e) {
                float v = k + e < a.cols ? (float)a.w[(uint64_t)row * a.cols + k + e] / scale : 0.f;
                if (!(v == v)) v = 0.f;
                const int code = (int)fminf(fmaxf(rintf(v), -8.f), 7.f) + 8;
                word |= (uint32_t)code << (4 * (e >> 1) + 16 * (e & 1));
            }
        }
    }
    a.out[i] = word;
}

bool w4_sizes_ok(size_t rows, size_t cols, size_t group) {
    return rows <= 0x7ffffff0u && cols <= 0x7fffff80u && group > 0 && group % 32 == 0 &&
           group <= 0x7fffffffu;
}

}  // namespace
}  // namespace attn

using namespace attn;

extern "C" {

size_t attn_w4_weight_bytes(size_t out_dim, size_t in_dim) {
    return (out_dim + 15) / 16 * ((in_dim + 127) / 128) * 1024;
}

size_t attn_w4_scale_count(size_t out_dim, size_t in_dim, size_t group_size) {
    return group_size ? (out_dim + 15) / 16 * 16 * ((in_dim + group_size - 1) / group_size) : 0;
}

int attn_w4_pack(const attn_f16_t* w, void* packed, attn_f16_t* scales, size_t out_dim,
                 size_t in_dim, size_t group_size, hipStream_t stream) {
    if (out_dim == 0 || in_dim == 0) return 0;
    if (!w4_sizes_ok(out_dim, in_dim, group_size) || !w || !packed || !scales ||
        ((uintptr_t)packed & 15u))
        return (int)hipErrorInvalidValue;
    W4PackArgs a{};
    a.w = reinterpret_cast<const f16*>(w);
    a.out = static_cast<uint32_t*>(packed);
    a.scales = reinterpret_cast<f16*>(scales);
    a.rows = (uint32_t)out_dim;
    a.cols = (uint32_t)in_dim;
    a.group = (uint32_t)group_size;
    a.row_tiles = (uint32_t)((out_dim + 15) / 16);
    a.col_tiles = (uint32_t)((in_dim + 127) / 128);
    const uint64_t groups = (in_dim + group_size - 1) / group_size;
    const uint64_t blocks = (uint64_t)a.row_tiles * a.col_tiles;
    if (groups > 65535 || blocks > 0x7fffffffull) return (int)hipErrorInvalidValue;
    hipLaunchKernelGGL(w4_scales, dim3(a.row_tiles * 4u, (uint32_t)groups), dim3(256), 0, stream, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
    hipLaunchKernelGGL(w4_codes, dim3((uint32_t)blocks), dim3(256), 0, stream, a);
    return (int)hipGetLastError();
}

int attn_w4_matvec(const attn_f16_t* x, attn_f16_t* y, const void* packed,
                   const attn_f16_t* scales, const attn_f16_t* residual, size_t num_tokens,
                   size_t in_dim, size_t out_dim, size_t group_size, size_t x_stride,
                   size_t y_stride, hipStream_t stream) {
    if (num_tokens == 0 || out_dim == 0) return 0;
    if (!w4_sizes_ok(out_dim, in_dim, group_size) || num_tokens > 65535 || !y ||
        (in_dim && (!x || !packed || !scales || ((uintptr_t)packed & 15u))))
        return (int)hipErrorInvalidValue;
    W4Args a{};
    a.x = reinterpret_cast<const f16*>(x);
    a.y = reinterpret_cast<f16*>(y);
    a.residual = reinterpret_cast<const f16*>(residual);
    a.w = static_cast<const uint32_t*>(packed);
    a.scales = reinterpret_cast<const f16*>(scales);
    a.x_stride = x_stride ? x_stride : in_dim;
    a.y_stride = y_stride ? y_stride : out_dim;
    a.tokens = (uint32_t)num_tokens;
    a.rows = (uint32_t)out_dim;
    a.cols = (uint32_t)in_dim;
    a.group = (uint32_t)group_size;
    a.row_tiles = (uint32_t)((out_dim + 15) / 16);
    a.col_tiles = (uint32_t)((in_dim + 127) / 128);
    hipLaunchKernelGGL(w4_matvec_simple, dim3((a.rows + 3u) / 4u, a.tokens), dim3(256), 0, stream,
                       a);
    return (int)hipGetLastError();
}

}  // extern "C"
