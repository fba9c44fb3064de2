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

// The eight columns of a word as fp16, in order: 1024 + code has the code in its lowest
// bits, and both it and the difference to 1032 are exact.
__device__ __forceinline__ f16x8 w4_values(uint32_t word) {
    f16x8 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t pair = ((word >> (4 * i)) & 0x000f000fu) | 0x64006400u;
        const f16x2 x = __builtin_bit_cast(f16x2, pair) - f16x2{(f16)1032.0f, (f16)1032.0f};
        v[2 * i] = x[0];
        v[2 * i + 1] = x[1];
    }
    return v;
}

// Eight columns of x from k on, zero from `cols` on.  VEC: 16-byte loads (rows 16-byte
// aligned, cols a multiple of 8).
template <bool VEC>
__device__ __forceinline__ f16x8 w4_load_x(const f16* row, uint32_t k, uint32_t cols) {
    f16x8 v = {};
    if constexpr (VEC) {
        if (k < cols) v = ld16(row + k);
    } else {
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e)
            if (k + e < cols) v[e] = row[k + e];
    }
    return v;
}

constexpr uint32_t kW4Waves = 8;

// One workgroup per 16 rows; its waves take the column tiles in turn and meet in LDS.
// TT: tiles of 16 tokens.  SPS: steps of 32 columns that share a scale at least (4: the
// group is a multiple of 128; 2: of 64; 1).  The products of a scale's columns are summed
// by the MFMAs from zero, then scaled and added in fp32, so no product is rounded.
template <int TT, int SPS, bool VEC>
__global__ __launch_bounds__(64 * kW4Waves) void w4_matvec(W4Args a) {
    constexpr int kRound = 4;  // column tiles in flight
    __shared__ float s_part[kW4Waves][16 * TT][17];
    const uint32_t tid = threadIdx.x, lane = tid & 63u;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t n = lane & 15u, gq = lane >> 4;
    const uint32_t rt = blockIdx.x, t0 = blockIdx.y * 16u * TT;
    const uint32_t live = min(a.tokens - t0, 16u * (uint32_t)TT);
    const uint64_t tile_words = (uint64_t)a.col_tiles * 256u;
    const BufRsrc rw = make_rsrc(a.w + rt * tile_words, a.col_tiles * 1024u);
    const f16* xr[TT];
#pragma unroll
    for (int tt = 0; tt < TT; ++tt)  // lanes past the last token repeat it; nothing of theirs is stored
        xr[tt] = a.x + (uint64_t)(t0 + min(16u * tt + n, live - 1u)) * a.x_stride + 8u * gq;
    const f16* const sc = a.scales + rt * 16u + 4u * gq;
    const uint64_t sc_stride = (uint64_t)a.row_tiles * 16u;

    f32x4 acc[TT];
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) acc[tt] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (uint32_t c0 = wave; c0 < a.col_tiles; c0 += kRound * kW4Waves) {
        u32x4 w[kRound];
#pragma unroll
        for (int i = 0; i < kRound; ++i)  // past the last tile: nothing is read
            w[i] = __builtin_bit_cast(
                u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                           rw, (int)((c0 + i * kW4Waves) * 1024u + 16u * lane), 0, 2));
#pragma unroll
        for (int i = 0; i < kRound; ++i) {
            const uint32_t c = c0 + i * kW4Waves;
            if (c >= a.col_tiles) break;
#pragma unroll
            for (int s0 = 0; s0 < 4; s0 += SPS) {
                const uint32_t k = 128u * c + 32u * s0;
                if (SPS < 4 && k >= a.cols) break;
                f32x4 part[TT];
#pragma unroll
                for (int tt = 0; tt < TT; ++tt) part[tt] = f32x4{0.f, 0.f, 0.f, 0.f};
                const f16x4 scale = *reinterpret_cast<const f16x4*>(sc + k / a.group * sc_stride);
#pragma unroll
                for (int s = s0; s < s0 + SPS; ++s) {
                    const f16x8 wv = w4_values(w[i][s]);
#pragma unroll
                    for (int tt = 0; tt < TT; ++tt) {
                        // x's rows start at column 8 gq
                        const f16x8 xv = w4_load_x<VEC>(xr[tt], 128u * c + 32u * s,
                                                        a.cols > 8u * gq ? a.cols - 8u * gq : 0u);
                        part[tt] = mfma16(wv, xv, part[tt]);
                    }
                }
#pragma unroll
                for (int tt = 0; tt < TT; ++tt)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        acc[tt][r] = __builtin_fmaf((float)scale[r], part[tt][r], acc[tt][r]);
            }
        }
    }
#pragma unroll
    for (int tt = 0; tt < TT; ++tt)
#pragma unroll
        for (int r = 0; r < 4; ++r) s_part[wave][16 * tt + n][4u * gq + r] = acc[tt][r];
    __syncthreads();
    for (uint32_t i = tid; i < live * 16u; i += 64u * kW4Waves) {
        const uint32_t t = i >> 4, r = i & 15u, row = rt * 16u + r;
        if (row >= a.rows) continue;
        float sum = 0.f;
#pragma unroll
        for (uint32_t x = 0; x < kW4Waves; ++x) sum += s_part[x][t][r];
        const uint64_t at = (uint64_t)(t0 + t) * a.y_stride + row;
        if (a.residual) sum += (float)a.residual[at];
        a.y[at] = (f16)sum;
    }
}

template <int TT, int SPS>
hipError_t launch_w4(const W4Args& a, bool vec, hipStream_t stream) {
    const dim3 grid(a.row_tiles, (a.tokens + 16u * TT - 1u) / (16u * TT)), block(64 * kW4Waves);
    if (vec)
        hipLaunchKernelGGL((w4_matvec<TT, SPS, true>), grid, block, 0, stream, a);
    else
        hipLaunchKernelGGL((w4_matvec<TT, SPS, false>), grid, block, 0, stream, a);
    return hipGetLastError();
}

template <int TT>
hipError_t launch_w4(const W4Args& a, bool vec, hipStream_t stream) {
    if (a.group % 128 == 0) return launch_w4<TT, 4>(a, vec, stream);
    if (a.group % 64 == 0) return launch_w4<TT, 2>(a, vec, stream);
    return launch_w4<TT, 1>(a, vec, stream);
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
    return rows <= 0x7ffffff0u && cols <= (1u << 28) && group > 0 && group % 32 == 0 &&
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
        (in_dim && (!x || !packed || !scales || ((uintptr_t)packed & 15u) ||
                    ((uintptr_t)scales & 7u))))
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
    const bool vec = aligned16(x) && a.x_stride % 8 == 0 && in_dim % 8 == 0;
    if (a.tokens <= 16) return (int)launch_w4<1>(a, vec, stream);
    if (a.tokens <= 32) return (int)launch_w4<2>(a, vec, stream);
    if (a.tokens <= 48) return (int)launch_w4<3>(a, vec, stream);
    return (int)launch_w4<4>(a, vec, stream);
}

}  // extern "C"
