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
//
// Bound by the weights' bytes for a few tokens and many rows (one token, 128256 x 2048: 135.7
// MB in 25.8 us, 5.3 TB/s), by latency for few rows (2048 x 2048: 3.2 us).  For a batch
// the load pipe and the unpacking bound it (33 tokens, 2048 x 11008, groups of 32: 12.0 us,
// of which the weights' 11.3 MB would take 2.7): each workgroup reads its tokens' whole rows
// of x, about 9 ns a KiB and CU wherever they lie, and the vector instructions take half
// the time.  Many rows share those reads between the waves of a workgroup; for few rows,
// sharing the columns between workgroups would divide them, but takes a workspace and a
// second kernel for the sums.
#include "attn_internal.hpp"
#include "../../include/attn_mi355x.h"

#include <algorithm>

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
    uint32_t group_mul;    // see w4_group
    uint32_t row_tiles;    // ceil(rows / 16)
    uint32_t col_tiles;    // ceil(cols / 128)
    uint32_t split;        // waves that share a row tile: 1, 2, 4 or 8
};

// The eight columns of a word as fp16, in order: code - 8.  With 0x6400 above it a code in
// the low four bits of a half reads 1024 + code, one in the next four bits 1024 + 16 code:
// less 1032, or over 16 and less 72, both exact in fp16.  The constants live in registers
// (hidden from the compiler), so that mask and or are one v_and_or_b32, which takes no
// literals: 9 instructions a word, 13 otherwise (33 tokens, 2048 x 11008,
// groups of 32: 13.0 us against 13.9 with eight waves).
struct W4Consts {
    uint32_t low, high, one;
    __device__ W4Consts() : low(0x000f000fu), high(0x00f000f0u), one(0x64006400u) {
        asm("" : "+s"(low), "+s"(high), "+v"(one));
    }
};
__device__ __forceinline__ f16x8 w4_values(uint32_t word, const W4Consts& k) {
    const uint32_t up = word >> 8;
    const f16x2 c0 = __builtin_bit_cast(f16x2, (word & k.low) | k.one);
    const f16x2 c1 = __builtin_bit_cast(f16x2, (word & k.high) | k.one);
    const f16x2 c2 = __builtin_bit_cast(f16x2, (up & k.low) | k.one);
    const f16x2 c3 = __builtin_bit_cast(f16x2, (up & k.high) | k.one);
    const f16x2 low = {(f16)-1032.0f, (f16)-1032.0f}, high = {(f16)-72.0f, (f16)-72.0f};
    const f16x2 part = {(f16)0.0625f, (f16)0.0625f};
    const f16x2 v0 = c0 + low, v2 = c2 + low;
    const f16x2 v1 = __builtin_elementwise_fma(c1, part, high);
    const f16x2 v3 = __builtin_elementwise_fma(c3, part, high);
    return f16x8{v0[0], v0[1], v1[0], v1[1], v2[0], v2[1], v3[0], v3[1]};
}

// 16 bytes of codes per lane.  Without the non-temporal hint: 16 tokens, 12000 x 12000 23.4
// us against 28.0 with it, one token, 128256 x 2048 (HBM-cold) level.
__device__ __forceinline__ u32x4 w4_load(BufRsrc rows, uint32_t byte_off) {
    return __builtin_bit_cast(u32x4,
                              __builtin_amdgcn_raw_buffer_load_b128(rows, (int)byte_off, 0, 0));
}

constexpr uint32_t kW4Waves = 8;
constexpr uint32_t kDead = 0xfffff000u;  // a buffer offset past every range: nothing is read

// Lane's eight columns of x from column k on, in column tile c, that start at element `at`
// of xb; zeros past the last.  VEC: rows 16-byte aligned and a multiple of 8 columns, through
// a range that reads nothing past it.  Otherwise rows at any element: the same 16 bytes as
// one unaligned load, element by element in the tile that holds the row's end (64 tokens,
// 2048 x 11009: 15.0 us; 44.1 with elements everywhere, one tile in flight, x not shared).
template <bool VEC>
__device__ __forceinline__ f16x8 w4_load_x(BufRsrc rx, const f16* xb, uint64_t at, uint32_t c,
                                           uint32_t k, uint32_t cols) {
    if constexpr (VEC) return buf_ld16(rx, k < cols ? 2u * (uint32_t)at : kDead);
    typedef f16x8 __attribute__((aligned(2))) f16x8_any;
    if (128u * c + 128u <= cols) return *reinterpret_cast<const f16x8_any*>(xb + at);
    f16x8 v = {};
    if (128u * c < cols) {
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) v[e] = k + e < cols ? xb[at + e] : (f16)0.f;
    }
    return v;
}

// index of the scale of column k: k / group.  group_mul is 2^31 over the group in steps of
// 32 columns, rounded up (0: one group): exact while steps times steps of a group stay
// below 2^31, as they do up to 2^20 columns.
__device__ __forceinline__ uint32_t w4_group(const W4Args& a, uint32_t k) {
    return __umulhi(k >> 5 << 1, a.group_mul);
}

// Sums of the waves that share a row tile: a.split (a power of two) of the workgroup's W,
// neighbours.  s_part is [wave][tokens][rows + 1].
template <int TOKENS, int R, int W>
__device__ __forceinline__ void w4_store(const W4Args& a, const float (*s_part)[TOKENS][16 * R + 1],
                                         uint32_t t0, uint32_t live) {
    const uint32_t tiles = W / a.split, first = blockIdx.x * tiles;
    const uint32_t per_tile = live * 16u * R;
    for (uint32_t i = threadIdx.x; i < tiles * per_tile; i += 64u * W) {
        const uint32_t tile = i / per_tile, j = i - tile * per_tile;
        const uint32_t t = j / (16u * R), r = j % (16u * R), row = (first + tile) * 16u * R + r;
        if (row >= a.rows) continue;
        float sum = 0.f;
        for (uint32_t x = 0; x < a.split; ++x) sum += s_part[tile * a.split + x][t][r];
        const uint64_t at = (uint64_t)(t0 + t) * a.y_stride + row;
        if (a.residual) sum += (float)a.residual[at];
        a.y[at] = (f16)sum;
    }
}

// A wave's column tiles first, first + step, .. below end, with D of them in flight.  Nothing
// past the end is loaded: a load that reads nothing holds the load pipe as long as any (one
// token, 2048 x 2048: 3.2 us against 3.8; 16 tokens, 4096 x 4096: 5.3 against 5.5).
template <int D, class Stage, class Load, class Compute>
__device__ __forceinline__ void w4_columns(uint32_t first, uint32_t step, uint32_t end,
                                           Stage (&st)[D], const Load& load,
                                           const Compute& compute) {
    uint32_t c = first;
#pragma unroll
    for (int i = 0; i < D; ++i)
        if (c + i * step < end) load(c + i * step, st[i]);
    for (; c + (2 * D - 1) * step < end; c += D * step) {
#pragma unroll
        for (int i = 0; i < D; ++i) {
            __builtin_amdgcn_sched_barrier(0);
            compute(st[i]);
            load(c + (i + D) * step, st[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < 2 * D - 1; ++i) {
        __builtin_amdgcn_sched_barrier(0);
        if (c + i * step >= end) break;
        compute(st[i % D]);
        if (i < D - 1 && c + (i + D) * step < end) load(c + (i + D) * step, st[i % D]);
    }
}

// Up to four tokens.  Column n of the MFMAs' result stands for token n % 4 and step n / 4
// of a column tile: lane (gq, n) loads x for that step only (one load per column tile
// instead of four), the operand of step s is zero in the other steps' columns, and each
// lane scales its column's sum by its own step's scales, whatever the group size.
template <bool VEC>
__global__ __launch_bounds__(64 * kW4Waves) void w4_matvec_narrow(W4Args a) {
    constexpr int kDepth = 4;  // column tiles in flight
    __shared__ float s_part[kW4Waves][4][17];
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t n = lane & 15u, gq = lane >> 4, step = n >> 2;
    const W4Consts consts;
    const uint32_t rt = (blockIdx.x * kW4Waves + wave) / a.split;
    const uint32_t first = wave & (a.split - 1u);
    const uint32_t token = min(n & 3u, a.tokens - 1u);
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    if (rt < a.row_tiles && a.col_tiles > 0) {
        const BufRsrc rw =
            make_rsrc(a.w + (uint64_t)rt * a.col_tiles * 256u, a.col_tiles * 1024u);
        const BufRsrc rx = make_rsrc(a.x, (uint32_t)(((a.tokens - 1u) * a.x_stride + a.cols) * 2u));
        const uint64_t x_at = token * a.x_stride;
        const f16* const sc = a.scales + rt * 16u + 4u * gq;
        const uint64_t sc_stride = (uint64_t)a.row_tiles * 16u;
        struct Stage {
            u32x4 w;
            f16x8 x;
            f16x4 scale;
        } st[kDepth];
        auto load = [&](uint32_t c, Stage& z) {
            z.w = w4_load(rw, c * 1024u + 16u * lane);
            const uint32_t k = 128u * c + 32u * step + 8u * gq;
            z.x = w4_load_x<VEC>(rx, a.x, x_at + k, c, k, a.cols);
            z.scale = *reinterpret_cast<const f16x4*>(
                sc + w4_group(a, min(128u * c + 32u * step, a.cols - 1u)) * sc_stride);
        };
        auto compute = [&](const Stage& z) {
            f32x4 part = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (uint32_t s = 0; s < 4; ++s)
                part = mfma16(w4_values(z.w[s], consts), step == s ? z.x : f16x8{}, part);
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[r] = __builtin_fmaf((float)z.scale[r], part[r], acc[r]);
        };
        w4_columns<kDepth>(first, a.split, a.col_tiles, st, load, compute);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {  // the four steps of a token
        float v = acc[r];
        v += dpp_f<kDppRor4>(v);
        v += dpp_f<kDppRor8>(v);
        if (step == 0) s_part[wave][n][4u * gq + r] = v;
    }
    __syncthreads();
    w4_store<4, 1, kW4Waves>(a, s_part, 0, a.tokens);
}

// the scales that lane L of a row of 16 lanes loaded, in all of them
template <int L>
__device__ __forceinline__ f16x4 w4_lane_scale(u32x2 mine) {
    u32x2 v;
#pragma unroll
    for (int i = 0; i < 2; ++i)  // row_newbcast L
        v[i] = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)mine[i], 0x150 + L, 0xF, 0xF, true);
    return __builtin_bit_cast(f16x4, v);
}

// Few rows: R row tiles x 16 tokens a wave, the waves of a row tile split the columns, each
// with its own x, 4 X tokens of it (8 tokens, 2048 x 11008, groups of 128: 7.5 us with two
// loads of x a tile, 8.7 with four).  SPS: steps of 32 columns that share a scale at least
// (4: the group is a multiple of 128; 2: of 64; 1).  The products of a scale's columns are summed by the MFMAs
// from zero, then scaled and added in fp32, so no product is rounded.
template <int R, int SPS, int X, int W, bool VEC>
__global__ __launch_bounds__(64 * W) void w4_matvec(W4Args a) {
    constexpr int kDepth = 2;  // column tiles in flight
    // a wave's x tile (16 tokens x 128 columns), then the waves' sums
    union Shared {
        f16x8 x[W][256];
        float part[W][16][16 * R + 1];
    };
    __shared__ __attribute__((aligned(16))) Shared s_mem;
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t n = lane & 15u, gq = lane >> 4;
    const uint32_t rt = (blockIdx.x * W + wave) / a.split * R;
    const uint32_t first = wave & (a.split - 1u);
    const uint32_t t0 = blockIdx.y * 16u;
    const uint32_t live = min(a.tokens - t0, 16u);
    const W4Consts consts;
    f32x4 acc[R];
#pragma unroll
    for (int q = 0; q < R; ++q) acc[q] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (rt < a.row_tiles && a.col_tiles > 0) {
        BufRsrc rw[R];
#pragma unroll
        for (int q = 0; q < R; ++q)  // row tiles past the last one repeat it and are not stored
            rw[q] = make_rsrc(a.w + (uint64_t)min(rt + q, a.row_tiles - 1u) * a.col_tiles * 256u,
                              a.col_tiles * 1024u);
        // Lane n takes the scales of step n / 4 and row tile n % R: one load, whose lanes on
        // the same line are neighbours (33 tokens, 2048 x 11008, groups of 32: 13.1 us
        // against 14.3 with step n % 4 and a load per row tile).
        const f16* const sc = a.scales + min(rt + n % R, a.row_tiles - 1u) * 16u + 4u * gq;
        const uint64_t sc_stride = (uint64_t)a.row_tiles * 16u;
        const f16* const xb = a.x + (uint64_t)t0 * a.x_stride;
        const BufRsrc rx = make_rsrc(xb, (uint32_t)(((live - 1u) * a.x_stride + a.cols) * 2u));
        // x is read in whole lines, four rows of 256 bytes an instruction (16 rows of 64
        // bytes, as the MFMA operand wants it, took the load pipe twice as long), and turned
        // in LDS: row r's 16-byte chunk i lies at chunk i ^ r, so that the 16 rows of an
        // operand read cover all banks.
        uint64_t x_at[X];  // elements; tokens past the last repeat it: nothing of theirs is stored
#pragma unroll
        for (uint32_t j = 0; j < X; ++j)
            x_at[j] = min(4u * j + gq, live - 1u) * a.x_stride + 8u * n;
        struct Stage {
            u32x4 w[R];
            f16x8 x[X];
            u32x2 scale;  // rows 4 gq ..
        } st[kDepth];
        auto load = [&](uint32_t c, Stage& z) {
#pragma unroll
            for (int q = 0; q < R; ++q) z.w[q] = w4_load(rw[q], c * 1024u + 16u * lane);
            z.scale = *reinterpret_cast<const u32x2*>(
                sc + w4_group(a, min(128u * c + 32u * (n >> 2), a.cols - 1u)) * sc_stride);
            const uint32_t k = 128u * c + 8u * n;
#pragma unroll
            for (uint32_t j = 0; j < X; ++j)
                z.x[j] = w4_load_x<VEC>(rx, xb, x_at[j] + 128u * c, c, k, a.cols);
        };
        auto compute = [&](const Stage& z) {
#pragma unroll
            for (uint32_t j = 0; j < X; ++j) {
                const uint32_t r = 4u * j + gq;
                s_mem.x[wave][16u * r + (n ^ r)] = z.x[j];
            }
            f32x4 part[R];
            auto step = [&]<int s>() {
                const f16x8 xv = s_mem.x[wave][16u * n + ((4u * s + gq) ^ n)];
#pragma unroll
                for (int q = 0; q < R; ++q) {
                    const f16x8 wv = w4_values(z.w[q][s], consts);
                    const f16x4 scale =
                    q == 0 ? w4_lane_scale<4 * s>(z.scale) : w4_lane_scale<4 * s + 1>(z.scale);
                    if (s % SPS == 0) part[q] = f32x4{0.f, 0.f, 0.f, 0.f};
                    part[q] = mfma16(wv, xv, part[q]);
                    if (s % SPS == SPS - 1)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            acc[q][r] = __builtin_fmaf((float)scale[r], part[q][r], acc[q][r]);
                }
            };
            step.template operator()<0>();
            step.template operator()<1>();
            step.template operator()<2>();
            step.template operator()<3>();
        };
        w4_columns<kDepth>(first, a.split, a.col_tiles, st, load, compute);
    }
    __syncthreads();  // every wave has read its x tiles
#pragma unroll
    for (int q = 0; q < R; ++q)
#pragma unroll
        for (int r = 0; r < 4; ++r) s_mem.part[wave][n][16 * q + 4u * gq + r] = acc[q][r];
    __syncthreads();
    w4_store<16, R, W>(a, s_mem.part, t0, live);
}

template <int R, int SPS, int X>
hipError_t launch_w4(W4Args a, bool vec, uint64_t cus, hipStream_t stream) {
    const uint32_t tiles = kW4Waves / a.split * R;
    const dim3 grid((a.row_tiles + tiles - 1u) / tiles, (a.tokens + 15u) / 16u);
    // Sixteen waves where a workgroup has its CU to itself and each wave four column tiles (33
    // tokens, 2048 x 11008, groups of 32: 12.1 us against 13.2; level at 4096 columns).  Rows of
    // x at any element would spill.
    if (vec && a.col_tiles >= 64 && (uint64_t)grid.x * grid.y <= cus) {
        a.split = 16;
        hipLaunchKernelGGL((w4_matvec<R, SPS, X, 16, true>),
                           dim3((a.row_tiles + R - 1u) / R, grid.y), dim3(64 * 16), 0, stream, a);
    } else if (vec) {
        hipLaunchKernelGGL((w4_matvec<R, SPS, X, kW4Waves, true>), grid, dim3(64 * kW4Waves), 0,
                           stream, a);
    } else {
        hipLaunchKernelGGL((w4_matvec<R, SPS, X, kW4Waves, false>), grid, dim3(64 * kW4Waves), 0,
                           stream, a);
    }
    return hipGetLastError();
}

template <int R, int X>
hipError_t launch_w4(const W4Args& a, bool vec, uint64_t cus, hipStream_t stream) {
    if (a.group % 128 == 0) return launch_w4<R, 4, X>(a, vec, cus, stream);
    if (a.group % 64 == 0) return launch_w4<R, 2, X>(a, vec, cus, stream);
    return launch_w4<R, 1, X>(a, vec, cus, stream);
}

template <int R>
hipError_t launch_w4(const W4Args& a, bool vec, uint64_t cus, hipStream_t stream) {
    return a.tokens <= 8 ? launch_w4<R, 2>(a, vec, cus, stream)
                         : launch_w4<R, 4>(a, vec, cus, stream);
}

// Many rows and tokens: RW of the W waves take row tiles of their own and share x, so that a
// workgroup reads x once for 16 RW rows and unpacks codes once for 16 TT tokens; the W / RW
// groups of waves split the columns.  x goes through two LDS tiles in turn: each wave of a
// group loads its part of the next tile into registers, and one barrier a column tile parts
// the writes from the reads.  Tiles past the last column are zeros through the range checks,
// so every wave runs the same number of rounds.  Sixteen waves where a workgroup has its CU
// to itself: eight leave it waiting for the barrier (64 tokens, 12000 x 12000: 40.6 us against
// 51.2; but two workgroups of sixteen do not fit a CU's registers).
template <int TT, int RW, int W, int SPS, bool VEC>
__global__ __launch_bounds__(64 * W) void w4_matmul(W4Args a) {
    constexpr uint32_t kGroups = W / RW;
    constexpr int kLoads = 4 * TT / RW;  // of a wave for a tile of x
    static_assert(kLoads * RW == 4 * TT);
    constexpr uint32_t kRows = 16 * RW;
    union Shared {
        f16x8 x[2][kGroups][TT][256];
        float part[kGroups][16 * TT][kRows + 1];
    };
    __shared__ __attribute__((aligned(16))) Shared s_mem;
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t n = lane & 15u, gq = lane >> 4;
    const uint32_t kg = wave / RW, rg = wave % RW;
    // a row tile past the last one repeats it and is not stored
    const uint32_t rt = min(blockIdx.x * RW + rg, a.row_tiles - 1u);
    const uint32_t t0 = blockIdx.y * 16u * TT;
    const uint32_t live = min(a.tokens - t0, 16u * (uint32_t)TT);
    const W4Consts consts;
    const BufRsrc rw = make_rsrc(a.w + (uint64_t)rt * a.col_tiles * 256u, a.col_tiles * 1024u);
    // lane n takes the scales of step n / 4
    const f16* const sc = a.scales + rt * 16u + 4u * gq;
    const uint64_t sc_stride = (uint64_t)a.row_tiles * 16u;
    const f16* const xb = a.x + (uint64_t)t0 * a.x_stride;
    const BufRsrc rx = make_rsrc(xb, (uint32_t)(((live - 1u) * a.x_stride + a.cols) * 2u));
    // load i of this wave: rows 4 (rg + RW i) .. + 3 of the token tiles, 256 bytes each
    uint64_t x_at[kLoads];  // elements
    uint32_t x_to[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const uint32_t q = rg + RW * i, r = 4u * (q & 3u) + gq;
        x_at[i] = min(4u * q + gq, live - 1u) * a.x_stride + 8u * n;
        x_to[i] = (q >> 2) * 256u + 16u * r + (n ^ r);
    }
    struct Weights {
        u32x4 w;
        u32x2 scale;  // rows 4 gq ..
    };
    f16x8 xr[kLoads];
    auto load_x = [&](uint32_t c) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
            xr[i] = w4_load_x<VEC>(rx, xb, x_at[i] + 128u * c, c, 128u * c + 8u * n, a.cols);
    };
    auto load_w = [&](uint32_t c, Weights& z) {
        z.w = w4_load(rw, c * 1024u + 16u * lane);
        z.scale = *reinterpret_cast<const u32x2*>(
            sc + w4_group(a, min(128u * c + 32u * (n >> 2), a.cols - 1u)) * sc_stride);
    };
    f32x4 acc[TT];
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) acc[tt] = f32x4{0.f, 0.f, 0.f, 0.f};
    // Groups of 32, three token tiles and more or sixteen waves: a step's sums are scaled
    // after the next step's products, which hide the MFMAs' latency (48 tokens, 16384 x 4096,
    // eight waves 18.3 us against 22.9; 32 tokens, 12000 x 12000, sixteen 31.8 against 38.3; with
    // wider groups the compiler's order is the better one, 15.4 against 17.2 with groups of 64).
    constexpr bool kLate = SPS == 1 && (TT > 2 || W == 16);
    auto compute = [&](const f16x8 (*x)[256], const Weights& z) {
        f32x4 part[kLate ? 2 : 1][TT];
        auto add = [&]<int g>() {
            const f16x4 scale = w4_lane_scale<4 * SPS * g>(z.scale);
#pragma unroll
            for (int tt = 0; tt < TT; ++tt)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    acc[tt][r] =
                        __builtin_fmaf((float)scale[r], part[kLate ? g & 1 : 0][tt][r], acc[tt][r]);
        };
        auto step = [&]<int s>() {
            constexpr int g = s / SPS, p = kLate ? g & 1 : 0;
            f16x8 xv[TT];
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) xv[tt] = x[tt][16u * n + ((4u * s + gq) ^ n)];
            const f16x8 wv = w4_values(z.w[s], consts);
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) {
                if (s % SPS == 0) part[p][tt] = f32x4{0.f, 0.f, 0.f, 0.f};
                part[p][tt] = mfma16(wv, xv[tt], part[p][tt]);
            }
            if constexpr (kLate && s > 0) {
                __builtin_amdgcn_sched_barrier(0);
                add.template operator()<g - 1>();
                __builtin_amdgcn_sched_barrier(0);
            }
            if constexpr (!kLate && s % SPS == SPS - 1) add.template operator()<g>();
            if constexpr (W == 16 && TT == 3 && SPS == 4)
                __builtin_amdgcn_sched_barrier(0);  // else 129 registers
        };
        step.template operator()<0>();
        step.template operator()<1>();
        step.template operator()<2>();
        step.template operator()<3>();
        if constexpr (kLate) add.template operator()<3>();
    };
    Weights wa, wb;
    load_w(kg, wa);
    load_x(kg);
    auto round = [&](uint32_t c, uint32_t buf, const Weights& now, Weights& next) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) (&s_mem.x[buf][kg][0][0])[x_to[i]] = xr[i];
        __syncthreads();
        load_w(c + kGroups, next);
        load_x(c + kGroups);
        compute(s_mem.x[buf][kg], now);
    };
    for (uint32_t c = kg; c < a.col_tiles + kg; c += 2u * kGroups) {
        round(c, 0u, wa, wb);
        round(c + kGroups, 1u, wb, wa);
    }
    __syncthreads();  // x is read
#pragma unroll
    for (int tt = 0; tt < TT; ++tt)
#pragma unroll
        for (int r = 0; r < 4; ++r)
            s_mem.part[kg][16 * tt + n][16u * rg + 4u * gq + r] = acc[tt][r];
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < live * kRows; i += 64u * W) {
        const uint32_t t = i / kRows, r = i % kRows, row = blockIdx.x * kRows + r;
        if (row >= a.rows) continue;
        float sum = 0.f;
#pragma unroll
        for (uint32_t x = 0; x < kGroups; ++x) sum += s_mem.part[x][t][r];
        const uint64_t at = (uint64_t)(t0 + t) * a.y_stride + row;
        if (a.residual) sum += (float)a.residual[at];
        a.y[at] = (f16)sum;
    }
}

template <int TT, int RW, int W, bool VEC>
hipError_t launch_w4_matmul(const W4Args& a, hipStream_t stream) {
    const dim3 grid((a.row_tiles + RW - 1u) / RW, (a.tokens + 16u * TT - 1u) / (16u * TT));
    const dim3 block(64 * W);
    if (a.group % 128 == 0)
        hipLaunchKernelGGL((w4_matmul<TT, RW, W, 4, VEC>), grid, block, 0, stream, a);
    else if (a.group % 64 == 0)
        hipLaunchKernelGGL((w4_matmul<TT, RW, W, 2, VEC>), grid, block, 0, stream, a);
    else if constexpr (W == 8 || TT < 4 || VEC)
        hipLaunchKernelGGL((w4_matmul<TT, RW, W, 1, VEC>), grid, block, 0, stream, a);
    else
        return hipErrorInvalidValue;  // not asked for
    return hipGetLastError();
}

template <int TT, int RW, int W>
hipError_t launch_w4_matmul(const W4Args& a, bool vec, hipStream_t stream) {
    return vec ? launch_w4_matmul<TT, RW, W, true>(a, stream)
               : launch_w4_matmul<TT, RW, W, false>(a, stream);
}

hipError_t launch_w4_narrow(const W4Args& a, bool vec, hipStream_t stream) {
    const uint32_t tiles = kW4Waves / a.split;
    const dim3 grid((a.row_tiles + tiles - 1u) / tiles);
    if (vec)
        hipLaunchKernelGGL(w4_matvec_narrow<true>, grid, dim3(64 * kW4Waves), 0, stream, a);
    else
        hipLaunchKernelGGL(w4_matvec_narrow<false>, grid, dim3(64 * kW4Waves), 0, stream, a);
    return hipGetLastError();
}

// Waves per row tile, no more than there are column tiles.  Narrow: enough for eight waves
// a CU.  Otherwise as many as there are (33 tokens, 2048 x 11008: 13 us with eight, 22 with
// four).
uint32_t w4_split(uint32_t row_tiles, uint32_t col_tiles, bool narrow, int cus) {
    uint32_t split = 1;
    while (split < kW4Waves && 2u * split <= col_tiles &&
           (!narrow || (uint64_t)row_tiles * split < 8ull * (uint32_t)cus))
        split *= 2;
    return split;
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
    return rows <= 0x7ffffff0u && cols <= (1u << 20) && group > 0 && group % 32 == 0 &&
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
        (num_tokens > 1 && y_stride && y_stride < out_dim) ||
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
    a.group_mul = group_size >= in_dim
                      ? 0u
                      : (uint32_t)(((1ull << 31) + group_size / 32 - 1) / (group_size / 32));
    int device = 0;
    const hipError_t e = hipGetDevice(&device);
    if (e != hipSuccess) return (int)e;
    a.split = w4_split(a.row_tiles, a.col_tiles, a.tokens <= 4, device_cu_count(device));
    // reads of x through one 32-bit range per workgroup
    const uint64_t x_range = (std::min<uint64_t>(a.tokens, 64) - 1) * a.x_stride + in_dim;
    const bool vec = aligned16(x) && a.x_stride % 8 == 0 && in_dim % 8 == 0 &&
                     a.x_stride < (1ull << 31) && x_range * 2 < kDead;
    if (a.tokens <= 4) return (int)launch_w4_narrow(a, vec, stream);
    // Which kernel, by the workgroups it makes.  P r: own x for every wave, r row tiles; S t w:
    // x shared by w waves of a row tile each, t token tiles, eight waves in all; L t: S t 4 with
    // sixteen (us in a graph, groups of 64; tokens x rows x columns, CUs 256):
    //                       P 1   P 2  S 1 2  S 1 4  S 2 4  S 3 4  S 4 4   L 2   L 3   L 4
    //  16 x 4096 x 4096     5.4   6.1   6.6    9.8   10.9   13.6   16.6
    //  16 x 8192 x 8192    12.4  10.7  12.3   18.3   20.2   24.7   30.4
    //  16 x 11008 x 2048    7.0   6.3   5.7    6.7    7.3    8.6   10.0   6.6   7.7   8.8
    //  16 x 128256 x 2048  49.8  38.0  33.6   29.4   37.3   46.7   55.5
    //  33 x 2048 x 2048     4.7   4.3   4.1    5.2    6.5    8.2    9.6
    //  64 x 2048 x 11008   14.8  12.0  15.0   23.4   26.3   33.6   40.6
    //  32 x 8192 x 8192    20.9  15.5  14.7   18.5   20.3   24.8   30.7  17.6  20.6  24.4
    //  64 x 4096 x 4096    11.8   9.3   8.7   10.0   11.1   14.2   16.7   9.8  12.0  14.2
    //  32 x 11008 x 2048          8.1   7.1    8.4    7.3    8.3    9.9   6.7   7.7   9.0
    //  32 x 24000 x 2048   18.1  14.8  12.4   11.7   10.2   12.5   14.8
    //  48 x 8192 x 4096    16.3  13.2  12.5   12.7   13.0   14.5   17.0  11.4  12.7  14.7
    //  33 x 16384 x 2048         13.4  11.4   10.2    9.9    8.9   10.2  11.9   8.3   9.2
    //  64 x 6000 x 4096    17.8  14.4  11.8   14.1   12.2   14.0   16.6  10.7  12.6  14.5
    //  64 x 8192 x 8192    36.4  26.5  25.4   22.6   21.3   25.2   29.4  18.6  21.7  25.2
    //  64 x 9000 x 4096                19.2   18.1   16.6   20.0   16.6  19.2  22.0  14.5
    //  64 x 20000 x 2048   27.8  22.4  18.2   19.9   13.6   19.3   15.8  18.2  20.6  17.2
    //  64 x 30000 x 2048         32.2  26.3   26.0   19.4   24.2   16.9
    //  64 x 128256 x 2048   160   122   106   91.9   66.1   90.5   63.2
    //  96 x 6000 x 4096    22.8  18.9  17.4   17.6   16.9   14.1   17.0  19.5  12.6  14.9
    const uint64_t cus = (uint32_t)device_cu_count(device);
    const uint64_t token_tiles = (a.tokens + 15u) / 16u;
    if (in_dim > 0) {
        const uint64_t quads = (a.row_tiles + 3u) / 4u, pairs = (a.row_tiles + 1u) / 2u;
        // Sixteen waves, a workgroup a CU at most: the fewest token tiles that make no more of
        // them (S 1 2 has more, but two a CU are as fast).
        if (pairs * token_tiles > 2u * cus && token_tiles > 1) {
            if (quads * ((token_tiles + 1u) / 2u) <= cus)
                return (int)launch_w4_matmul<2, 4, 16>(a, vec, stream);
            if (quads * ((token_tiles + 2u) / 3u) <= cus)
                return (int)launch_w4_matmul<3, 4, 16>(a, vec, stream);
            // (groups of 32 with rows of x at any element would spill 22 registers)
            if (quads * ((token_tiles + 3u) / 4u) <= cus && (vec || group_size % 64 == 0))
                return (int)launch_w4_matmul<4, 4, 16>(a, vec, stream);
        }
        // Eight: the most token tiles that fit the tokens (a fifth more at most) and leave
        // enough workgroups, in quarters of the CUs.
        const uint64_t enough[5] = {0, 16, 4, 4, 7};
        for (uint64_t tt = std::min<uint64_t>(4, token_tiles); tt > 0; --tt) {
            const uint64_t parts = (token_tiles + tt - 1u) / tt;
            if (5u * (parts * tt - token_tiles) > token_tiles) continue;
            if (4u * quads * parts < enough[tt] * cus) continue;
            if (tt == 4) return (int)launch_w4_matmul<4, 4, 8>(a, vec, stream);
            if (tt == 3) return (int)launch_w4_matmul<3, 4, 8>(a, vec, stream);
            if (tt == 2) return (int)launch_w4_matmul<2, 4, 8>(a, vec, stream);
            return (int)launch_w4_matmul<1, 4, 8>(a, vec, stream);
        }
        // more than one a CU, or nearly one and few column tiles (their barriers)
        const uint64_t groups = pairs * token_tiles;
        if (groups > cus || (4u * groups >= 3u * cus && a.col_tiles <= 32u))
            return (int)launch_w4_matmul<1, 2, 8>(a, vec, stream);
    }
    if (a.row_tiles * token_tiles > cus) return (int)launch_w4<2>(a, vec, cus, stream);
    return (int)launch_w4<1>(a, vec, cus, stream);
}

}  // extern "C"
