// Decode attention over a paged KV cache: one new token for each of a batch of
// sequences, out[b][h] = sum_j softmax_j(q[b][h] . k_j / sqrt(D)) v_j over the
// kv_lens[b] cached rows of sequence b, whose pages row b of the page table names.
//
// A sequence of length 0 (a row of a padded batch) leaves its output as it was.  A
// page number out of range makes its sequence's output NaN: nothing is read for it.
//
// Bound by the K/V bytes, 4 * Hkv * D per key; by latency for short contexts.  Measured
// (16/4 heads): 64 sequences of 100 to 16384 keys, heads of 128, 353 MB: split 65.0 us (5.4
// TB/s) and join 4.2 traced, 70.3 a call; one of 32768: 12.0 and 2.7, 16.9; 32 of 20 to 4096
// keys, heads of 64, 38 MB: 10.9 and 3.0, 13.9; one of 254: 5.1.
//
// Split.  The lengths are known on the device only, and differ.  The keys of all
// sequences, in units of 32 keys and one after the other, make one line of units; each
// workgroup of a KV head takes an equal, contiguous share of it (its position in the
// line comes from a scan of the lengths that every wave does by itself).  So every
// workgroup reads the same number of bytes whatever the lengths are, and the grid and
// the workspace depend on neither batch nor lengths.  A share may hold the end of one
// sequence, some whole ones and the start of another: whole ones are written to the
// output at once, pieces to the workspace as fp32 states (running maximum, sum,
// unnormalised output), and a second kernel joins a sequence's pieces.  Where no table
// row can hold more than a few hundred keys, a workgroup per sequence and KV head and no
// second kernel.
//
// A unit.  Four waves take units in turn, each with two in flight.  Scores are S^T = K
// Q^T on v_mfma_f32_16x16x32_f16 (32 keys x up to 16 query heads of the KV head, so K and
// V are read once for all of them; larger groups take further workgroups), with the key
// rows ordered so that the result is the B operand of O^T = V^T P^T: lane (gq, n) holds
// query n and keys 8 gq .. 8 gq + 7.  Pages enter through LDS: the workgroup turns its
// part of the table into the pool row of every eight keys (of every key where the page
// size is no multiple of 8), which a lane's loads start from.
//
// Rounding.  Scores, maxima, sums and states are fp32.  The weights are rounded to fp16
// for the PV product, scaled by 2^15 (weights are at most 1): they keep 11 bits down to
// 2^-29 of the largest, and the denominator sums the rounded ones.  V rows past the
// sequence's end are set to zero in registers (the cache may hold anything there).
#include "paged_internal.hpp"
#include "../../include/attn_mi355x.h"

#include <algorithm>
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

// A score in the log2 domain, rounded before anything is taken from it, and 2^(x - m +
// bits): x - m is then never above 0, however large the scores are.  (One multiply-add of
// score, scale and -m is off by half a step of m instead, 32 at scores of 10^9, and the
// weight overflows.)
__device__ __forceinline__ float scaled_score(float dot, float scale) {
#pragma clang fp contract(off)
    return dot * scale;
}
__device__ __forceinline__ float weight(float x, float m, float bits) {
#pragma clang fp contract(off)
    return fast_exp2((x - m) + bits);
}

// Head dims other than 64 and 128, unaligned tensors: one workgroup per sequence and
// query head, tiles of 256 keys, one score per thread, then a dim per
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
            s = scaled_score(dot, a.scale_log2);
        }
        const float wm = wave_max(s);
        if ((tid & 63u) == 0) s_red[0][wave] = wm;
        __syncthreads();
        const float m_new = fmaxf(fmaxf(fmaxf(s_red[0][0], s_red[0][1]),
                                        fmaxf(s_red[0][2], s_red[0][3])), m_run);
        const float p = j < len ? weight(s, m_new, 0.f) : 0.f;
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

// ------------------------------------------------------------------ split and merge

constexpr uint32_t kWaves = 4;
constexpr uint32_t kThreads = 64 * kWaves;
constexpr uint32_t kUnit = 32;          // keys
constexpr uint32_t kMinUnits = 4;       // least share of a workgroup: a unit per wave
constexpr uint32_t kLead = 4;           // units that the start of a sequence counts for
constexpr uint32_t kMaxGroups = 512;    // workgroups over all head groups (two per CU)
// longest table rows that take no split: any batch, and batches that give half the CUs a
// workgroup (see attn_paged_decode)
constexpr uint32_t kWholeKeys = 512, kWholeKeysBatch = 1024;
constexpr uint32_t kEntries = 1024;     // pool rows staged at once
constexpr float kNoMax = -1.0e30f;      // finite: masked scores (-inf) get weight 0
constexpr float kWeightBits = 15.0f;

struct PagedSplitArgs {
    PagedDecodeArgs d;
    float* acc;           // [head groups][2 wgs][heads][D]  (workspace)
    float* m;             // [head groups][2 wgs][heads], log2 domain
    float* l;
    uint32_t* plan;       // [num_seqs][2]: first and last workgroup of a sequence
    uint32_t parts;       // head groups per KV head
    uint32_t head_groups; // Hkv * parts
    uint32_t heads;       // heads of a state: min(group, 16)
    uint32_t wgs;         // workgroups per head group
    uint32_t dim_parts;   // merge: workgroups per sequence and head
};

// v summed over the lanes up to this one: DPP row shifts within 16 lanes, then row
// broadcasts
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xF, 0xF, false);  // row_shr:1
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false);  // row_bcast:15
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false);  // row_bcast:31
    return v;
}

__device__ __forceinline__ uint32_t len_of(const PagedDecodeArgs& a, uint32_t b) {
    return b < a.num_seqs ? clamp_len(a.lens[b], a.max_pages, a.page_size) : 0u;
}

// Places of a sequence in the line: its units behind a lead, which stands for the time
// that taking a sequence up costs a workgroup besides its keys (queries, pages, the first
// loads' latency, the waves' meeting).
__device__ __forceinline__ uint32_t line_units(uint32_t len) {
    return len ? (len + kUnit - 1u) / kUnit + kLead : 0u;
}

// Pools by size: rows below 4 GiB a plane are read through a buffer resource, whose 32-bit
// offsets take a multiply-add per row and whose reads of rows that are not live fetch
// nothing (an offset past the range); larger ones through 64-bit addresses.  K and V of a
// layer that the last-level cache (256 MiB) may keep from one call to the next are read
// without the non-temporal hint, which else pays off because each byte is read once.  us
// without / with it: 64 ragged sequences, 353 MB 74.6 / 71.0; 16 of 4 K keys, 134 MB 32.1 /
// 30.4; one of 32768, 67 MB 18.5 / 20.3; 32 of 64-dim heads, 38 MB 15.0 / 15.5.
enum { kPoolCached = 0, kPoolStreamed = 1, kPoolHuge = 2 };
constexpr uint64_t kCachedBytes = 100ull << 20;  // of one K or V plane pair

template <int POOL>
struct PoolRows {
    const char* base;
    BufRsrc rsrc;
    uint32_t row_bytes, lane_bytes;
    __device__ PoolRows(const f16* plane, uint64_t bytes, uint32_t row, uint32_t lane)
        : base(reinterpret_cast<const char*>(plane) + lane),
          rsrc(make_rsrc(plane, (uint32_t)bytes)),
          row_bytes(row),
          lane_bytes(lane) {}
    template <class T>
    __device__ __forceinline__ T get(uint32_t row, uint32_t extra, bool live) const {
        constexpr int AUX = POOL == kPoolCached ? 0 : 2;  // bit 1: non-temporal
        if constexpr (POOL == kPoolHuge) {
            return __builtin_nontemporal_load(
                reinterpret_cast<const T*>(base + (uint64_t)row * row_bytes + extra));
        } else {
            const uint32_t at = live ? row * row_bytes + lane_bytes : 0xfffff000u;
            if constexpr (sizeof(T) == 16)
                return __builtin_bit_cast(
                    T, __builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)(at + extra), 0, AUX));
            else
                return __builtin_bit_cast(
                    T, __builtin_amdgcn_raw_buffer_load_b64(rsrc, (int)(at + extra), 0, AUX));
        }
    }
};

// D: head dim (128 or 64).  OCT: the page size is a multiple of 8.  WHOLE: workgroup
// (head group, sequence) takes the whole sequence.
template <int D, bool OCT, bool WHOLE, int POOL>
__global__ __launch_bounds__(kThreads, 2) void paged_decode_split(PagedSplitArgs sa) {
    constexpr int kSteps = D / 32;            // MFMAs of a score tile
    constexpr int kTiles = D / 16;            // output tiles, dims {kTiles m + mt}
    constexpr uint32_t kGran = OCT ? 8 : 1;   // keys per staged row
    constexpr uint32_t kBlock = kEntries * kGran / kUnit;  // units staged at once
    constexpr int kPitch = D + 4;
    typedef _Float16 VRow __attribute__((ext_vector_type(kTiles)));
    __shared__ uint32_t s_row[kEntries];
    __shared__ __attribute__((aligned(16))) float s_acc[kWaves][16][kPitch];
    __shared__ float s_m[kWaves][16], s_l[kWaves][16];
    __shared__ uint32_t s_bad;
    const PagedDecodeArgs& a = sa.d;
    const uint32_t tid = threadIdx.x, lane = tid & 63u;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t n = lane & 15u, gq = lane >> 4;
    const uint32_t hg = WHOLE ? blockIdx.x : blockIdx.x % sa.head_groups;
    const uint32_t w = WHOLE ? 0u : blockIdx.x / sa.head_groups;
    const uint32_t g = hg / sa.parts, part = hg - g * sa.parts;
    const uint32_t h0 = g * a.group + 16u * part;
    const uint32_t heads = min(16u, a.group - 16u * part);
    const uint32_t row_bytes = a.num_kv_heads * D * 2u;
    const uint64_t plane = (uint64_t)a.num_pages * a.page_size * row_bytes;
    const PoolRows<POOL> rows_k(a.kp, plane, row_bytes, (g * D + 8u * gq) * 2u);
    const PoolRows<POOL> rows_v(a.vp, plane, row_bytes, (g * D + (uint32_t)kTiles * n) * 2u);
    struct Batch {
        f16x8 k[2][kSteps];
        VRow v[8];
    };
    // S^T row m of score tile tt is key 8 (m / 4) + 4 tt + m % 4 of the unit
    const uint32_t koct = n >> 2, kin = n & 3u;

    // this workgroup's units [u0, u1) of the line, the sequence that holds u0 and that
    // sequence's first unit
    uint32_t b, u, u1, base, len, share = 1;
    // WHOLE: the row's pages are fetched together with its length, which says later how many
    // of them count (128 sequences of 50 keys: 5.8 us against 6.3; one of 254: 5.5, 5.6)
    constexpr uint32_t kAhead = WHOLE ? (kWholeKeysBatch / kGran + kThreads - 1) / kThreads : 1;
    uint32_t page_ahead[kAhead];
    if constexpr (WHOLE) {
        if (tid == 0) s_bad = 0;
        b = blockIdx.y;
        u = base = 0;
#pragma unroll
        for (uint32_t x = 0; x < kAhead; ++x) {
            const uint32_t j = (tid + x * kThreads) * kGran / a.page_size;
            page_ahead[x] = j < a.max_pages ? (uint32_t)a.table[(uint64_t)b * a.max_pages + j] : 0u;
        }
        len = clamp_len(a.lens[b], a.max_pages, a.page_size);
        u1 = (len + kUnit - 1u) / kUnit;
    } else {
        const uint32_t len0 = len_of(a, lane), mine0 = line_units(len0), incl0 = wave_scan(mine0);
        uint32_t total = (uint32_t)__builtin_amdgcn_readlane((int)incl0, 63);
        for (uint32_t b0 = 64; b0 < a.num_seqs; b0 += 64u)
            total += (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(line_units(len_of(a, b0 + lane))), 63);
        // the line begins behind the first sequence's lead
        const uint32_t line = total > kLead ? total - kLead : 0u;
        share = max(kMinUnits, (line + sa.wgs - 1u) / sa.wgs);
        if ((uint64_t)w * share >= line) return;
        u = kLead + w * share;
        u1 = min(total, u + share);
        b = base = 0;
        uint32_t mine_len = len0, mine = mine0, incl = incl0;
        for (uint32_t b0 = 0;; b0 += 64u) {
            if (b0 > 0) {
                mine_len = len_of(a, b0 + lane);
                mine = line_units(mine_len);
                incl = wave_scan(mine);
            }
            const uint64_t past = __ballot(base + incl > u);
            if (past) {
                const int at = (int)__builtin_ctzll(past);
                b = b0 + (uint32_t)at;
                base += (uint32_t)__builtin_amdgcn_readlane((int)(incl - mine), at);
                len = (uint32_t)__builtin_amdgcn_readlane((int)mine_len, at);
                break;
            }
            base += (uint32_t)__builtin_amdgcn_readlane((int)incl, 63);
        }
    }

    constexpr uint32_t kSkip = WHOLE ? 0u : kLead;
    while (u < u1) {
        const uint32_t units = (len + kUnit - 1u) / kUnit;
        if (units == 0) {
            ++b;
            len = clamp_len(a.lens[b], a.max_pages, a.page_size);
            continue;
        }
        if (u < base + kSkip) {  // the lead of the sequence holds no keys
            u = base + kSkip;
            continue;
        }
        const uint32_t rel = u - base - kSkip;            // first unit of this piece
        const uint32_t count = min(units - rel, u1 - u);  // its units
        const bool complete = count == units;

        // Q^T as the B operand: lane (gq, n) holds Q[n][32 s + 8 gq ..]
        f16x8 qb[kSteps];
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
            qb[s] = n < heads ? ld16(a.q + b * a.q_stride + (uint64_t)(h0 + n) * D + 32 * s + 8 * gq)
                              : f16x8{};
        f32x4 acc[kTiles];
#pragma unroll
        for (int mt = 0; mt < kTiles; ++mt) acc[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
        float m_run = kNoMax, l_run = 0.f;
        if (!WHOLE && tid == 0) s_bad = 0;

        for (uint32_t blk = 0; blk < (WHOLE ? 1u : count); blk += kBlock) {
            const uint32_t nu = min(kBlock, count - blk);  // units of this block
            const uint32_t key0 = (rel + blk) * kUnit;
            __syncthreads();  // the last block's rows are read; s_bad is cleared
            auto stage = [&](uint32_t i, auto page_of) {
                const uint32_t key = key0 + i * kGran;
                uint32_t row = 0;
                if (key < len) {
                    const uint32_t j = key / a.page_size, page = page_of(j);
                    if (page < a.num_pages)
                        row = page * a.page_size + (key - j * a.page_size);
                    else
                        s_bad = 1;
                }
                s_row[i] = row;
            };
            if constexpr (WHOLE) {
#pragma unroll
                for (uint32_t x = 0; x < kAhead; ++x) {
                    const uint32_t i = tid + x * kThreads;
                    if (i < nu * (kUnit / kGran)) stage(i, [&](uint32_t) { return page_ahead[x]; });
                }
            } else {
                for (uint32_t i = tid; i < nu * (kUnit / kGran); i += kThreads)
                    stage(i, [&](uint32_t j) {
                        return (uint32_t)a.table[(uint64_t)b * a.max_pages + j];
                    });
            }
            __syncthreads();
            const uint32_t nk = min(len - key0, nu * kUnit);  // keys of this block

            auto load = [&](uint32_t un, Batch& x) {
                const bool live = un < nu;  // a load past the block fetches nothing of it
#pragma unroll
                for (int tt = 0; tt < 2; ++tt) {
                    const uint32_t kr = OCT ? s_row[live ? 4u * un + koct : 0u] + 4u * tt + kin
                                            : s_row[live ? 32u * un + 8u * koct + 4u * tt + kin : 0u];
#pragma unroll
                    for (int s = 0; s < kSteps; ++s)
                        x.k[tt][s] = rows_k.template get<f16x8>(kr, 64u * s, live);
                }
#pragma unroll
                for (uint32_t r = 0; r < 8; ++r) {
                    const uint32_t vr = OCT ? s_row[live ? 4u * un + gq : 0u] + r
                                            : s_row[live ? 32u * un + 8u * gq + r : 0u];
                    x.v[r] = rows_v.template get<VRow>(vr, 0u, live);
                }
            };
            auto compute = [&](uint32_t un, Batch& x) {
                f32x4 st[2];
#pragma unroll
                for (int tt = 0; tt < 2; ++tt) {
                    st[tt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int s = 0; s < kSteps; ++s) st[tt] = mfma16(x.k[tt][s], qb[s], st[tt]);
                }
                if ((un + 1u) * kUnit > nk) {  // the unit that holds the sequence's end
                    const uint32_t left = nk - un * kUnit;
#pragma unroll
                    for (uint32_t r = 0; r < 8; ++r)
                        if (8u * gq + r >= left) {
                            st[r >> 2][r & 3] = -INFINITY;
                            x.v[r] = VRow{};
                        }
                }
                float x_log2[8], mx = -INFINITY;
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    x_log2[r] = scaled_score(st[r >> 2][r & 3], a.scale_log2);
                    mx = fmaxf(mx, x_log2[r]);
                }
                mx = max_xor<32>(max_xor<16>(mx));
                const float m_new = fmaxf(m_run, mx);
                const float alpha = fast_exp2(m_run - m_new);
                f16x8 p;
#pragma unroll
                for (int r = 0; r < 8; ++r) p[r] = (f16)weight(x_log2[r], m_new, kWeightBits);
                const f16x2 one = {(f16)1.0f, (f16)1.0f};
                float sum = 0.f;
#pragma unroll
                for (int r = 0; r < 8; r += 2)
                    sum = __builtin_amdgcn_fdot2(f16x2{p[r], p[r + 1]}, one, sum, false);
                l_run = l_run * alpha + sum;
                m_run = m_new;
#pragma unroll
                for (int mt = 0; mt < kTiles; ++mt) {
                    f16x8 va;
#pragma unroll
                    for (int r = 0; r < 8; ++r) va[r] = x.v[r][mt];
                    acc[mt] = mfma16(va, p, acc[mt] * alpha);
                }
            };

            // Units wave, wave + 4, ...; two in flight, the next load going out as soon as
            // a unit is computed.  Every path into the loop has exactly A and B in flight,
            // so that the compiler's wait for A leaves B's loads running; the scheduler
            // barriers keep the loads of one unit out of the arithmetic of another (without
            // them the 128-dim kernels spilled 128 registers).
            // Planes of 4 GiB or more take one unit at a time (two and their 64-bit addresses do
            // not fit the registers).
            uint32_t un = wave;
            Batch A, B;
            if constexpr (POOL == kPoolHuge) {
                for (; un < nu; un += kWaves) {
                    load(un, A);
                    compute(un, A);
                }
            } else if (un + kWaves < nu) {
                load(un, A);
                load(un + kWaves, B);
                while (un + 2u * kWaves < nu) {
                    __builtin_amdgcn_sched_barrier(0);
                    compute(un, A);
                    load(un + 2u * kWaves, A);
                    __builtin_amdgcn_sched_barrier(0);
                    compute(un + kWaves, B);
                    load(un + 3u * kWaves, B);
                    un += 2u * kWaves;
                }
                __builtin_amdgcn_sched_barrier(0);
                compute(un, A);
                __builtin_amdgcn_sched_barrier(0);
                if (un + kWaves < nu) compute(un + kWaves, B);
            } else if (un < nu) {
                load(un, A);
                compute(un, A);
            }
        }

        // the waves' states meet in LDS
        l_run = add_xor<32>(add_xor<16>(l_run));
        if (n < heads) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int t4 = 0; t4 < kTiles; t4 += 4)
                    *reinterpret_cast<f32x4*>(&s_acc[wave][n][kTiles * (4 * gq + i) + t4]) =
                        f32x4{acc[t4][i], acc[t4 + 1][i], acc[t4 + 2][i], acc[t4 + 3][i]};
        }
        if (gq == 0) {
            s_m[wave][n] = m_run;
            s_l[wave][n] = l_run;
        }
        __syncthreads();
        const uint64_t slot = WHOLE ? 0 : (uint64_t)hg * 2u * sa.wgs + 2u * w + (rel == 0 ? 1u : 0u);
        for (uint32_t i = tid; i < heads * (D / 4); i += kThreads) {
            const uint32_t h = i / (D / 4), d = 4u * (i - h * (D / 4));
            float M = s_m[0][h];
#pragma unroll
            for (uint32_t x = 1; x < kWaves; ++x) M = fmaxf(M, s_m[x][h]);
            f32x4 sum = {0.f, 0.f, 0.f, 0.f};
            float L = 0.f;
#pragma unroll
            for (uint32_t x = 0; x < kWaves; ++x) {
                const float wt = fast_exp2(s_m[x][h] - M);
                sum += *reinterpret_cast<const f32x4*>(&s_acc[x][h][d]) * wt;
                L += s_l[x][h] * wt;
            }
            if (s_bad) L = __builtin_nanf("");
            if (complete) {
                const float inv = 1.0f / L;
                const f16x4 o = {(f16)(sum[0] * inv), (f16)(sum[1] * inv), (f16)(sum[2] * inv),
                                 (f16)(sum[3] * inv)};
                *reinterpret_cast<f16x4*>(a.out + ((uint64_t)b * a.num_heads + h0 + h) * D + d) = o;
            } else if constexpr (!WHOLE) {
                const uint64_t st = slot * sa.heads + h;
                *reinterpret_cast<f32x4*>(sa.acc + st * D + d) = sum;
                if (d == 0) {
                    sa.m[st] = M;
                    sa.l[st] = L;
                }
            }
        }
        if constexpr (!WHOLE) {
            if (rel == 0 && hg == 0 && tid == 0) {
                sa.plan[2 * b] = w;
                sa.plan[2 * b + 1] = (base + units - 1u) / share;  // unit base + lead + units - 1
            }
        }
        if constexpr (WHOLE) return;
        __syncthreads();  // the states are read
        u += count;
        base += kSkip + units;
        ++b;
        if (u < u1) len = clamp_len(a.lens[b], a.max_pages, a.page_size);
    }
}

// Joins the pieces of sequence blockIdx.y for one query head (for a part of its dims): the
// largest maximum, then 4 dims a thread, the pieces shared out over the thread groups.
// A sequence in one piece is written already.
template <int D>
__global__ __launch_bounds__(kThreads) void paged_decode_merge(PagedSplitArgs sa) {
    __shared__ float s_max[kWaves];
    __shared__ __attribute__((aligned(16))) f32x4 s_x[kWaves][D / 4];
    __shared__ float s_den[kWaves];
    const PagedDecodeArgs& a = sa.d;
    const uint32_t b = blockIdx.y, tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    const uint32_t h = blockIdx.x / sa.dim_parts, dp = blockIdx.x - h * sa.dim_parts;
    const uint32_t g = h / a.group, in_group = h - g * a.group;
    const uint32_t hg = g * sa.parts + in_group / 16u;
    const uint64_t hg0 = (uint64_t)hg * 2u * sa.wgs;
    // state of piece j of a sequence that begins with workgroup wf, within its share
    auto state = [&](uint32_t wf, uint32_t j) {
        return (hg0 + 2u * (wf + j) + (j == 0 ? 1u : 0u)) * sa.heads + in_group % 16u;
    };
    // `lanes` threads (4 to 32) hold a state's dims; lane c of a group dims 4 c ..
    const uint32_t lanes = D / 4 / sa.dim_parts, groups = kThreads / lanes;
    const uint32_t grp = tid / lanes, c = tid - grp * lanes, d = dp * (D / sa.dim_parts) + 4u * c;
    // The first pieces of each group.  A batch of one begins with workgroup 0: its states
    // are fetched before the plan is known, a memory round trip less (one of 32768 keys
    // 18.5 -> 17.4 us); those past its pieces hold anything and are not used.
    constexpr uint32_t kFirst = 4;
    f32x4 x0[kFirst];
    float m0[kFirst], l0[kFirst];
    auto fetch = [&](uint32_t wf, uint32_t end) {  // below `end` only
#pragma unroll
        for (uint32_t i = 0; i < kFirst; ++i) {
            x0[i] = f32x4{0.f, 0.f, 0.f, 0.f};
            m0[i] = -INFINITY;
            l0[i] = 0.f;
            const uint32_t j = grp + groups * i;
            if (j < end) {
                const uint64_t st = state(wf, j);
                x0[i] = *reinterpret_cast<const f32x4*>(sa.acc + st * D + d);
                m0[i] = sa.m[st];
                l0[i] = sa.l[st];
            }
        }
    };
    if (a.num_seqs == 1) fetch(0u, sa.wgs);
    const uint32_t wf = sa.plan[2 * b], wl = sa.plan[2 * b + 1];  // nothing there without keys
    const uint32_t pieces = wl - wf + 1u;
    if (len_of(a, b) == 0 || pieces == 1) return;
    if (a.num_seqs != 1) fetch(wf, pieces);
    float M = -INFINITY;
#pragma unroll
    for (uint32_t i = 0; i < kFirst; ++i) {
        if (grp + groups * i >= pieces) {
            x0[i] = f32x4{0.f, 0.f, 0.f, 0.f};
            m0[i] = -INFINITY;
            l0[i] = 0.f;
        }
        M = fmaxf(M, m0[i]);
    }
    for (uint32_t j = groups * kFirst + tid; j < pieces; j += kThreads)
        M = fmaxf(M, sa.m[state(wf, j)]);
    M = wave_max(M);
    if (lane == 0) s_max[wave] = M;
    __syncthreads();
    M = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    float den = 0.f;
#pragma unroll
    for (uint32_t i = 0; i < kFirst; ++i) {
        const float wt = fast_exp2(m0[i] - M);  // past the last piece: 0
        x += x0[i] * wt;
        den += l0[i] * wt;
    }
#pragma unroll 4
    for (uint32_t j = grp + groups * kFirst; j < pieces; j += groups) {
        const uint64_t st = state(wf, j);
        const float wt = fast_exp2(sa.m[st] - M);
        x += *reinterpret_cast<const f32x4*>(sa.acc + st * D + d) * wt;
        den += sa.l[st] * wt;
    }
    // the groups of a wave, then the waves
    for (uint32_t mask = 32; mask >= lanes; mask >>= 1) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] += xor_lane(x[e], (int)mask);
        den += xor_lane(den, (int)mask);
    }
    if (lane < lanes) s_x[wave][lane] = x;
    if (lane == 0) s_den[wave] = den;
    __syncthreads();
    if (tid >= lanes) return;
    x = (s_x[0][tid] + s_x[1][tid]) + (s_x[2][tid] + s_x[3][tid]);
    const float inv = 1.0f / ((s_den[0] + s_den[1]) + (s_den[2] + s_den[3]));
    const f16x4 o = {(f16)(x[0] * inv), (f16)(x[1] * inv), (f16)(x[2] * inv), (f16)(x[3] * inv)};
    *reinterpret_cast<f16x4*>(a.out + ((uint64_t)b * a.num_heads + h) * D + d) = o;
}

// ------------------------------------------------------------------ host side

// Sizes of the split plan, and the workspace's arrays as byte offsets
struct PagedPlan {
    uint32_t parts, head_groups, heads, wgs;
    uint64_t at_m, at_l, at_acc, bytes;
};

PagedPlan paged_plan(size_t num_seqs, size_t num_heads, size_t num_kv_heads, size_t head_dim) {
    PagedPlan p{};
    const size_t group = num_heads / num_kv_heads;
    p.parts = (uint32_t)((group + 15) / 16);
    p.head_groups = (uint32_t)num_kv_heads * p.parts;
    p.heads = (uint32_t)std::min<size_t>(group, 16);
    p.wgs = std::max(1u, kMaxGroups / p.head_groups);
    const uint64_t states = 2ull * p.head_groups * p.wgs * p.heads;
    p.at_m = (num_seqs * 8 + 15) / 16 * 16;
    p.at_l = p.at_m + (states * 4 + 15) / 16 * 16;
    p.at_acc = p.at_l + (states * 4 + 15) / 16 * 16;
    p.bytes = p.at_acc + states * head_dim * 4;
    return p;
}

bool paged_split_dim(size_t head_dim) { return head_dim == 128 || head_dim == 64; }

template <int D, bool OCT, int POOL>
hipError_t launch_split(const PagedSplitArgs& a, bool whole, hipStream_t stream) {
    if (whole) {
        hipLaunchKernelGGL((paged_decode_split<D, OCT, true, POOL>),
                           dim3(a.head_groups, a.d.num_seqs), dim3(kThreads), 0, stream, a);
        return hipGetLastError();
    }
    hipLaunchKernelGGL((paged_decode_split<D, OCT, false, POOL>), dim3(a.head_groups * a.wgs),
                       dim3(kThreads), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((paged_decode_merge<D>), dim3(a.d.num_heads * a.dim_parts, a.d.num_seqs),
                       dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

template <int D, int POOL>
hipError_t launch_split(const PagedSplitArgs& a, bool whole, hipStream_t stream) {
    return a.d.page_size % 8 == 0 ? launch_split<D, true, POOL>(a, whole, stream)
                                  : launch_split<D, false, POOL>(a, whole, stream);
}

template <int D>
hipError_t launch_split(const PagedSplitArgs& a, bool whole, hipStream_t stream) {
    const uint64_t plane =
        (uint64_t)a.d.num_pages * a.d.page_size * a.d.num_kv_heads * D * 2;
    // buffer offsets reach 0xffffefff; the ones past it stand for rows that are not read
    if (plane > 0xffffe000ull) return launch_split<D, kPoolHuge>(a, whole, stream);
    if (2 * plane > kCachedBytes) return launch_split<D, kPoolStreamed>(a, whole, stream);
    return launch_split<D, kPoolCached>(a, whole, stream);
}

}  // namespace
}  // namespace attn

using namespace attn;

extern "C" {

size_t attn_paged_decode_workspace_bytes(size_t num_seqs, size_t num_heads, size_t num_kv_heads,
                                         size_t head_dim) {
    if (!paged_split_dim(head_dim) || num_kv_heads == 0 || num_heads < num_kv_heads) return 16;
    return paged_plan(num_seqs, num_heads, num_kv_heads, head_dim).bytes;
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
        !workspace || !aligned16(workspace))
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
    const uint64_t row_units = (max_pages * page_size + kUnit - 1) / kUnit;
    if (paged_split_dim(head_dim) && num_pages > 0 && a.q_stride % 8 == 0 && aligned16(q) &&
        aligned16(k_pages) && aligned16(v_pages) && aligned16(out) &&
        paged_mul(num_seqs, row_units + kLead) <= 0x7fffffffull &&
        get_option(kOptDecodeForceGeneric) == 0) {
        const PagedPlan p = paged_plan(num_seqs, num_heads, num_kv_heads, head_dim);
        PagedSplitArgs sa{};
        sa.d = a;
        char* const ws = static_cast<char*>(workspace);
        sa.plan = reinterpret_cast<uint32_t*>(ws);
        sa.m = reinterpret_cast<float*>(ws + p.at_m);
        sa.l = reinterpret_cast<float*>(ws + p.at_l);
        sa.acc = reinterpret_cast<float*>(ws + p.at_acc);
        sa.parts = p.parts;
        sa.head_groups = p.head_groups;
        sa.heads = p.heads;
        sa.wgs = p.wgs;
        // few sequences: more workgroups of fewer dims each join a long one's pieces
        sa.dim_parts = num_seqs * num_heads < 128 ? 4u : 1u;
        // One kernel, a workgroup per sequence and KV head, against two (us, 16/4 heads of
        // 128, rows of up to as many keys).  500 keys: 7.8 / 8.4 for one sequence, 10.7 / 15.9
        // for 64; 1000 keys: 12.0 / 8.4, 13.0 / 11.2 for 16, 13.7 / 14.7 for 32, 17.2 / 21.2 for
        // 64; 2000 keys: 40.7 / 37.9 for 64.
        const uint64_t keys = max_pages * page_size;
        int device = 0;
        const hipError_t e = hipGetDevice(&device);
        if (e != hipSuccess) return (int)e;
        const bool whole =
            keys <= kWholeKeys ||
            (keys <= kWholeKeysBatch &&
             2 * num_seqs * p.head_groups >= (uint64_t)device_cu_count(device));
        return (int)(head_dim == 128 ? launch_split<128>(sa, whole, stream)
                                     : launch_split<64>(sa, whole, stream));
    }
    hipLaunchKernelGGL(paged_decode_generic, dim3(a.num_heads, a.num_seqs), dim3(kTile), 0, stream,
                       a);
    return (int)hipGetLastError();
}

}  // extern "C"
