// Attention of a few new tokens per sequence over a paged key-value cache.
//
//   out[r] = sum_p softmax_p(c q_r . k_p) v_p,   p <= len - new + token(r),
//
// for the rows r = (new token, query head of the KV head's group).  Every cached byte is used once for
// 2 * rows * (bytes per value)^-1 multiply-adds -- 8 operations a byte for a group of four and bf16 -- so the
// cache has to stream from HBM at full rate and everything else has to stay out of its way.
//
// Work split.  An entry is one (sequence, KV head, tile of rows); its keys are cut into units of 64.  All
// units of all entries form one line that is cut into as many equal ranges as there are CTAs, whatever the
// lengths: a batch of unequal sequences and a single long one fill the GPU alike.  Where a cut falls inside an
// entry, the CTAs on its sides leave (maximum, sum, unnormalised row) and join_kernel adds them up
// in the order of the keys; so results depend on the lengths alone, not on timing.
//
// Inside a CTA every warp streams its own 16 keys of a unit through its own ring in shared memory
// (cp.async, no barrier between warps in the loop) and keeps its own softmax state; the four states are
// added up where an entry ends.  Scores are computed transposed, S^T = K Q^T: the keys fill the 16 rows of the
// matrix instruction and 8 queries its columns, so a group of 4 wastes half of a tile of 8 instead of three
// quarters of one of 16; the probabilities then need one 8x8 transpose to become the operand of
// O^T = V^T P^T.  mma.sync is enough: a tensor-core tile of 128 rows would be filled with padding, and the
// instruction rate needed is a sixth of what mma.sync reaches.
//
// Accuracy.  Scores, softmax state and outputs are held in 32 bits.  With bf16 pages a probability goes into
// the second product as the sum of two bf16 values (15 bits), so that only the output is rounded to 8;
// the extra instructions hide behind the loads.  With e4m3 pages both products run in f16, in which every
// code is exact and a probability keeps 11 bits; queries are scaled by a power of two per row to fit f16.
#pragma once
#include "paged_common.cuh"

namespace aa {
namespace paged {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kTileKeys = 16;                       // keys of one warp and step
constexpr int kUnitKeys = kWarps * kTileKeys;       // keys of one CTA and step
constexpr int kCombStride = 132;                    // floats; 132 keeps the transposed writes off each other's banks
constexpr int kCombBytes = kWarps * 8 * kCombStride * 4;
constexpr int kRingBytes = 96 * 1024;               // with the join buffer, two CTAs fill an SM's shared memory
constexpr int kCtasPerSm = 2;

constexpr int tile_bytes(bool fp8) { return kTileKeys * kD * (fp8 ? 1 : 2); }
constexpr int stages(bool fp8) { return kRingBytes / (kWarps * 2 * tile_bytes(fp8)); }
constexpr int kSmemBytes = kRingBytes + kCombBytes;

struct AttendParams {
    Cache c;
    const __nv_bfloat16* q;
    int64_t q_sb, q_sn, q_sh;                       // elements
    __nv_bfloat16* out;
    int64_t o_sb, o_sn, o_sh;
    float* lse;                                     // [B, nq, H] or null
    const int32_t* pages;                           // [B, Hkv, list_width] logical pages, or null: all pages
    const int32_t* page_counts;                     // [B, Hkv]
    int list_width;
    int B, H, Hkv, Hg, nq;
    int rows, row_tiles;                            // rows = nq * Hg in tiles of 8 * NT
    float scale_log2;                               // softmax scale times log2 e
    float* part_o;                                  // [ctas, 2, 8 NT, 128]
    float2* part_ml;                                // [ctas, 2, 8 NT]
    int32_t* cut_entry;                             // [ctas]: the entry a CTA's range starts inside of, or -1
};

// Keys an entry streams over (list entries count as whole pages) and the units they make; an empty one still
// makes a unit, so that some CTA writes its zeros.
__device__ __forceinline__ int entry_units(const AttendParams& p, int e) {
    const int bh = e / p.row_tiles;
    int64_t keys;
    if (p.pages) {
        keys = (int64_t)min(max(p.page_counts[bh], 0), p.list_width) << p.c.log2_page;
    } else {
        keys = seq_len(p.c, bh / p.Hkv);
    }
    return max(1, (int)((keys + kUnitKeys - 1) / kUnitKeys));
}

// One warp's place in the line of units.
struct Cursor {
    int entry, unit, units;                         // unit: next one of the entry
    int b, h, len;
};

__device__ __forceinline__ void enter(const AttendParams& p, Cursor& c, int entry) {
    c.entry = entry;
    c.units = entry_units(p, entry);
    const int bh = entry / p.row_tiles;
    c.b = bh / p.Hkv;
    c.h = bh - c.b * p.Hkv;
    c.len = seq_len(p.c, c.b);
}

// Where the 16 keys of (cursor, warp) are: the pool page, or -1 for none; `pos` their first position.
__device__ __forceinline__ int locate(const AttendParams& p, const Cursor& c, int warp, int& pos) {
    const int64_t flat = ((int64_t)c.unit * kWarps + warp) * kTileKeys;
    int logical = (int)(flat >> p.c.log2_page);
    const int within = (int)(flat & ((1 << p.c.log2_page) - 1));
    if (p.pages) {
        const int bh = c.b * p.Hkv + c.h;
        if (logical >= min(max(p.page_counts[bh], 0), p.list_width)) return -1;
        logical = p.pages[(int64_t)bh * p.list_width + logical];
        if (logical < 0 || ((int64_t)logical << p.c.log2_page) >= c.len) {
            raise_status(p.c, kStatusBadPage);
            return -1;
        }
    }
    const int64_t at = ((int64_t)logical << p.c.log2_page) + within;
    if (at >= c.len) return -1;
    pos = (int)at;
    const int page = pool_page(p.c, c.b, logical);
    if (page < 0) raise_status(p.c, kStatusBadPage);
    return page;
}

template <bool FP8>
__device__ __forceinline__ uint32_t tile_addr(uint32_t base, int row, int chunk) {
    // 16-byte chunks of a row, XORed with the row so that eight rows of a column of chunks fall on different banks
    return base + row * (FP8 ? kD : 2 * kD) + ((chunk ^ (row & 7)) << 4);
}

// One warp copies the keys and values of its 16 positions; rows behind the sequence's end become zeros.
template <bool FP8>
__device__ __forceinline__ void load_tile(const AttendParams& p, uint32_t slot, int page, int h, int pos, int len, int lane) {
    constexpr int kChunks = FP8 ? 8 : 16;
    const int row0 = pos & ((1 << p.c.log2_page) - 1);
    const uint8_t* k = p.c.k.ptr + page * p.c.k.page + h * p.c.k.head + row0 * p.c.k.row;
    const uint8_t* v = p.c.v.ptr + page * p.c.v.page + h * p.c.v.head + row0 * p.c.v.row;
    const int live = min(kTileKeys, len - pos);
#pragma unroll
    for (int i = 0; i < kTileKeys * kChunks / 32; ++i) {
        const int row = i * (32 / kChunks) + lane / kChunks, chunk = lane % kChunks;
        const bool in = row < live;
        cp_async16(tile_addr<FP8>(slot, row, chunk), k + (in ? row * p.c.k.row : 0) + chunk * 16, in ? 16 : 0);
        cp_async16(tile_addr<FP8>(slot + tile_bytes(FP8), row, chunk), v + (in ? row * p.c.v.row : 0) + chunk * 16,
                   in ? 16 : 0);
    }
}

// Query rows of an entry as operands of S^T = K Q^T, f16 and scaled by a power of two for e4m3 pages.
// Lane (g, t) holds row g of each tile of 8: the values that meet a lane's K values in step s.
template <bool FP8, int NT>
struct Queries {
    uint32_t f[NT][8][2];
    float unscale[NT][2];                           // of this lane's score columns 2t, 2t + 1 (e4m3 only)
};

template <bool FP8, int NT>
__device__ __forceinline__ void load_queries(const AttendParams& p, int b, int h, int row0, int lane, Queries<FP8, NT>& qf) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int r = row0 + n * 8 + g;
        const bool in = r < p.rows;
        const int j = in ? r / p.Hg : 0, i = in ? r - j * p.Hg : 0;
        const uint32_t* src =
            reinterpret_cast<const uint32_t*>(p.q + b * p.q_sb + j * p.q_sn + (int64_t)(h * p.Hg + i) * p.q_sh);
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            const int at = FP8 ? s * 8 + t * 2 : s * 8 + t;          // in pairs of values
            qf.f[n][s][0] = in ? src[at] : 0u;
            qf.f[n][s][1] = in ? src[at + (FP8 ? 1 : 4)] : 0u;
        }
        if (FP8) {
            uint32_t big = 0;                       // largest |q| of the row, as bf16 bits
#pragma unroll
            for (int s = 0; s < 8; ++s)
#pragma unroll
                for (int w = 0; w < 2; ++w)
                    big = max(big, max(qf.f[n][s][w] & 0x7FFFu, (qf.f[n][s][w] >> 16) & 0x7FFFu));
            big = max(big, __shfl_xor_sync(0xFFFFFFFFu, big, 1));
            big = max(big, __shfl_xor_sync(0xFFFFFFFFu, big, 2));
            // the row times 2^-e has its largest value in [256, 512): f16 then keeps 2^-32 of it
            const int expo = max(min((int)(big >> 7), 254) - 127 - 8, -126);
            const float down = __uint_as_float((uint32_t)(127 - expo) << 23);
            const float up = __uint_as_float((uint32_t)(127 + expo) << 23);
#pragma unroll
            for (int s = 0; s < 8; ++s)
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    const uint32_t x = qf.f[n][s][w];
                    qf.f[n][s][w] = pack_f16x2(__uint_as_float(x << 16) * down, __uint_as_float(x & 0xFFFF0000u) * down);
                }
            qf.unscale[n][0] = __shfl_sync(0xFFFFFFFFu, up, t * 8);
            qf.unscale[n][1] = __shfl_sync(0xFFFFFFFFu, up, t * 8 + 4);
        }
    }
}

// Accumulates P^T into the accumulators of one group of values: a = 16 values x 16 keys.  MASK: only the columns
// (query rows 2t, 2t+1 of a tile) in `own` take their part.
template <bool FP8, bool MASK>
__device__ __forceinline__ void value_mma(float (&o)[4], const uint32_t (&a)[4], const uint32_t (&ph)[2], const uint32_t (&pl)[2],
                                          const bool (&own)[2]) {
    if (!MASK) {
        if (FP8) {
            mma_f16(o, a, ph[0], ph[1]);
        } else {
            mma_bf16(o, a, ph[0], ph[1]);
            mma_bf16(o, a, pl[0], pl[1]);
        }
    } else {
        float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (FP8) {
            mma_f16(part, a, ph[0], ph[1]);
        } else {
            mma_bf16(part, a, ph[0], ph[1]);
            mma_bf16(part, a, pl[0], pl[1]);
        }
#pragma unroll
        for (int x = 0; x < 4; ++x)
            if (own[x & 1]) o[x] += part[x];
    }
}

// O^T += V^T P^T for one tile.  MASK: the values of this lane's keys (2t, 2t+1) and (2t+8, 2t+9) are masked by
// keep0, keep1, and only the columns in `own` are added to.
template <bool FP8, int NT, bool MASK>
__device__ __forceinline__ void value_product(uint32_t v_slot, int lane, const uint32_t (&ph)[NT][2], const uint32_t (&pl)[NT][2],
                                              float (&o)[NT][8][4], uint32_t keep0, uint32_t keep1, const bool (&own)[NT][2]) {
    const int mi = lane >> 3;
    if (!FP8) {
        const int key = (lane & 7) + ((mi >> 1) << 3);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            uint32_t a[4];
            ldmatrix4_trans(tile_addr<false>(v_slot, key, 2 * i + (mi & 1)), a);
            if (MASK) {
                a[0] &= keep0; a[1] &= keep0; a[2] &= keep1; a[3] &= keep1;
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) value_mma<FP8, MASK>(o[n][i], a, ph[n], pl[n], own[n]);
        }
    } else {
        const int key = (lane & 7) + ((mi & 1) << 3);
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            uint32_t x[4];
            ldmatrix4_trans(tile_addr<true>(v_slot, key, i + (mi >> 1)), x);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                // a pair of 16-bit units = (value 2g, 2g+1) of keys 2t and 2t+1: regroup by value
                const uint32_t lo = __byte_perm(x[2 * u], 0, 0x3120), hi = __byte_perm(x[2 * u + 1], 0, 0x3120);
                uint32_t a[4] = {e4m3x2_to_f16x2(lo), e4m3x2_to_f16x2(lo >> 16), e4m3x2_to_f16x2(hi), e4m3x2_to_f16x2(hi >> 16)};
                if (MASK) {
                    a[0] &= keep0; a[1] &= keep0; a[2] &= keep1; a[3] &= keep1;
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) value_mma<FP8, MASK>(o[n][i + u], a, ph[n], pl[n], own[n]);
            }
        }
    }
}

// The value index (0 .. 127) of accumulator o[.][i][2 * up] in lane row g.
template <bool FP8>
__device__ __forceinline__ int value_index(int i, int up, int g) {
    return FP8 ? 16 * i + 2 * g + up : 16 * i + 8 * up + g;
}

template <bool FP8, int NT>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) paged_attend_kernel(const __grid_constant__ AttendParams p) {
    constexpr int kStages = stages(FP8);
    constexpr int kRows = 8 * NT;
    extern __shared__ __align__(128) uint8_t paged_smem[];
    uint8_t* smem = paged_smem;
    __shared__ int s_warp_sum[kWarps];
    __shared__ int s_entry, s_unit;
    __shared__ int s_pos[kWarps][kStages];          // first position of the tile in a ring slot, -1: none
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int g = lane >> 2, t = lane & 3;
    const uint32_t ring = smem_u32(smem) + warp * (kRingBytes / kWarps);
    float* comb = reinterpret_cast<float*>(smem + kRingBytes);

#if __CUDA_ARCH__ >= 900
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
#endif

    // ---- this CTA's range of the line of units
    const int entries = p.B * p.Hkv * p.row_tiles;
    const int chunk = (entries + kThreads - 1) / kThreads;
    int mine = 0;
    for (int e = tid * chunk; e < min(entries, (tid + 1) * chunk); ++e) mine += entry_units(p, e);
    int incl = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int x = __shfl_up_sync(0xFFFFFFFFu, incl, d);
        if (lane >= d) incl += x;
    }
    if (lane == 31) s_warp_sum[warp] = incl;
    __syncthreads();
    int before = incl - mine, total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += s_warp_sum[w];
        total += s_warp_sum[w];
    }
    const int ctas = min((int)gridDim.x, total);
    if ((int)blockIdx.x >= ctas) {
        if (tid == 0) p.cut_entry[blockIdx.x] = -1;
        return;
    }
    const int begin = (int)((int64_t)total * blockIdx.x / ctas);
    int left = (int)((int64_t)total * (blockIdx.x + 1) / ctas) - begin;     // units to do, at least one
    if (begin >= before && begin < before + mine) {
        int e = tid * chunk, at = before;
        for (int n = entry_units(p, e); at + n <= begin; n = entry_units(p, e)) {
            at += n;
            ++e;
        }
        s_entry = e;
        s_unit = begin - at;
    }
    __syncthreads();

    Cursor ahead;                                   // the next tile to copy
    enter(p, ahead, s_entry);
    ahead.unit = s_unit;
    Cursor now = ahead;                             // the tile to compute
    if (tid == 0) p.cut_entry[blockIdx.x] = s_unit > 0 ? s_entry : -1;
    if (blockIdx.x == 0)                            // the row of the block table bounds a sequence: report a longer one
        for (int b = tid; b < p.B; b += kThreads)
            if (p.c.seq_lens[b] > ((int64_t)p.c.table_width << p.c.log2_page)) raise_status(p.c, kStatusTooLong);
    int to_copy = left;
    int pos_ahead = 0, page_ahead = locate(p, ahead, warp, pos_ahead);
    uint32_t slot_in = 0, slot_out = 0;             // ring slots, modulo kStages

    auto copy_next = [&]() {
        if (to_copy > 0) {
            if (lane == 0) s_pos[warp][slot_in] = page_ahead >= 0 ? pos_ahead : -1;
            if (page_ahead >= 0)
                load_tile<FP8>(p, ring + slot_in * (2 * tile_bytes(FP8)), page_ahead, ahead.h, pos_ahead, ahead.len, lane);
            if (--to_copy > 0) {
                if (++ahead.unit == ahead.units) {
                    enter(p, ahead, ahead.entry + 1);
                    ahead.unit = 0;
                }
                page_ahead = locate(p, ahead, warp, pos_ahead);   // used at the next step: its latency is hidden
            }
        }
        slot_in = slot_in + 1 == kStages ? 0 : slot_in + 1;
        cp_async_commit();
    };
    for (int s = 0; s < kStages - 1; ++s) copy_next();

    while (left > 0) {
        // ---- one entry, or the part of it that lies in this range
        const int row0 = (now.entry % p.row_tiles) * kRows;
        const int unit0 = now.unit;
        const int todo = min(left, now.units - now.unit);
        Queries<FP8, NT> qf;
        load_queries<FP8, NT>(p, now.b, now.h, row0, lane, qf);
        const float c0 = p.scale_log2 * (FP8 ? p.c.k_scale[now.h] : 1.0f);
        float o[NT][8][4], m[NT][2], l[NT][2];
        int limit[NT][2];                           // this lane's two rows of a tile see positions below it
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int x = 0; x < 4; ++x) o[n][i][x] = 0.0f;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                m[n][x] = -INFINITY;
                l[n][x] = 0.0f;
                limit[n][x] = now.len - p.nq + 1 + min(row0 + n * 8 + 2 * t + x, p.rows - 1) / p.Hg;
            }
        }
        const int all_see = now.len - p.nq + 1;     // every row sees the positions below it

        for (int step = 0; step < todo; ++step, ++now.unit) {
            cp_async_wait<kStages - 2>();
            __syncwarp();
            const int pos = s_pos[warp][slot_out];
            copy_next();                            // into the slot that the step before has read
            if (pos >= 0) {
                const uint32_t slot = ring + slot_out * (2 * tile_bytes(FP8));
                float s[NT][4];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int x = 0; x < 4; ++x) s[n][x] = 0.0f;
                if (!FP8) {
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks) {
                        uint32_t a[4];
                        ldmatrix4(tile_addr<false>(slot, lane & 15, 2 * ks + (lane >> 4)), a);
#pragma unroll
                        for (int n = 0; n < NT; ++n) mma_bf16(s[n], a, qf.f[n][ks][0], qf.f[n][ks][1]);
                    }
                } else {
#pragma unroll
                    for (int ks = 0; ks < 8; ks += 2) {
                        uint32_t x[4];
                        ldmatrix4(tile_addr<true>(slot, lane & 15, ks + (lane >> 4)), x);
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            uint32_t a[4] = {e4m3x2_to_f16x2(x[2 * u]), e4m3x2_to_f16x2(x[2 * u + 1]),
                                             e4m3x2_to_f16x2(x[2 * u] >> 16), e4m3x2_to_f16x2(x[2 * u + 1] >> 16)};
#pragma unroll
                            for (int n = 0; n < NT; ++n) mma_f16(s[n], a, qf.f[n][ks + u][0], qf.f[n][ks + u][1]);
                        }
                    }
                }
                // ---- softmax step: s[n] = keys (g, g, g+8, g+8) x rows (2t, 2t+1, 2t, 2t+1)
                const bool edge = pos + kTileKeys > all_see;
                uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const float scale = FP8 ? c0 * qf.unscale[n][x & 1] : c0;
                        s[n][x] *= scale;
                        if (edge && pos + g + (x >> 1) * 8 >= limit[n][x & 1]) s[n][x] = -INFINITY;
                    }
                    float corr[2];
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        float top = fmaxf(s[n][x], s[n][x + 2]);
                        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 4));
                        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 8));
                        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 16));
                        const float m_new = fmaxf(m[n][x], top);
                        const float ref = m_new == -INFINITY ? 0.0f : m_new;   // a row that has seen nothing yet
                        corr[x] = fast_exp2(m[n][x] - ref);
                        m[n][x] = m_new;
                        s[n][x] = fast_exp2(s[n][x] - ref);
                        s[n][x + 2] = fast_exp2(s[n][x + 2] - ref);
                        l[n][x] = l[n][x] * corr[x] + (s[n][x] + s[n][x + 2]);
                    }
                    if (corr[0] != 1.0f || corr[1] != 1.0f) {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
#pragma unroll
                            for (int x = 0; x < 4; ++x) o[n][i][x] *= corr[x & 1];
                    }
                    __syncwarp();
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const float a = s[n][2 * half], b = s[n][2 * half + 1];
                        if (FP8) {
                            ph[n][half] = movmatrix_trans(pack_f16x2(a, b));
                            pl[n][half] = 0;
                        } else {
                            // the upper 8 bits, and the rest -- a hair more of it, so that a probability above
                            // zero has two parts above zero and an infinite value stays infinite, not NaN
                            const uint32_t hi = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
                            const float more = 1.0f + 0x1p-23f;
                            ph[n][half] = movmatrix_trans(hi);
                            pl[n][half] = movmatrix_trans(pack_bf16x2(fmaf(a, more, -__uint_as_float(hi << 16)),
                                                                      fmaf(b, more, -__uint_as_float(hi & 0xFFFF0000u))));
                        }
                    }
                }
                const uint32_t v_slot = slot + tile_bytes(FP8);
                bool own[NT][2] = {};
                if (!edge || p.nq == 1) {
                    value_product<FP8, NT, false>(v_slot, lane, ph, pl, o, 0, 0, own);
                } else {
                    // Keys that only some of the rows may see: a masked probability of zero does not protect a
                    // row from an infinity or NaN in a value, so every new token gets a product of its own with
                    // the values behind its position cleared (one or two tiles of an entry).
                    const int j1 = (min(row0 + kRows, p.rows) - 1) / p.Hg;
#pragma unroll 1
                    for (int j = row0 / p.Hg; j <= j1; ++j) {
                        const int seen = all_see + j - pos;                     // keys of the tile this token sees
                        if (seen <= 0) continue;
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int x = 0; x < 2; ++x) own[n][x] = (row0 + n * 8 + 2 * t + x) / p.Hg == j;
                        const uint32_t k0 = (2 * t < seen ? 0xFFFFu : 0u) | (2 * t + 1 < seen ? 0xFFFF0000u : 0u);
                        const uint32_t k1 = (2 * t + 8 < seen ? 0xFFFFu : 0u) | (2 * t + 9 < seen ? 0xFFFF0000u : 0u);
                        value_product<FP8, NT, true>(v_slot, lane, ph, pl, o, k0, k1, own);
                    }
                }
            }
            __syncwarp();                           // the slot has been read
            slot_out = slot_out + 1 == kStages ? 0 : slot_out + 1;
        }
        left -= todo;

        // ---- add up the warps' states, eight rows at a time
        const bool whole = unit0 == 0 && now.unit == now.units;
        const int64_t part = ((int64_t)blockIdx.x * 2 + (unit0 > 0 ? 0 : 1)) * kRows;
        const float v_scale = FP8 ? p.c.v_scale[now.h] : 1.0f;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            if (row0 + n * 8 >= p.rows) break;
            float* mine_o = comb + warp * 8 * kCombStride;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                float sum = l[n][x];
                sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 4);
                sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 8);
                sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 16);
                if (g == 0) {
                    mine_o[(2 * t + x) * kCombStride + kD] = m[n][x];
                    mine_o[(2 * t + x) * kCombStride + kD + 1] = sum;
                }
#pragma unroll
                for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int up = 0; up < 2; ++up)
                        mine_o[(2 * t + x) * kCombStride + value_index<FP8>(i, up, g)] = o[n][i][2 * up + x];
            }
            __syncthreads();
#pragma unroll 1
            for (int rr = 0; rr < 8; ++rr) {
                const int r = row0 + n * 8 + rr;
                if (r >= p.rows) break;
                float top = -INFINITY;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) top = fmaxf(top, comb[(w * 8 + rr) * kCombStride + kD]);
                const float ref = top == -INFINITY ? 0.0f : top;
                float sum = 0.0f, acc = 0.0f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    const float* from = comb + (w * 8 + rr) * kCombStride;
                    const float f = fast_exp2(from[kD] - ref);
                    sum += f * from[kD + 1];
                    acc += f * from[tid];
                }
                if (whole) {
                    const int j = r / p.Hg, head = now.h * p.Hg + (r - j * p.Hg);
                    p.out[now.b * p.o_sb + j * p.o_sn + head * p.o_sh + tid] =
                        __float2bfloat16_rn(sum == 0.0f ? 0.0f : acc * v_scale / sum);
                    if (p.lse && tid == 0)
                        p.lse[((int64_t)now.b * p.nq + j) * p.H + head] =
                            sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
                } else {
                    p.part_o[(part + n * 8 + rr) * kD + tid] = acc;
                    if (tid == 0) p.part_ml[part + n * 8 + rr] = make_float2(top, sum);
                }
            }
            __syncthreads();
        }
        if (left > 0) {
            enter(p, now, now.entry + 1);
            now.unit = 0;
        }
    }
    cp_async_wait<0>();
}

// Adds up the parts of the entries that a cut of the line went through.  Block (c, r): if CTA c's range starts
// inside an entry and no earlier one's starts inside the same, row r of that entry is c - 1's part (which began
// it) and those of c, c + 1, ... as long as they start inside it.
constexpr int kJoinThreads = 256;

template <bool FP8>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const __grid_constant__ AttendParams p, int ctas, int tile_rows) {
    __shared__ float s_weight[512];
    __shared__ float s_red[kJoinThreads / 32];
    __shared__ float4 s_acc[kJoinThreads / 32][32];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int c = blockIdx.x + 1, rr = blockIdx.y;
#if __CUDA_ARCH__ >= 900
    asm volatile("griddepcontrol.wait;" ::: "memory");
#endif
    const int entry = p.cut_entry[c];
    if (entry < 0 || p.cut_entry[c - 1] == entry) return;
    const int row0 = (entry % p.row_tiles) * tile_rows;
    const int r = row0 + rr;
    if (r >= p.rows) return;
    int parts = 2;                                  // parts i = 0 .. parts - 1 come from CTAs c - 1 + i
    while (c + parts - 1 < ctas && p.cut_entry[c + parts - 1] == entry) ++parts;
    auto index = [&](int i) { return ((int64_t)(c - 1 + i) * 2 + (i == 0 ? 1 : 0)) * tile_rows + rr; };

    float top = -INFINITY;
    for (int i = tid; i < parts; i += kJoinThreads) top = fmaxf(top, p.part_ml[index(i)].x);
#pragma unroll
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
    if (lane == 0) s_red[warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kJoinThreads / 32; ++w) top = fmaxf(top, s_red[w]);
    __syncthreads();
    const float ref = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
    for (int i = tid; i < parts; i += kJoinThreads) {
        const float2 ml = p.part_ml[index(i)];
        const float f = fast_exp2(ml.x - ref);
        s_weight[i] = f;
        sum += f * ml.y;
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
    if (lane == 0) s_red[warp] = sum;
    __syncthreads();
    sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kJoinThreads / 32; ++w) sum += s_red[w];

    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int i = warp; i < parts; i += kJoinThreads / 32) {
        const float4 x = reinterpret_cast<const float4*>(p.part_o + index(i) * kD)[lane];
        const float f = s_weight[i];
        acc.x += f * x.x; acc.y += f * x.y; acc.z += f * x.z; acc.w += f * x.w;
    }
    s_acc[warp][lane] = acc;
    __syncthreads();
    if (tid < kD) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < kJoinThreads / 32; ++w) v += reinterpret_cast<const float*>(&s_acc[w][0])[tid];
        const int bh = entry / p.row_tiles, b = bh / p.Hkv, h = bh - b * p.Hkv;
        const int j = r / p.Hg, head = h * p.Hg + (r - j * p.Hg);
        const float v_scale = FP8 ? p.c.v_scale[h] : 1.0f;
        p.out[b * p.o_sb + j * p.o_sn + head * p.o_sh + tid] =
            __float2bfloat16_rn(sum == 0.0f ? 0.0f : v * v_scale / sum);
        if (p.lse && tid == 0)
            p.lse[((int64_t)b * p.nq + j) * p.H + head] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
    }
}

}  // namespace paged
}  // namespace aa
