// Attention of a few new tokens per sequence over a paged key-value cache.
//
//   out[r] = sum_p softmax_p(c q_r . k_p) v_p,   p <= len - new + token(r),
//
// for the rows r = (new token, query head of the KV head's group).  Every cached value meets as many
// multiply-adds as there are rows -- 4 operations a byte for a group of four and bf16 -- so the cache has to stream from
// HBM at full rate and everything else has to stay out of its way.
//
// Work split.  An entry is one (sequence, KV head, tile of up to 32 rows); its keys are cut into units.  All
// units of all entries form one line that is cut into as many equal ranges as there are CTAs, whatever the
// lengths: a batch of unequal sequences and a single long one fill the GPU alike.  Where a cut falls inside an
// entry, the CTAs on its sides leave (reference, sum, unnormalised row) and paged_join_kernel adds them
// up in the order of the keys.  Entries of a few units stay whole.  Where the cuts fall, and with them the order of the sums,
// depends on the lengths, the width of the table or lists and the number of SMs, never on timing.
//
// Inside a CTA a producer warp walks the units: it looks up their pages and has the TMA copy them (128-byte swizzle)
// into a ring of stages.  The keys of a unit go to lanes of RW warps, 16 to
// 64 keys a lane (see Shape); every lane keeps a softmax state of its own, and the states are added up where an entry ends.
// The RW warps of a lane own eight query rows each.  Everything but the arithmetic is the producer's: with the copies and
// page lookups in the computing warps (cp.async, a ring for every lane) an e4m3 tile took 467 warp instructions and
// the instruction rate was the limit, at 4.9 TB/s.
// Scores are computed transposed, S^T = K Q^T: the keys fill the 16 rows of the matrix instruction and 8 queries its
// columns, so a group of 4 wastes half of a tile of 8 instead of three quarters of one of 16; the
// probabilities then need one 8x8 transpose to become the operand of O^T = V^T P^T.  mma.sync is enough for one tile of rows:
// the tensor pipe is busy 16 % of the time with one tile (bf16), 38 % with three.  With several tiles each of them reads the keys
// and values from shared memory again.  The same transposed form on tcgen05.mma (keys, then head values, as its 128
// rows; one reading for all tiles) has not been tried.
//
// Measured (B200, whole calls, from the fastest to the slowest run on several GPUs): 32 sequences of up to 32768 tokens, 32/8
// heads: bf16 357 to 369 us, 6.6 to 6.8 TB/s; e4m3 188 to 206 us, 5.9 to 6.4 TB/s;
// one sequence of 131072 tokens 87.5 to 89.2 us, 6.0 to 6.1 TB/s; 16 of up to 4001 tokens 21 to 23 us, where the bytes alone
// take 10; five new tokens for 8 sequences of up to 16001 75 to 82 us, bound by latencies inside a tile.
// That every warp reports a wait that gave up, and the producer sees its copies land, costs 0.5 to 2 % with e4m3 pages (one token
// 41.0 and 41.4 us, three 55.5 and 56.5, those 8 sequences), nothing with bf16; the lift of the e4m3 probabilities (see Accuracy)
// costs nothing.  Registers: 162 to 168, 128 with three row tiles; the e4m3
// forms of two and four row tiles spill 12 bytes, that of three 68.
// Without the join kernel (its results then incomplete) calls take 2 us less on the GPU for one short sequence, 3 to 5 us
// for most, 8 us for the five new tokens.
//
// Accuracy.  Scores, softmax state and outputs are held in 32 bits.  With bf16 pages a probability goes into
// the second product as the sum of two bf16 values (15 bits), so that only the output is rounded to 8;
// the extra instructions hide behind the loads.  With e4m3 pages both products run in f16, in which every
// code is exact; queries are scaled by a power of two per row to fit f16.  A lane's probabilities are held relative to 2^15 at
// its largest, so that f16 keeps 11 bits of those down to 2^-29 of it and loses none above 2^-40; the sum of the
// denominator is of the values before that rounding.
#pragma once
#include "paged_common.cuh"
#include "tc_ptx.cuh"

namespace aa {
namespace paged {

constexpr int kTileKeys = 16;                       // keys of one matrix instruction
constexpr int kCombStride = 132;                    // floats; 132 keeps the transposed writes off each other's banks
constexpr int kCombRows = 32;                       // rows of partial results a round of adding up holds
constexpr int kCombBytes = kCombRows * kCombStride * 4;
constexpr int kRingBytes = 96 * 1024;               // with the join buffer, two CTAs fill an SM's shared memory
constexpr int kCtasPerSm = 2;
constexpr int kSegments = 16;                       // entries of a CTA's range whose lengths are kept at hand
constexpr int kMiscBytes = 512;
constexpr int kSmemBytes = kRingBytes + kCombBytes + kMiscBytes;

// The warps of a CTA (and one more, the producer) and the stages of its ring.  Four computing warps where it can be: two CTAs
// then have ten warps, three of them on one quarter of the SM, which leaves each thread 168 registers, and a warp that takes two
// or four tiles of 16 keys a step has enough of its own to hide its latencies.  Measured, each pair in one run, at 32 sequences of up to 32768 tokens, e4m3, a group of 4: 8 lanes of one tile 196 us, 4 of
// two 188 us; eight sequences of up to 16001 tokens, bf16: 20 rows 85 us with one tile, 74 us with two, 32 rows 99 us with 2 lanes
// of two tiles, 87 us with one of four, 12 rows 76 us with 4 lanes of one, 66 us with 2 of two; e4m3, 12 rows: 63 and 53 us.
template <bool FP8, int RW>
struct Shape {
    static constexpr int kLanes = RW == 1 ? 4 : RW < 4 ? 2 : 1;
    static constexpr int kDepth = RW == 1 ? (FP8 ? 2 : 1) : FP8 || RW == 4 ? 4 : 2;     // tiles of a lane and step
    static constexpr int kTiles = kLanes * kDepth;                                      // of a unit
    static constexpr int kWarps = kLanes * RW;
    static constexpr int kThreads = (kWarps + 1) * 32;
    static constexpr int kUnitKeys = kTiles * kTileKeys;
    static constexpr int kParts = FP8 ? 2 : 4;                       // of 128 bytes a key: keys, values, or halves of them
    static constexpr int kPartBytes = kUnitKeys * 128;
    static constexpr int kUnitBytes = kParts * kPartBytes;
    static constexpr int kStages = kRingBytes / kUnitBytes < 8 ? kRingBytes / kUnitBytes : 8;
    static constexpr int kRows = 8 * RW;
    static constexpr int kRoundRows = kCombRows / kLanes < kRows ? kCombRows / kLanes : kRows;   // rows added up at a time
};

// How the coordinates of a copy are ordered in a pool's tensor map (dimension 0 is the row of 128 values).
struct MapOrder {
    int row, head, page;                            // 0 .. 2
};

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
    int rows, row_tiles;                            // rows = nq * Hg, in tiles of 8 * RW
    float scale_log2;                               // softmax scale times log2 e
    bool whole;                                     // ranges end where entries do: nothing is cut
    float* part_o;                                  // [ctas, 2, 8 RW, 128]
    float2* part_ml;                                // [ctas, 2, 8 RW]
    int2* cuts;                                     // [ctas]: (entry, parts) where a CTA's range is the first to start
                                                    // inside that entry, which the CTA before it began and `parts` CTAs
                                                    // share; else (-1, 0)
    MapOrder k_order, v_order;
    int log2_box;                                   // keys of one copy: the smaller of page and unit
    uint32_t wait_polls;                            // after which a computing warp gives up on a copy
};

// Keys an entry streams over (list entries count as whole pages) and the units they make; an empty one still
// makes a unit, so that some CTA writes its zeros.
__device__ __forceinline__ int entry_units(const AttendParams& p, int e, int unit_keys) {
    const int bh = e / p.row_tiles;
    int64_t keys;
    if (p.pages) {
        keys = (int64_t)min(max(p.page_counts[bh], 0), p.list_width) << p.c.log2_page;
    } else {
        keys = seq_len(p.c, bh / p.Hkv);
    }
    return max(1, (int)((keys + unit_keys - 1) / unit_keys));
}

// One lane's place in the line of units.
struct Cursor {
    int entry, unit, units;                         // unit: next one of the entry
    int b, h, len;
};

__device__ __forceinline__ void enter(const AttendParams& p, Cursor& c, int entry, int unit_keys, const int2* segments, int first_entry) {
    c.entry = entry;
    const int bh = entry / p.row_tiles;
    c.b = bh / p.Hkv;
    c.h = bh - c.b * p.Hkv;
    if (entry - first_entry < kSegments) {
        c.units = segments[entry - first_entry].x;
        c.len = segments[entry - first_entry].y;
    } else {
        c.units = entry_units(p, entry, unit_keys);
        c.len = seq_len(p.c, c.b);
    }
}

// Where the 16 keys of a tile of the cursor's unit are: the pool page, or -1 for none; `pos` their first position.
__device__ __forceinline__ int locate(const AttendParams& p, const Cursor& c, int tiles, int tile, int& pos) {
    const int64_t flat = ((int64_t)c.unit * tiles + tile) * kTileKeys;
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

// A 16-byte chunk of a lane's row (0 .. 15) in its part of a stage: the TMA's 128-byte swizzle, and for bf16 the second
// half of a row's 256 bytes in the next part.
template <bool FP8, int RW>
__device__ __forceinline__ uint32_t tile_addr(uint32_t base, int row, int chunk) {
    return base + (FP8 ? 0 : (chunk >> 3) * Shape<FP8, RW>::kPartBytes) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4);
}

// Eight query rows of an entry as operands of S^T = K Q^T.  Lane (g, t) holds row g: the values that meet its K values
// in step s.
struct Queries {
    uint32_t f[8][2];
    float unscale[2];                               // of this lane's score columns 2t, 2t + 1 (e4m3 only)
};

template <bool FP8>
__device__ __forceinline__ void fetch_queries(const AttendParams& p, const Cursor& c, int row0, int lane, Queries& qf) {
    const int g = lane >> 2, t = lane & 3;
    const int r = row0 + g;
    const bool in = r < p.rows;
    const int j = in ? r / p.Hg : 0, i = in ? r - j * p.Hg : 0;
    const uint32_t* src =
        reinterpret_cast<const uint32_t*>(p.q + c.b * p.q_sb + j * p.q_sn + (int64_t)(c.h * p.Hg + i) * p.q_sh);
#pragma unroll
    for (int s = 0; s < 8; ++s) {
        const int at = FP8 ? s * 8 + t * 2 : s * 8 + t;              // in pairs of values
        qf.f[s][0] = in ? src[at] : 0u;
        qf.f[s][1] = in ? src[at + (FP8 ? 1 : 4)] : 0u;
    }
}

// bf16 -> f16, scaled by a power of two so that a row's largest value lies in [256, 512): f16 then keeps 2^-32 of it.
__device__ __forceinline__ void queries_to_f16(int lane, Queries& qf) {
    uint32_t big = 0;                               // largest |q| of the row, as bf16 bits
#pragma unroll
    for (int s = 0; s < 8; ++s)
#pragma unroll
        for (int w = 0; w < 2; ++w) big = max(big, max(qf.f[s][w] & 0x7FFFu, (qf.f[s][w] >> 16) & 0x7FFFu));
    big = max(big, __shfl_xor_sync(0xFFFFFFFFu, big, 1));
    big = max(big, __shfl_xor_sync(0xFFFFFFFFu, big, 2));
    const int expo = max(min((int)(big >> 7), 254) - 127 - 8, -126);
    const float down = __uint_as_float((uint32_t)(127 - expo) << 23);
    const float up = __uint_as_float((uint32_t)(127 + expo) << 23);
#pragma unroll
    for (int s = 0; s < 8; ++s)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const uint32_t x = qf.f[s][w];
            qf.f[s][w] = pack_f16x2(__uint_as_float(x << 16) * down, __uint_as_float(x & 0xFFFF0000u) * down);
        }
    qf.unscale[0] = __shfl_sync(0xFFFFFFFFu, up, (lane & 3) * 8);
    qf.unscale[1] = __shfl_sync(0xFFFFFFFFu, up, (lane & 3) * 8 + 4);
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
template <bool FP8, int RW, bool MASK>
__device__ __forceinline__ void value_product(uint32_t v_slot, int lane, const uint32_t (&ph)[2], const uint32_t (&pl)[2],
                                              float (&o)[8][4], uint32_t keep0, uint32_t keep1, const bool (&own)[2]) {
    const int mi = lane >> 3;
    if (!FP8) {
        const int key = (lane & 7) + ((mi >> 1) << 3);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            uint32_t a[4];
            ldmatrix4_trans(tile_addr<false, RW>(v_slot, key, 2 * i + (mi & 1)), a);
            if (MASK) {
                a[0] &= keep0; a[1] &= keep0; a[2] &= keep1; a[3] &= keep1;
            }
            value_mma<FP8, MASK>(o[i], a, ph, pl, own);
        }
    } else {
        const int key = (lane & 7) + ((mi & 1) << 3);
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            uint32_t x[4];
            ldmatrix4_trans(tile_addr<true, RW>(v_slot, key, i + (mi >> 1)), x);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                // a pair of 16-bit units = (value 2g, 2g+1) of keys 2t and 2t+1: regroup by value
                const uint32_t lo = __byte_perm(x[2 * u], 0, 0x3120), hi = __byte_perm(x[2 * u + 1], 0, 0x3120);
                uint32_t a[4] = {e4m3x2_to_f16x2(lo), e4m3x2_to_f16x2(lo >> 16), e4m3x2_to_f16x2(hi), e4m3x2_to_f16x2(hi >> 16)};
                if (MASK) {
                    a[0] &= keep0; a[1] &= keep0; a[2] &= keep1; a[3] &= keep1;
                }
                value_mma<FP8, MASK>(o[i + u], a, ph, pl, own);
            }
        }
    }
}

// A finished row, four values a thread; a row that has seen nothing is 0.
__device__ __forceinline__ void store_row(__nv_bfloat16* to, int lane, const float4& acc, float sum, float v_scale) {
    const float f = sum == 0.0f ? 0.0f : v_scale / sum;
    const bool none = sum == 0.0f;
    reinterpret_cast<uint2*>(to)[lane] = make_uint2(pack_bf16x2(none ? 0.0f : acc.x * f, none ? 0.0f : acc.y * f),
                                                    pack_bf16x2(none ? 0.0f : acc.z * f, none ? 0.0f : acc.w * f));
}
// The natural logarithm of a softmax sum from its reference (log2 units) and the sum behind it.
__device__ __forceinline__ float log_sum(float top, float sum) {
    return sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
}

// The value index (0 .. 127) of accumulator o[.][i][2 * up] in lane row g.
template <bool FP8>
__device__ __forceinline__ int value_index(int i, int up, int g) {
    return FP8 ? 16 * i + 2 * g + up : 16 * i + 8 * up + g;
}

template <bool FP8, int RW>
__global__ void __launch_bounds__(Shape<FP8, RW>::kThreads, kCtasPerSm)
    paged_attend_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                        const __grid_constant__ AttendParams p) {
    using S = Shape<FP8, RW>;
    constexpr int kStages = S::kStages, kDepth = S::kDepth;
    // A state (m, l, o) stands for 2^m l and 2^m o; with e4m3 pages m is the running maximum less this, rounded up: a probability is
    // at most 2^15 in f16 for scores of any size (from 2^24 on, a difference rounded to nearest could be 16).
    constexpr float kLift = 15.0f;
    extern __shared__ __align__(1024) uint8_t paged_attend_smem[];
    float* comb = reinterpret_cast<float*>(paged_attend_smem + kRingBytes);
    // the last 512 bytes: barriers, lengths of this range's entries, tile positions of the stages, scratch of the start
    const uint32_t ring = smem_u32(paged_attend_smem);
    const uint32_t bars = ring + kRingBytes + kCombBytes;
    auto full = [&](uint32_t stage) { return bars + 8u * stage; };
    auto empty = [&](uint32_t stage) { return bars + 8u * (kStages + stage); };
    int2* segments = reinterpret_cast<int2*>(paged_attend_smem + kRingBytes + kCombBytes + 16 * kStages);
    int* s_pos = reinterpret_cast<int*>(segments + kSegments);                    // [stages][tiles], -1: no keys
    int* s_sum = s_pos + S::kTiles * kStages;                                     // [warps], then (entry, unit)
    volatile int* abort_flag = s_sum + S::kWarps + 3;
    static_assert(16 * kStages + kSegments * 8 + (S::kTiles * kStages + S::kWarps + 4) * 4 <= kMiscBytes, "the last 512 bytes");
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    start_next_kernel();
    if (tid == 0) {
        for (int i = 0; i < kStages; ++i) {
            tc::mbar_init(full(i), 1);
            tc::mbar_init(empty(i), S::kWarps);
        }
        *abort_flag = 0;
        tc::fence_mbar_init();
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&k_map)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&v_map)) : "memory");
    }
    wait_for_kernels_before();

    // ---- this CTA's range of the line of units
    const int entries = p.B * p.Hkv * p.row_tiles;
    const int chunk = (entries + S::kThreads - 1) / S::kThreads;
    const int my_first = tid * chunk, my_end = min(entries, my_first + chunk);
    int mine = 0;
    if (p.whole) {                                  // the line of entries is cut instead
        mine = max(0, my_end - my_first);
    } else {
        for (int e = my_first; e < my_end; ++e) mine += entry_units(p, e, S::kUnitKeys);
    }
    int incl = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int x = __shfl_up_sync(0xFFFFFFFFu, incl, d);
        if (lane >= d) incl += x;
    }
    if (lane == 31) s_sum[warp] = incl;
    __syncthreads();
    int before = incl - mine, total = 0;
#pragma unroll
    for (int w = 0; w < S::kWarps + 1; ++w) {
        if (w < warp) before += s_sum[w];
        total += s_sum[w];
    }
    const int ctas = min((int)gridDim.x, total);
    if ((int)blockIdx.x >= ctas) {
        if (tid == 0 && !p.whole) p.cuts[blockIdx.x] = make_int2(-1, 0);
        return;
    }
    // CTA c owns the units [total c / ctas, total (c + 1) / ctas), in 32-bit arithmetic (ctas is at most 512)
    const int whole_part = total / ctas, rest = total - whole_part * ctas;
    auto range_start = [&](int c) { return whole_part * c + rest * c / ctas; };
    const int begin = range_start(blockIdx.x), end = range_start(blockIdx.x + 1);
    if (begin >= before && begin < before + mine) {
        int e = my_first, at = before;
        if (p.whole) {
            e += begin - before;
            at = begin;
        } else {
            for (int n = entry_units(p, e, S::kUnitKeys); at + n <= begin; n = entry_units(p, e, S::kUnitKeys)) {
                at += n;
                ++e;
            }
        }
        s_sum[S::kWarps + 1] = e;
        s_sum[S::kWarps + 2] = begin - at;
    }
    __syncthreads();
    const int first_entry = s_sum[S::kWarps + 1], first_unit = s_sum[S::kWarps + 2];
    if (before < end && before + mine > begin) {
        int at = before;
        for (int e = my_first; e < my_end && at < end && e - first_entry < kSegments; ++e) {
            const int n = chunk == 1 && !p.whole ? mine : entry_units(p, e, S::kUnitKeys);
            if (e >= first_entry) segments[e - first_entry] = make_int2(n, seq_len(p.c, e / p.row_tiles / p.Hkv));
            at += p.whole ? 1 : n;
        }
    }
    if (blockIdx.x == 0)                            // the row of the block table bounds a sequence: report a longer one
        for (int b = tid; b < p.B; b += S::kThreads)
            if (p.c.seq_lens[b] > ((int64_t)p.c.table_width << p.c.log2_page)) raise_status(p.c, kStatusTooLong);
    __syncthreads();

    int left = end - begin;                         // units to do, at least one
    if (p.whole) {
        left = 0;
        for (int e = begin; e < end; ++e) left += e - begin < kSegments ? segments[e - begin].x : entry_units(p, e, S::kUnitKeys);
    }
    Cursor now;
    enter(p, now, first_entry, S::kUnitKeys, segments, first_entry);
    now.unit = first_unit;
    if (tid == 0 && !p.whole) {
        const int starts = begin - first_unit;
        int2 cut = make_int2(-1, 0);
        if (first_unit > 0 && range_start(blockIdx.x - 1) <= starts) {
            // unit u belongs to CTA ((u + 1) ctas - 1) / total: 40 bits by 31, exact in double precision
            const int last = (int)(((double)(starts + now.units) * ctas - 1.0) / total);
            cut = make_int2(first_entry, last - (int)blockIdx.x + 2);
        }
        p.cuts[blockIdx.x] = cut;
    }

    if (warp == S::kWarps) {
        // ================================================== producer
        // lane i < kTiles looks up tile i of the unit; lane 8 * part + box issues a copy
        const int boxes = S::kUnitKeys >> p.log2_box, box_bytes = 128 << p.log2_box;
        const int box = lane & 7, part = lane >> 3;
        const bool issues = part < S::kParts && box < boxes;
        const bool of_values = part >= S::kParts / 2;
        const CUtensorMap* map = of_values ? &v_map : &k_map;
        const MapOrder order = of_values ? p.v_order : p.k_order;
        const int x = FP8 ? 0 : (part & 1) * 64;
        const uint32_t box_at = part * S::kPartBytes + box * box_bytes;
        int pos = 0, page = lane < S::kTiles ? locate(p, now, S::kTiles, lane, pos) : -1;
        uint32_t stage = 0, parity = 1;             // of the stage's previous use: the first pass waits for nothing
        int issued = 0;
        for (int i = 0; i < left; ++i) {
            // One answer for the warp, whose lanes exchange pages below.  A computing warp that gives up raises the flag before
            // it hands the stage back, so a stage whose copy may still be in flight is not filled again.
            const bool may_fill = tc::mbar_wait(empty(stage), parity, abort_flag) && !*abort_flag;
            if (!__all_sync(0xFFFFFFFFu, may_fill)) break;
            const int first_tile = (box << p.log2_box) / kTileKeys;
            const int box_page = __shfl_sync(0xFFFFFFFFu, page, first_tile & 31);
            const int box_pos = __shfl_sync(0xFFFFFFFFu, pos, first_tile & 31);
            const bool issue = issues && box_page >= 0;
            const uint32_t bytes = __popc(__ballot_sync(0xFFFFFFFFu, issue)) * box_bytes;
            if (lane < S::kTiles) s_pos[stage * S::kTiles + lane] = page >= 0 ? pos : -1;
            __syncwarp();
            if (lane == 0) tc::mbar_arrive_expect_tx(full(stage), bytes);
            __syncwarp();
            if (issue) {
                const int row = box_pos & ((1 << p.c.log2_page) - 1);
                int at[3];
#pragma unroll
                for (int d = 0; d < 3; ++d) at[d] = order.row == d ? row : order.head == d ? now.h : box_page;
                tc::tma_load_4d(ring + stage * S::kUnitBytes + box_at, map, full(stage), x, at[0], at[1], at[2]);
            }
            issued = i + 1;
            if (i + 1 < left) {
                if (++now.unit == now.units) {
                    enter(p, now, now.entry + 1, S::kUnitKeys, segments, first_entry);
                    now.unit = 0;
                }
                page = lane < S::kTiles ? locate(p, now, S::kTiles, lane, pos) : -1;   // used after the next wait
            }
            if (++stage == kStages) {
                stage = 0;
                parity ^= 1;
            }
        }
        // The block's shared memory is not handed on before the last copies have landed: a computing warp that gives up on
        // one of them does not wait for it.
        bool all_landed = true;
        for (int i = max(issued - kStages, 0); i < issued; ++i)
            all_landed = tc::mbar_drain(full(i % kStages), (i / kStages) & 1) && all_landed;
        if (issued < left || !all_landed) raise_status(p.c, kStatusTimeout);
        return;
    }

    // ====================================================== the computing warps
    const int g = lane >> 2, t = lane & 3;
    const int kl = warp / RW, rw = warp % RW;       // key lane; which eight rows
    auto compute_sync = [] { asm volatile("bar.sync 1, %0;" ::"n"(S::kWarps * 32) : "memory"); };
    uint32_t stage = 0, parity = 0;
    Queries qf;
    fetch_queries<FP8>(p, now, now.entry % p.row_tiles * S::kRows + rw * 8, lane, qf);

    while (left > 0) {
        // ---- one entry, or the part of it that lies in this range
        const int row_base = now.entry % p.row_tiles * S::kRows;
        const int row0 = row_base + rw * 8;         // this warp's rows
        const int unit0 = now.unit;
        const int todo = min(left, now.units - now.unit);
        if (FP8) queries_to_f16(lane, qf);
        const float c0 = p.scale_log2 * (FP8 ? p.c.k_scale[now.h] : 1.0f);
        const float scale[2] = {FP8 ? c0 * qf.unscale[0] : c0, FP8 ? c0 * qf.unscale[1] : c0};
        float o[8][4], m[2], l[2];
        int limit[2];                               // this lane's two rows see positions below it
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int x = 0; x < 4; ++x) o[i][x] = 0.0f;
        const int all_see = now.len - p.nq + 1;     // every row sees the positions below it
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            m[x] = -INFINITY;
            l[x] = 0.0f;
            limit[x] = all_see + min(row0 + 2 * t + x, p.rows - 1) / p.Hg;
        }

        for (int step = 0; step < todo; ++step) {
            const uint32_t free_bar = empty(stage);
            const bool landed = tc::mbar_wait(full(stage), parity, abort_flag, p.wait_polls);
            int pos[kDepth];
            bool any = false;
#pragma unroll
            for (int j = 0; j < kDepth; ++j) {
                pos[j] = landed ? s_pos[stage * S::kTiles + kl * kDepth + j] : -1;
                any = any || pos[j] >= 0;
            }
            const uint32_t slot0 = ring + stage * S::kUnitBytes + kl * kDepth * (kTileKeys * 128);
            if (++stage == kStages) {
                stage = 0;
                parity ^= 1;
            }
            if (!__all_sync(0xFFFFFFFFu, any)) {
                __syncwarp();                       // a raised flag is visible before the stage is handed back
                if (lane == 0) tc::mbar_arrive(free_bar);
                continue;
            }
            // ---- scores, in two sums a tile: s = keys (g, g, g+8, g+8) x rows (2t, 2t+1, 2t, 2t+1)
            float s[kDepth][4];
            bool edge = false;                      // some row does not see all keys
#pragma unroll
            for (int j = 0; j < kDepth; ++j) {
                const uint32_t slot = slot0 + j * (kTileKeys * 128);
                float s1[4] = {0.0f, 0.0f, 0.0f, 0.0f}, s2[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                if (!FP8) {
#pragma unroll
                    for (int ks = 0; ks < 8; ks += 2) {
                        uint32_t a[4], a2[4];
                        ldmatrix4(tile_addr<false, RW>(slot, lane & 15, 2 * ks + (lane >> 4)), a);
                        ldmatrix4(tile_addr<false, RW>(slot, lane & 15, 2 * ks + 2 + (lane >> 4)), a2);
                        mma_bf16(s1, a, qf.f[ks][0], qf.f[ks][1]);
                        mma_bf16(s2, a2, qf.f[ks + 1][0], qf.f[ks + 1][1]);
                    }
                } else {
#pragma unroll
                    for (int ks = 0; ks < 8; ks += 2) {
                        uint32_t x[4];
                        ldmatrix4(tile_addr<true, RW>(slot, lane & 15, ks + (lane >> 4)), x);
                        const uint32_t a[4] = {e4m3x2_to_f16x2(x[0]), e4m3x2_to_f16x2(x[1]), e4m3x2_to_f16x2(x[0] >> 16),
                                               e4m3x2_to_f16x2(x[1] >> 16)};
                        const uint32_t a2[4] = {e4m3x2_to_f16x2(x[2]), e4m3x2_to_f16x2(x[3]), e4m3x2_to_f16x2(x[2] >> 16),
                                                e4m3x2_to_f16x2(x[3] >> 16)};
                        mma_f16(s1, a, qf.f[ks][0], qf.f[ks][1]);
                        mma_f16(s2, a2, qf.f[ks + 1][0], qf.f[ks + 1][1]);
                    }
                }
                const bool cut_off = pos[j] < 0 || pos[j] + kTileKeys > all_see;
                edge = edge || cut_off;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    s[j][x] = (s1[x] + s2[x]) * scale[x & 1];
                    if (cut_off && (pos[j] < 0 || pos[j] + g + (x >> 1) * 8 >= limit[x & 1])) s[j][x] = -INFINITY;
                }
            }
            // ---- softmax step
            float corr[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                float top = fmaxf(s[0][x], s[0][x + 2]);
#pragma unroll
                for (int j = 1; j < kDepth; ++j) top = fmaxf(top, fmaxf(s[j][x], s[j][x + 2]));
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 4));
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 8));
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 16));
                const float m_new = fmaxf(m[x], FP8 ? __fadd_ru(top, -kLift) : top);
                const float ref = m_new == -INFINITY ? 0.0f : m_new;       // a row that has seen nothing yet
                corr[x] = fast_exp2(m[x] - ref);
                m[x] = m_new;
                float more = 0.0f;
#pragma unroll
                for (int j = 0; j < kDepth; ++j) {
                    s[j][x] = fast_exp2(s[j][x] - ref);
                    s[j][x + 2] = fast_exp2(s[j][x + 2] - ref);
                    more += s[j][x] + s[j][x + 2];
                }
                l[x] = l[x] * corr[x] + more;
            }
            if (__any_sync(0xFFFFFFFFu, corr[0] != 1.0f || corr[1] != 1.0f)) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int x = 0; x < 4; ++x) o[i][x] *= corr[x & 1];
            }
#pragma unroll
            for (int j = 0; j < kDepth; ++j) {
                uint32_t ph[2], pl[2];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const float a = s[j][2 * half], b = s[j][2 * half + 1];
                    if (FP8) {
                        ph[half] = movmatrix_trans(pack_f16x2(a, b));
                        pl[half] = 0;
                    } else {
                        // the upper 8 bits, and the rest -- a hair more of it, so that a probability above
                        // zero has two parts above zero and an infinite value stays infinite, not NaN
                        const uint32_t hi = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
                        const float more = 1.0f + 0x1p-23f;
                        ph[half] = movmatrix_trans(hi);
                        pl[half] = movmatrix_trans(pack_bf16x2(fmaf(a, more, -__uint_as_float(hi << 16)),
                                                               fmaf(b, more, -__uint_as_float(hi & 0xFFFF0000u))));
                    }
                }
                const uint32_t v_slot = slot0 + j * (kTileKeys * 128) + S::kUnitBytes / 2;
                bool own[2] = {false, false};
                if (!edge) {
                    value_product<FP8, RW, false>(v_slot, lane, ph, pl, o, 0, 0, own);
                } else if (pos[j] >= 0) {
                    // Keys behind the end, or that only some of the rows may see: a masked probability of zero does not
                    // protect a row from an infinity or NaN in a value, so every new token gets a product of its own
                    // with the values behind its position cleared (one or two tiles of an entry).
                    const int j1 = (min(row0 + 8, p.rows) - 1) / p.Hg;
#pragma unroll 1
                    for (int token = row0 / p.Hg; token <= j1; ++token) {
                        const int seen = all_see + token - pos[j];              // keys of the tile this token sees
                        if (seen <= 0) continue;
#pragma unroll
                        for (int x = 0; x < 2; ++x) own[x] = (row0 + 2 * t + x) / p.Hg == token;
                        const uint32_t k0 = (2 * t < seen ? 0xFFFFu : 0u) | (2 * t + 1 < seen ? 0xFFFF0000u : 0u);
                        const uint32_t k1 = (2 * t + 8 < seen ? 0xFFFFu : 0u) | (2 * t + 9 < seen ? 0xFFFF0000u : 0u);
                        value_product<FP8, RW, true>(v_slot, lane, ph, pl, o, k0, k1, own);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(free_bar);
        }
        left -= todo;
        now.unit += todo;

        // ---- add up the lanes' states, kRoundRows rows at a time; a warp takes a row, a thread four values
        const bool whole = unit0 == 0 && now.unit == now.units;
        const int64_t part = ((int64_t)blockIdx.x * 2 + (unit0 > 0 ? 0 : 1)) * S::kRows;
        const float v_scale = FP8 ? p.c.v_scale[now.h] : 1.0f;
        const int b_done = now.b, h_done = now.h;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            l[x] += __shfl_xor_sync(0xFFFFFFFFu, l[x], 4);
            l[x] += __shfl_xor_sync(0xFFFFFFFFu, l[x], 8);
            l[x] += __shfl_xor_sync(0xFFFFFFFFu, l[x], 16);
        }
        if (left > 0) {                             // the next entry's queries arrive meanwhile
            enter(p, now, now.entry + 1, S::kUnitKeys, segments, first_entry);
            now.unit = 0;
            fetch_queries<FP8>(p, now, now.entry % p.row_tiles * S::kRows + rw * 8, lane, qf);
        }
        for (int base = 0; base < S::kRows && row_base + base < p.rows; base += S::kRoundRows) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int at = rw * 8 + 2 * t + x - base;
                if (at >= 0 && at < S::kRoundRows) {
                    float* to = comb + (kl * S::kRoundRows + at) * kCombStride;
                    if (g == 0) {
                        to[kD] = m[x];
                        to[kD + 1] = l[x];
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i)
#pragma unroll
                        for (int up = 0; up < 2; ++up) to[value_index<FP8>(i, up, g)] = o[i][2 * up + x];
                }
            }
            compute_sync();
            for (int rr = warp; rr < min(S::kRoundRows, S::kRows - base); rr += S::kWarps) {
                const int r = row_base + base + rr;
                if (r >= p.rows) break;
                float top = -INFINITY, weight[S::kLanes];
#pragma unroll
                for (int w = 0; w < S::kLanes; ++w) {
                    weight[w] = comb[(w * S::kRoundRows + rr) * kCombStride + kD];
                    top = fmaxf(top, weight[w]);
                }
                const float ref = top == -INFINITY ? 0.0f : top;
                float sum = 0.0f;
                float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < S::kLanes; ++w) {
                    const float* from = comb + (w * S::kRoundRows + rr) * kCombStride;
                    const float f = fast_exp2(weight[w] - ref);
                    const float4 x = reinterpret_cast<const float4*>(from)[lane];
                    sum += f * from[kD + 1];
                    acc.x += f * x.x; acc.y += f * x.y; acc.z += f * x.z; acc.w += f * x.w;
                }
                if (whole) {
                    const int j = r / p.Hg, head = h_done * p.Hg + (r - j * p.Hg);
                    store_row(p.out + b_done * p.o_sb + j * p.o_sn + head * p.o_sh, lane, acc, sum, v_scale);
                    if (p.lse && lane == 0) p.lse[((int64_t)b_done * p.nq + j) * p.H + head] = log_sum(top, sum);
                } else {
                    reinterpret_cast<float4*>(p.part_o + (part + base + rr) * kD)[lane] = acc;
                    if (lane == 0) p.part_ml[part + base + rr] = make_float2(top, sum);
                }
            }
            compute_sync();
        }
    }
    // A wait of this block gave up, and some keys are missing above.  A warp whose own wait did sees its flag here, whether or not
    // the producer is still there to report it.
    if (*abort_flag) raise_status(p.c, kStatusTimeout);
}

// Adds up the parts of the entries that a cut of the line went through.  Block (c - 1, r) takes row r of the entry that CTA
// c leads (see `cuts`): CTA c - 1 began it, c, c + 1, ... start inside it.
constexpr int kJoinThreads = 128;

template <bool FP8>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const __grid_constant__ AttendParams p, int tile_rows) {
    constexpr int kWarps = kJoinThreads / 32, kAhead = 4;
    __shared__ float s_sum[kWarps];
    __shared__ float4 s_acc[kWarps][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int c = blockIdx.x + 1, rr = blockIdx.y;
    start_next_kernel();
    wait_for_kernels_before();
    const int2 cut = p.cuts[c];
    const int entry = cut.x, parts = cut.y;         // parts i = 0 .. parts - 1 come from CTAs c - 1 + i
    if (entry < 0) return;
    const int row0 = (entry % p.row_tiles) * tile_rows;
    const int r = row0 + rr;
    if (r >= p.rows) return;
    auto index = [&](int i) { return ((int64_t)(c - 1 + i) * 2 + (i == 0 ? 1 : 0)) * tile_rows + rr; };

    // warp w takes parts w, w + 4, ...; the first are on their way while every warp finds the maximum of all
    float4 x[kAhead];
    float2 ml[kAhead];
    auto fetch = [&](int i0) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (i0 + u * kWarps < parts) {
                ml[u] = p.part_ml[index(i0 + u * kWarps)];
                x[u] = reinterpret_cast<const float4*>(p.part_o + index(i0 + u * kWarps) * kD)[lane];
            }
    };
    fetch(warp);
    float top = -INFINITY;
    for (int i = lane; i < parts; i += 32) top = fmaxf(top, p.part_ml[index(i)].x);
#pragma unroll
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
    const float ref = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int i0 = warp; i0 < parts; i0 += kAhead * kWarps) {
        if (i0 > warp) fetch(i0);
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (i0 + u * kWarps >= parts) break;
            const float f = fast_exp2(ml[u].x - ref);
            sum += f * ml[u].y;
            acc.x += f * x[u].x; acc.y += f * x[u].y; acc.z += f * x[u].z; acc.w += f * x[u].w;
        }
    }
    s_acc[warp][lane] = acc;
    if (lane == 0) s_sum[warp] = sum;
    __syncthreads();
    if (warp == 0) {
#pragma unroll
        for (int w = 1; w < kWarps; ++w) {
            const float4 y = s_acc[w][lane];
            acc.x += y.x; acc.y += y.y; acc.z += y.z; acc.w += y.w;
            sum += s_sum[w];
        }
        const int bh = entry / p.row_tiles, b = bh / p.Hkv, h = bh - b * p.Hkv;
        const int j = r / p.Hg, head = h * p.Hg + (r - j * p.Hg);
        store_row(p.out + b * p.o_sb + j * p.o_sn + head * p.o_sh, lane, acc, sum, FP8 ? p.c.v_scale[h] : 1.0f);
        if (p.lse && lane == 0) p.lse[((int64_t)b * p.nq + j) * p.H + head] = log_sum(top, sum);
    }
}

}  // namespace paged
}  // namespace aa
