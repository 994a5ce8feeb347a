// Picks the pages of a long cache that a decode step attends, by a score of every page's mean key.
//
//   score(page) = max over the rows r of the group of  (code_r . code_page) scale_r  *  scale_page
//
// with the query rows and the page means (paged_append.cuh) in 8 bits: a page costs 132 bytes instead of
// page_size * 512, and as the dot products are whole numbers the order of a sum cannot move a page across the
// cut.  The first and the last pages of a sequence are always kept; the rest go by score, ties to the lower
// page, and come out in ascending order.
//
// One block per (sequence, KV head): warps score 16 pages at a time with the 8-bit matrix instruction (pages as
// its 16 rows, 8 query rows as its columns), the scores stay in shared memory as ordered 32-bit keys, four
// counting passes over 8 bits each find the last key that gets in, and one more pass writes the list.
#pragma once
#include "paged_common.cuh"

namespace aa {
namespace paged {

constexpr int kSelectThreads = 512;
constexpr int kSelectWarps = kSelectThreads / 32;
constexpr int kMaxSelectRows = 256;                 // new tokens * group: 33 KB of query codes
constexpr int kMaxSelectPages = 40960;              // 160 KB of keys

struct SelectParams {
    Cache c;                                        // table, seq_lens, pages, log2_page, status
    const __nv_bfloat16* q;
    int64_t q_sb, q_sn, q_sh;
    const int8_t* codes;                            // [pages, Hkv, 128]
    const float* code_scales;                       // [pages, Hkv]
    int32_t* out;                                   // [B, Hkv, top]
    int32_t* counts;                                // [B, Hkv]
    int B, H, Hkv, Hg, nq, rows, top, keep_first, keep_last;
};

__host__ __device__ inline int select_row_tiles(int rows) { return (rows + 7) / 8; }
inline size_t select_smem_bytes(int rows, int table_width) {
    return (size_t)select_row_tiles(rows) * 8 * (kD + 4) + (size_t)table_width * 4;
}

// larger score, larger key; +0 and -0 alike
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t u = __float_as_uint(__fadd_rn(x, 0.0f));
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(kSelectThreads) page_select_kernel(const __grid_constant__ SelectParams p) {
    extern __shared__ __align__(128) uint8_t paged_smem[];
    uint8_t* smem = paged_smem;
    __shared__ int s_hist[256];
    __shared__ int s_warp[2][kSelectWarps];
    __shared__ uint32_t s_prefix;
    __shared__ int s_need;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int bh = blockIdx.x, b = bh / p.Hkv, h = bh - b * p.Hkv;
    const int padded = select_row_tiles(p.rows) * 8;
    uint32_t* s_q = reinterpret_cast<uint32_t*>(smem);                            // [padded][32] four codes each
    float* s_scale = reinterpret_cast<float*>(smem + (size_t)padded * kD);        // [padded]
    uint32_t* s_key = reinterpret_cast<uint32_t*>(smem + (size_t)padded * (kD + 4));

    const int len = seq_len(p.c, b);
    if (tid == 0 && h == 0 && p.c.seq_lens[b] > ((int64_t)p.c.table_width << p.c.log2_page)) raise_status(p.c, kStatusTooLong);
    const int live = (int)(((int64_t)len + (1 << p.c.log2_page) - 1) >> p.c.log2_page);
    const int count = min(live, p.top);
    int32_t* out = p.out + (int64_t)bh * p.top;
    if (tid == 0) p.counts[bh] = count;
    for (int i = count + tid; i < p.top; i += kSelectThreads) out[i] = -1;
    if (live <= p.top) {
        for (int i = tid; i < live; i += kSelectThreads) out[i] = i;
        return;
    }

    // ---- query rows in 8 bits
    for (int r = warp; r < padded; r += kSelectWarps) {
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (r < p.rows) {
            const int j = r / p.Hg;
            const uint2 x = reinterpret_cast<const uint2*>(p.q + b * p.q_sb + j * p.q_sn + (int64_t)(h * p.Hg + r - j * p.Hg) * p.q_sh)[lane];
            v[0] = __uint_as_float(x.x << 16);
            v[1] = __uint_as_float(x.x & 0xFFFF0000u);
            v[2] = __uint_as_float(x.y << 16);
            v[3] = __uint_as_float(x.y & 0xFFFF0000u);
        }
        float big = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
#pragma unroll
        for (int d = 16; d; d >>= 1) big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, d));
        const float scale = __fmul_rn(big, kInv127);
        uint32_t packed = 0;
        if (scale > 0.0f)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                packed |= ((uint32_t)(int)fminf(fmaxf(rintf(__fdiv_rn(v[i], scale)), -127.0f), 127.0f) & 0xFFu) << (8 * i);
        s_q[r * 32 + lane] = packed;
        if (lane == 0) s_scale[r] = r < p.rows ? scale : 0.0f;
    }
    __syncthreads();

    // ---- score 16 pages a warp; a lane's words of a page: bytes 16 t .. 16 t + 15 and 64 + 16 t .. 64 + 16 t + 15
    const int row_tiles = padded / 8;
    for (int base = warp * 16; base < live; base += kSelectWarps * 16) {
        uint32_t a[2][8];
        float scale[2];
        int page[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int logical = base + g + 8 * x;
            page[x] = -1;
            if (logical < live) {
                page[x] = pool_page(p.c, b, logical);
                if (page[x] < 0) raise_status(p.c, kStatusBadPage);
            }
            uint4 u = make_uint4(0, 0, 0, 0), w = u;
            scale[x] = 0.0f;
            if (page[x] >= 0) {
                const int64_t at = (int64_t)page[x] * p.Hkv + h;
                u = __ldg(reinterpret_cast<const uint4*>(p.codes + at * kD) + t);
                w = __ldg(reinterpret_cast<const uint4*>(p.codes + at * kD) + 4 + t);
                scale[x] = __ldg(p.code_scales + at);
            }
            a[x][0] = u.x; a[x][1] = u.y; a[x][2] = u.z; a[x][3] = u.w;
            a[x][4] = w.x; a[x][5] = w.y; a[x][6] = w.z; a[x][7] = w.w;
        }
        float best[2] = {-INFINITY, -INFINITY};
        for (int n = 0; n < row_tiles; ++n) {
            const uint4* q = reinterpret_cast<const uint4*>(s_q + (n * 8 + g) * 32);
            const uint4 u = q[t], w = q[4 + t];
            int d[4] = {0, 0, 0, 0};
            const uint32_t a0[4] = {a[0][0], a[1][0], a[0][1], a[1][1]};
            const uint32_t a1[4] = {a[0][2], a[1][2], a[0][3], a[1][3]};
            const uint32_t a2[4] = {a[0][4], a[1][4], a[0][5], a[1][5]};
            const uint32_t a3[4] = {a[0][6], a[1][6], a[0][7], a[1][7]};
            mma_s8(d, a0, u.x, u.y);
            mma_s8(d, a1, u.z, u.w);
            mma_s8(d, a2, w.x, w.y);
            mma_s8(d, a3, w.z, w.w);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int r = n * 8 + 2 * t + (x & 1);
                if (r < p.rows) best[x >> 1] = fmaxf(best[x >> 1], __fmul_rn((float)d[x], s_scale[r]));
            }
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            best[x] = fmaxf(best[x], __shfl_xor_sync(0xFFFFFFFFu, best[x], 1));
            best[x] = fmaxf(best[x], __shfl_xor_sync(0xFFFFFFFFu, best[x], 2));
            const int logical = base + g + 8 * x;
            if (t == 0 && logical < live) {
                uint32_t key = page[x] >= 0 ? order_key(__fmul_rn(best[x], scale[x])) : 0u;
                if (logical < p.keep_first || logical >= live - p.keep_last) key = 0xFFFFFFFFu;
                s_key[logical] = key;
            }
        }
    }

    // ---- the count-th largest key, 8 bits at a time from the top
    uint32_t prefix = 0;
    int need = count;                               // how many of the keys with this prefix get in
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) s_hist[tid] = 0;
        __syncthreads();
        const uint32_t mask = shift == 24 ? 0u : 0xFFFFFFFFu << (shift + 8);
        for (int i = tid; i < live; i += kSelectThreads) {
            const uint32_t k = s_key[i];
            if ((k & mask) == prefix) atomicAdd(&s_hist[(k >> shift) & 255u], 1);
        }
        __syncthreads();
        if (warp == 0) {                            // lane: bins 8 (31 - lane) .. + 7, the highest bins first
            int sum = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) sum += s_hist[8 * (31 - lane) + i];
            int incl = sum;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int x = __shfl_up_sync(0xFFFFFFFFu, incl, d);
                if (lane >= d) incl += x;
            }
            int above = incl - sum;                 // keys in higher bins
            if (above < need && incl >= need) {
                int bin = 8 * (31 - lane) + 7;
                while (above + s_hist[bin] < need) above += s_hist[bin--];
                s_prefix = prefix | ((uint32_t)bin << shift);
                s_need = need - above;
            }
        }
        __syncthreads();
        prefix = s_prefix;
        need = s_need;
    }

    // ---- keys above the cut, and the first `need` of those equal to it, in the order of the pages
    int done = 0, equal_done = 0;
    for (int i0 = 0; i0 < live; i0 += kSelectThreads) {
        const int i = i0 + tid;
        const uint32_t k = i < live ? s_key[i] : 0u;
        const bool more = i < live && k > prefix, equal = i < live && k == prefix;
        const uint32_t m_more = __ballot_sync(0xFFFFFFFFu, more), m_equal = __ballot_sync(0xFFFFFFFFu, equal);
        if (lane == 0) {
            s_warp[0][warp] = __popc(m_more);
            s_warp[1][warp] = __popc(m_equal);
        }
        __syncthreads();
        int more_before = done, equal_before = equal_done;
#pragma unroll
        for (int w = 0; w < kSelectWarps; ++w) {
            if (w < warp) {
                more_before += s_warp[0][w];
                equal_before += s_warp[1][w];
            }
            done += s_warp[0][w];
            equal_done += s_warp[1][w];
        }
        const uint32_t below = (1u << lane) - 1u;
        more_before += __popc(m_more & below);
        equal_before += __popc(m_equal & below);
        if (more || (equal && equal_before < need)) out[more_before + min(equal_before, need)] = i;
        __syncthreads();
    }
}

}  // namespace paged
}  // namespace aa
