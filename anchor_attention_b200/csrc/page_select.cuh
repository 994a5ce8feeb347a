// Picks the pages of a long cache that a decode step attends, by a score of every page's mean key.
//
//   score(page) = max over the rows r of the group of  (code_r . code_page) scale_r  *  scale_page
//
// with the query rows and the page means (paged_append.cuh) in 8 bits: a page costs 132 bytes instead of
// page_size * 512, and as the dot products are whole numbers the order of a sum cannot move a page across the
// cut.  The first and the last pages of a sequence are always kept; the rest go by score, ties to the lower
// page, and come out in ascending order.
//
// A cluster of blocks works on one (sequence, KV head).  Its warps score 16 pages at a time, four lanes a page, with
// four-byte dot products (with the loads and the counting left out, the 8-bit matrix instructions took 3.7 of the batch's
// 13.3 us), and leave the scores as ordered 32-bit keys in the first block's shared memory; that block finds the last key
// that gets in by counting over 11 + 11 + 10 bits and writes the list.  The scores are a few dependent loads per page, so a
// small batch is a matter of latency: eight blocks share a sequence there, and each warp has 32 pages' loads in flight.
//
// Measured (B200, whole calls): one sequence of 131072 tokens in pages of 64 8.7 us; 32 of up to 65536 in pages of 32 25 us for
// 45 MB; a kernel that only reads 42 MB in rows of 128 bytes at random takes 10 to 13.  The rest is unequal lengths and a chain
// of waits: lengths, page numbers, codes, counts.  Blocks for a sequence and head of that batch, on the GPU: one 28.0 us,
// two 24.4 (what the rule takes), four 27.7, eight 32.8.
#pragma once
#include "paged_common.cuh"

namespace aa {
namespace paged {

constexpr int kSelectThreads = 256;
constexpr int kSelectWarps = kSelectThreads / 32;
constexpr int kMaxSelectRows = 256;                 // new tokens * group: 33 KB of query codes
constexpr int kMaxSelectPages = 40960;              // 160 KB of keys
constexpr int kMaxSelectCluster = 8;
constexpr int kBins = 2048;                         // of one counting pass
constexpr int kBinsPerThread = kBins / kSelectThreads;

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
// keys (rounded up to whole vectors for every thread), counts, query codes and scales
__host__ __device__ inline int select_key_slots(int table_width) {
    return (table_width + 4 * kSelectThreads - 1) / (4 * kSelectThreads) * (4 * kSelectThreads);
}
inline size_t select_smem_bytes(int rows, int table_width) {
    return (size_t)select_key_slots(table_width) * 4 + kBins * 4 + (size_t)select_row_tiles(rows) * 8 * (kD + 4);
}

// larger score, larger key; +0 and -0 alike
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t u = __float_as_uint(__fadd_rn(x, 0.0f));
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// the address in block 0 of the cluster of a shared-memory address of this block
__device__ __forceinline__ uint32_t in_first_block(uint32_t addr) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
    return r;
}
__device__ __forceinline__ void store_cluster(uint32_t addr, uint32_t x) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(x) : "memory");
}

// Sum of x over the threads below this one; `total`: over all.  Two barriers.
__device__ __forceinline__ int2 block_scan(int2 x, int2& total, int2* s_warp) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int2 incl = x;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int a = __shfl_up_sync(0xFFFFFFFFu, incl.x, d), b = __shfl_up_sync(0xFFFFFFFFu, incl.y, d);
        if (lane >= d) {
            incl.x += a;
            incl.y += b;
        }
    }
    if (lane == 31) s_warp[warp] = incl;
    __syncthreads();
    int2 before = make_int2(incl.x - x.x, incl.y - x.y);
    total = make_int2(0, 0);
#pragma unroll
    for (int w = 0; w < kSelectWarps; ++w) {
        const int2 n = s_warp[w];
        if (w < warp) {
            before.x += n.x;
            before.y += n.y;
        }
        total.x += n.x;
        total.y += n.y;
    }
    __syncthreads();
    return before;
}

// A lane's share of 16 pages' mean keys: lane (g, t) holds the bytes 16 t .. 16 t + 15 and 64 + 16 t .. 64 + 16 t + 15 of
// pages g and g + 8.
struct PageTile {
    uint4 lo[2], hi[2];
    float scale[2];
    int page[2];
};

__global__ void __launch_bounds__(kSelectThreads, 4) page_select_kernel(const __grid_constant__ SelectParams p, int cluster) {
    extern __shared__ __align__(128) uint8_t page_select_smem[];
    __shared__ int2 s_warp[kSelectWarps];
    __shared__ uint32_t s_prefix;
    __shared__ int s_need;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int bh = blockIdx.x / cluster, b = bh / p.Hkv, h = bh - b * p.Hkv;
    const int rank = cluster > 1 ? (int)cluster_rank() : 0;
    const int padded = select_row_tiles(p.rows) * 8;
    uint32_t* s_key = reinterpret_cast<uint32_t*>(page_select_smem);
    int* s_hist = reinterpret_cast<int*>(s_key + select_key_slots(p.c.table_width));
    uint32_t* s_q = reinterpret_cast<uint32_t*>(s_hist + kBins);                  // [padded][32] four codes each
    float* s_scale = reinterpret_cast<float*>(s_q + padded * 32);                 // [padded]

    start_next_kernel();
    wait_for_kernels_before();
    const int len = seq_len(p.c, b);
    if (tid == 0 && h == 0 && rank == 0 && p.c.seq_lens[b] > ((int64_t)p.c.table_width << p.c.log2_page))
        raise_status(p.c, kStatusTooLong);
    const int live = (int)(((int64_t)len + (1 << p.c.log2_page) - 1) >> p.c.log2_page);
    const int count = min(live, p.top);
    int32_t* out = p.out + (int64_t)bh * p.top;
    if (rank == 0) {
        if (tid == 0) p.counts[bh] = count;
        for (int i = count + tid; i < p.top; i += kSelectThreads) out[i] = -1;
    }
    if (live <= p.top) {                            // the same for all blocks of the cluster
        if (rank == 0)
            for (int i = tid; i < live; i += kSelectThreads) out[i] = i;
        return;
    }
    if (cluster > 1) cluster_arrive();              // every block has started: before the first store to another

    // ---- page numbers of this warp's first two tiles, while the queries arrive
    const int stride = cluster * kSelectWarps * 16;
    auto find = [&](int base, PageTile& x) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int logical = base + g + 8 * i;
            x.page[i] = logical < live ? p.c.table[b * p.c.table_stride + logical] : -1;
        }
    };
    auto load = [&](int base, PageTile& x) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if ((uint32_t)x.page[i] >= (uint32_t)p.c.pages) {
                if (base + g + 8 * i < live) raise_status(p.c, kStatusBadPage);
                x.page[i] = -1;
            }
            x.lo[i] = x.hi[i] = make_uint4(0, 0, 0, 0);
            x.scale[i] = 0.0f;
            if (x.page[i] >= 0) {
                const int64_t at = (int64_t)x.page[i] * p.Hkv + h;
                x.lo[i] = *(reinterpret_cast<const uint4*>(p.codes + at * kD) + t);
                x.hi[i] = *(reinterpret_cast<const uint4*>(p.codes + at * kD) + 4 + t);
                x.scale[i] = p.code_scales[at];
            }
        }
    };
    const int base0 = (rank * kSelectWarps + warp) * 16;
    PageTile x0, x1;
    find(base0, x0);
    find(base0 + stride, x1);

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
    load(base0, x0);
    load(base0 + stride, x1);
    __syncthreads();
    if (cluster > 1) cluster_wait();

    // ---- scores
    const uint32_t keys_at = cluster > 1 ? in_first_block(smem_u32(s_key)) : 0;
    auto score = [&](int base, const PageTile& x) {
        float best[2] = {-INFINITY, -INFINITY};
        const uint32_t w0[8] = {x.lo[0].x, x.lo[0].y, x.lo[0].z, x.lo[0].w, x.hi[0].x, x.hi[0].y, x.hi[0].z, x.hi[0].w};
        const uint32_t w1[8] = {x.lo[1].x, x.lo[1].y, x.lo[1].z, x.lo[1].w, x.hi[1].x, x.hi[1].y, x.hi[1].z, x.hi[1].w};
#pragma unroll 1
        for (int r0 = 0; r0 < p.rows; r0 += 4) {
            int d[2][4];                            // this lane's share of the products of its pages with four rows
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint4* q = reinterpret_cast<const uint4*>(s_q + (r0 + r) * 32);
                const uint4 u = q[t], v = q[4 + t];
                const uint32_t c[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
                int e0 = 0, e1 = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    e0 = __dp4a((int)w0[i], (int)c[i], e0);
                    e1 = __dp4a((int)w1[i], (int)c[i], e1);
                }
                d[0][r] = e0;
                d[1][r] = e1;
            }
            // added up over the four lanes of a page, so that lane t ends with row r0 + t
            const float row_scale = s_scale[r0 + t];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const bool up1 = t & 2, up0 = t & 1;
                const int k0 = (up1 ? d[i][2] : d[i][0]) + __shfl_xor_sync(0xFFFFFFFFu, up1 ? d[i][0] : d[i][2], 2);
                const int k1 = (up1 ? d[i][3] : d[i][1]) + __shfl_xor_sync(0xFFFFFFFFu, up1 ? d[i][1] : d[i][3], 2);
                const int all = (up0 ? k1 : k0) + __shfl_xor_sync(0xFFFFFFFFu, up0 ? k0 : k1, 1);
                if (r0 + t < p.rows) best[i] = fmaxf(best[i], __fmul_rn((float)all, row_scale));
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            best[i] = fmaxf(best[i], __shfl_xor_sync(0xFFFFFFFFu, best[i], 1));
            best[i] = fmaxf(best[i], __shfl_xor_sync(0xFFFFFFFFu, best[i], 2));
            const int logical = base + g + 8 * i;
            if (t == 0 && logical < live) {
                uint32_t key = x.page[i] >= 0 ? order_key(__fmul_rn(best[i], x.scale[i])) : 0u;
                if (logical < p.keep_first || logical >= live - p.keep_last) key = 0xFFFFFFFFu;
                if (cluster > 1)
                    store_cluster(keys_at + logical * 4, key);
                else
                    s_key[logical] = key;
            }
        }
    };
    for (int base = base0; base < live; base += 2 * stride) {
        score(base, x0);
        if (base + stride < live) score(base + stride, x1);
        if (base + 2 * stride < live) {
            find(base + 2 * stride, x0);
            find(base + 3 * stride, x1);
            load(base + 2 * stride, x0);
            load(base + 3 * stride, x1);
        }
    }
    if (cluster > 1) {
        cluster_arrive();
        cluster_wait();
        if (rank > 0) return;
    } else {
        __syncthreads();
    }

    // ---- the count-th largest key, 11, 11 and 10 bits at a time from the top
    uint32_t prefix = 0;
    int need = count;                               // how many of the keys with this prefix get in
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const uint32_t digits = pass == 2 ? 1023u : 2047u;
        const uint32_t mask = pass == 0 ? 0u : pass == 1 ? 0xFFE00000u : 0xFFFFFC00u;
#pragma unroll
        for (int i = 0; i < kBinsPerThread; ++i) s_hist[tid + i * kSelectThreads] = 0;
        __syncthreads();
        for (int i = tid; i < live; i += kSelectThreads) {
            const uint32_t k = s_key[i];
            if ((k & mask) == prefix) atomicAdd(&s_hist[(k >> shift) & digits], 1);
        }
        __syncthreads();
        // thread: bins kBinsPerThread (threads - 1 - tid) .. + kBinsPerThread - 1, the highest bins first
        const int bin0 = kBinsPerThread * (kSelectThreads - 1 - tid);
        int bins[kBinsPerThread], sum = 0;
#pragma unroll
        for (int i = 0; i < kBinsPerThread; ++i) sum += bins[i] = s_hist[bin0 + i];
        int2 total;
        int above = block_scan(make_int2(sum, 0), total, s_warp).x;               // keys in higher bins
        if (above < need && above + sum >= need) {
            int bin = kBinsPerThread - 1;
#pragma unroll
            for (int i = kBinsPerThread - 1; i > 0; --i)
                if (bin == i && above + bins[i] < need) {
                    above += bins[i];
                    bin = i - 1;
                }
            s_prefix = prefix | ((uint32_t)(bin0 + bin) << shift);
            s_need = need - above;
        }
        __syncthreads();
        prefix = s_prefix;
        need = s_need;
    }

    // ---- keys above the cut, and the first `need` of those equal to it: a thread takes a run of keys
    const int run = (live + 4 * kSelectThreads - 1) / (4 * kSelectThreads) * 4;
    const int begin = min(tid * run, live), end = min(begin + run, live);
    int2 mine = make_int2(0, 0), total;
    for (int i = begin; i < end; i += 4) {
        const uint4 k4 = *reinterpret_cast<const uint4*>(s_key + i);
        const uint32_t k[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            mine.x += i + x < end && k[x] > prefix;
            mine.y += i + x < end && k[x] == prefix;
        }
    }
    int2 before = block_scan(mine, total, s_warp);
    if (mine.x + mine.y > 0)
        for (int i = begin; i < end; ++i) {
            const uint32_t k = s_key[i];
            if (k > prefix || (k == prefix && before.y < need)) out[before.x + min(before.y, need)] = i;
            before.x += k > prefix;
            before.y += k == prefix;
        }
}

}  // namespace paged
}  // namespace aa
