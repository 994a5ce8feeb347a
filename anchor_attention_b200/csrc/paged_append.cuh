// Appends new keys and values to the pages of a cache, rotating keys (and queries) on the way.
//
//   x'[d]      = x[d] cos[pos][d] - x[d + 64] sin[pos][d]
//   x'[d + 64] = x[d + 64] cos[pos][d] + x[d] sin[pos][d]        d < 64, in 32 bits, rounded once: to bf16, or to
//                                                                the e4m3 code of x' / scale[head]
//
// A page of one KV head belongs to one block: it writes all new rows of the page, so when the page's last row
// is among them the block can form the page's mean key, rows of earlier calls included, without a word from any
// other block.  The mean is kept in 8 bits, scale = max|mean| * (1 / 127) and code = rint(mean / scale): 132 bytes
// instead of page_size * 256 for the page selection to read.  The sum runs in 64 bits, where adding a page's keys
// loses nothing, so codes do not depend on the order of the sum.
//
// The kernel moves bytes: 8 threads take a row of 256 bytes in 16-byte pieces, a thread owning the values d and
// d + 64 of a rotation.  For prompts a block takes several heads of a page, so that a row's cosines and sines are read once
// for all of them and two heads' loads are in flight while the page number arrives; a single token's append is
// latency alone and takes a block for every head.  Measured (B200): 26667 tokens of five prompts, 32/8 heads, bf16 124 us,
// 5.8 TB/s of reads and writes mixed, 4 us of them for the means; 14232 tokens into e4m3 pages, 28/4 heads,
// 55 us, 4.6 TB/s (one head's loads in flight instead of two: 55 against 57 us; two for bf16: 124 against 128 us); 64 single tokens 3 us on the GPU.
#pragma once
#include <cuda_fp8.h>

#include "paged_common.cuh"

namespace aa {
namespace paged {

constexpr int kAppendThreads = 256;                // for prompts; a single token a sequence takes kSingleThreads
constexpr int kSingleThreads = 128;
constexpr int kStagedRows = 128;                    // rows of keys (over all heads) a block adds up in shared memory

struct Rows {                                       // [tokens, heads, 128] bf16, strides in elements
    __nv_bfloat16* ptr;
    int64_t token, head;
};

struct AppendParams {
    Cache c;
    Rows key, value, query;                         // query.ptr may be null
    Rows query_out, key_out;                        // key_out.ptr may be null
    const int32_t* cu;                              // [B + 1] first token of every sequence, or null: T / B each
    const float *cos, *sin;                         // [rope_rows, 64], or null: no rotation
    int rope_rows;
    int8_t* codes;                                  // [pages, Hkv, 128] or null
    float* code_scales;                             // [pages, Hkv]
    int T, B, H, Hkv;
    int kv_heads, kv_blocks, q_heads;               // heads of a block; blocks y < kv_blocks take keys and values
    int per_seq;                                    // cu == null: tokens of every sequence
    bool staged;                                    // shared memory holds a block's pages
};

// New positions [start, end) of a sequence (negative ones are padding and are left out) and its first token.
struct Span {
    int start, end, token;                          // token: that of position `start`
};

__device__ __forceinline__ Span new_span(const AppendParams& p, int b) {
    int first, n;
    if (p.cu) {
        first = p.cu[b];
        const int last = p.cu[b + 1];
        if (first < 0 || last < first || last > p.T) return Span{0, 0, 0};       // tokens outside the inputs
        n = last - first;
    } else {
        first = b * p.per_seq;
        n = p.per_seq;
    }
    const int end = max(p.c.seq_lens[b], 0);
    const int start = max(end - n, 0);
    return Span{start, end, first + n - (end - start)};
}

__device__ __forceinline__ int span_pages(const Span& s, int log2_page) {
    return s.end > s.start ? ((s.end - 1) >> log2_page) - (s.start >> log2_page) + 1 : 0;
}

struct Piece {                                      // the 8 + 8 values of a row one thread owns
    float lo[8], hi[8];
};

__device__ __forceinline__ void unpack8(const uint4& x, float (&f)[8]) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
}
__device__ __forceinline__ uint2 pack8_e4m3(const float (&f)[8], const Divisor& d) {
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; i += 2)
        w[i >> 2] |= (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(divide(f[i], d), divide(f[i + 1], d)), __NV_SATFINITE, __NV_E4M3)
                     << (8 * (i & 3));
    return make_uint2(w[0], w[1]);
}
__device__ __forceinline__ void load_piece(const Rows& r, int token, int head, int c, uint4& lo, uint4& hi) {
    const uint4* src = reinterpret_cast<const uint4*>(r.ptr + token * r.token + head * r.head);
    lo = __ldcs(src + c);                           // read once
    hi = __ldcs(src + c + 8);
}
__device__ __forceinline__ void store_piece(const Rows& r, int token, int head, int c, const uint4& lo, const uint4& hi) {
    uint4* dst = reinterpret_cast<uint4*>(r.ptr + token * r.token + head * r.head);
    dst[c] = lo;
    dst[c + 8] = hi;
}

struct Turn {
    float cos[8], sin[8];
};
__device__ __forceinline__ Turn load_turn(const AppendParams& p, int pos, int c) {
    Turn t;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float4 a = reinterpret_cast<const float4*>(p.cos + (int64_t)pos * 64)[2 * c + i];
        const float4 b = reinterpret_cast<const float4*>(p.sin + (int64_t)pos * 64)[2 * c + i];
        t.cos[4 * i] = a.x; t.cos[4 * i + 1] = a.y; t.cos[4 * i + 2] = a.z; t.cos[4 * i + 3] = a.w;
        t.sin[4 * i] = b.x; t.sin[4 * i + 1] = b.y; t.sin[4 * i + 2] = b.z; t.sin[4 * i + 3] = b.w;
    }
    return t;
}
// products and sums rounded one by one (no fused multiply-add): the result does not depend on the compiler
__device__ __forceinline__ void rotate(Piece& x, const Turn& t) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float a = x.lo[i], b = x.hi[i];
        x.lo[i] = __fsub_rn(__fmul_rn(a, t.cos[i]), __fmul_rn(b, t.sin[i]));
        x.hi[i] = __fadd_rn(__fmul_rn(b, t.cos[i]), __fmul_rn(a, t.sin[i]));
    }
}

// Mean key of a complete page in 8 bits.  Every row of the page is visible to the block, at `base` (shared memory or the
// pool), `stride` bytes apart.
template <bool FP8, int THREADS>
__device__ void summarise_page(const AppendParams& p, int page, int h, const uint8_t* base, int64_t stride) {
    constexpr int kGroups = THREADS / 32;          // a warp adds up two rows at a time, a thread 8 of their values
    __shared__ double s_sum[kGroups][kD];
    __shared__ float s_max[kD / 32];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rows = 1 << p.c.log2_page;
    base += (tid & 15) * (FP8 ? 8 : 16);
    double sum[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[i] = 0.0;
#pragma unroll 8
    for (int r = tid >> 4; r < rows; r += 2 * kGroups) {              // 16 rows or more
        float f[8];
        if (FP8) {                                  // e4m3 codes through f16, exactly
            const uint2 x = *reinterpret_cast<const uint2*>(base + r * stride);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t y = e4m3x2_to_f16x2((i < 2 ? x.x : x.y) >> (16 * (i & 1)));
                const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&y));
                f[2 * i] = v.x;
                f[2 * i + 1] = v.y;
            }
        } else {
            unpack8(*reinterpret_cast<const uint4*>(base + r * stride), f);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] += (double)f[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[i] += __shfl_xor_sync(0xFFFFFFFFu, sum[i], 16);
    __syncthreads();                                // the sums of the head before have been read
    if (lane < 16)
#pragma unroll
        for (int i = 0; i < 8; ++i) s_sum[warp][lane * 8 + i] = sum[i];
    __syncthreads();
    float mean = 0.0f;
    if (tid < kD) {
        double x = 0.0;
#pragma unroll
        for (int w = 0; w < kGroups; ++w) x += s_sum[w][tid];
        mean = (float)(x / rows);                                     // rows is a power of two: exact before rounding
        if (FP8) mean = __fmul_rn(mean, p.c.k_scale[h]);
        float big = fabsf(mean);
        bool finite = big < INFINITY;
#pragma unroll
        for (int d = 16; d; d >>= 1) big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, d));
        finite = __all_sync(0xFFFFFFFFu, finite);
        if (lane == 0) s_max[warp] = finite ? big : INFINITY;
    }
    __syncthreads();
    if (tid < kD) {
        const float big = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
        // a page with an infinity or NaN among its keys gets the score 0
        const float scale = big < INFINITY ? __fmul_rn(big, kInv127) : 0.0f;
        const int64_t at = (int64_t)page * p.Hkv + h;
        p.codes[at * kD + tid] = scale > 0.0f ? (int8_t)fminf(fmaxf(rintf(__fdiv_rn(mean, scale)), -127.0f), 127.0f) : (int8_t)0;
        if (tid == 0) p.code_scales[at] = scale;
    }
}

// grid (tasks, kv_blocks + blocks of query heads): a task is one page a sequence writes to.
template <bool FP8, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == kAppendThreads ? 3 : 4) paged_append_kernel(const __grid_constant__ AppendParams p) {
    constexpr int kSlots = THREADS / 8;
    extern __shared__ __align__(128) uint8_t paged_append_smem[];                // rows of the keys as they are stored
    const int tid = threadIdx.x, lane = tid & 31, c = tid & 7;
    start_next_kernel();
    wait_for_kernels_before();
    // ---- which sequence and page: every warp walks the sequences 32 at a time, nothing is shared
    Span span{0, 0, 0};
    int b = 0, page_index = -1;
    if (!p.cu && p.per_seq == 1) {
        b = blockIdx.x;
        span = new_span(p, b);
        if (span_pages(span, p.c.log2_page) > 0) page_index = span.start >> p.c.log2_page;
    } else {
        int before = 0;
        for (int b0 = 0; b0 < p.B && page_index < 0; b0 += 32) {
            const Span s = b0 + lane < p.B ? new_span(p, b0 + lane) : Span{0, 0, 0};
            const int n = span_pages(s, p.c.log2_page);
            int incl = n;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int x = __shfl_up_sync(0xFFFFFFFFu, incl, d);
                if (lane >= d) incl += x;
            }
            const int want = (int)blockIdx.x - before;
            const uint32_t hit = __ballot_sync(0xFFFFFFFFu, want < incl);
            if (hit) {
                const int at = __ffs(hit) - 1;
                b = b0 + at;
                span.start = __shfl_sync(0xFFFFFFFFu, s.start, at);
                span.end = __shfl_sync(0xFFFFFFFFu, s.end, at);
                span.token = __shfl_sync(0xFFFFFFFFu, s.token, at);
                page_index = (span.start >> p.c.log2_page) + want - __shfl_sync(0xFFFFFFFFu, incl - n, at);
            }
            before += __shfl_sync(0xFFFFFFFFu, incl, 31);
        }
    }
    if (page_index < 0) return;
    const int rows = 1 << p.c.log2_page;
    const int first = page_index << p.c.log2_page;
    const int lo = max(span.start, first), hi = first + min(span.end - first, rows);    // positions of this task
    const int token0 = span.token - span.start;                                // token of position x: token0 + x

    // slots of 8 threads, a row each; where there are fewer rows, several heads go side by side
    int slot_rows = 1;
    while (slot_rows < kSlots && slot_rows < hi - lo) slot_rows *= 2;
    const int slot = tid >> 3;
    const int slot_row = slot % slot_rows, slot_head = slot / slot_rows, head_step = kSlots / slot_rows;
    bool beyond = false;                            // a position beyond the rotary tables

    if ((int)blockIdx.y >= p.kv_blocks) {
        const int h0 = ((int)blockIdx.y - p.kv_blocks) * p.q_heads, h1 = min(h0 + p.q_heads, p.H);
        for (int i = slot_row; i < hi - lo; i += slot_rows) {
            const int pos = lo + i;                    // lo + i + slot_rows could pass 2^31
            if (p.cos && pos >= p.rope_rows) {
                beyond = true;
                continue;
            }
            Turn turn;
            if (p.cos) turn = load_turn(p, pos, c);
            constexpr int kAhead = 4;
            for (int h = h0 + slot_head; h < h1; h += kAhead * head_step) {
                uint4 a[kAhead], d[kAhead];
#pragma unroll
                for (int u = 0; u < kAhead; ++u)
                    if (h + u * head_step < h1) load_piece(p.query, token0 + pos, h + u * head_step, c, a[u], d[u]);
#pragma unroll
                for (int u = 0; u < kAhead; ++u) {
                    if (h + u * head_step >= h1) break;
                    if (p.cos) {
                        Piece x;
                        unpack8(a[u], x.lo);
                        unpack8(d[u], x.hi);
                        rotate(x, turn);
                        a[u] = pack8(x.lo);
                        d[u] = pack8(x.hi);
                    }
                    store_piece(p.query_out, token0 + pos, h + u * head_step, c, a[u], d[u]);
                }
            }
        }
        if (beyond) raise_status(p.c, kStatusTooLong);
        return;
    }

    const int h0 = blockIdx.y * p.kv_heads, h1 = min(h0 + p.kv_heads, p.Hkv);
    const bool in_table = page_index < p.c.table_width;
    const int page = in_table ? pool_page(p.c, b, page_index) : -1;
    // the page fills up: its mean is wanted, from shared memory where it fits
    const bool fills = p.codes && page >= 0 && hi - first == rows && (!p.cos || hi <= p.rope_rows);
    const bool staged = fills && p.staged;
    constexpr int kRowBytes8 = FP8 ? 128 : 256;
    if (staged)                                     // rows of earlier calls
        for (int i = tid; i < (lo - first) * (h1 - h0) * (kRowBytes8 / 16); i += THREADS) {
            const int at = i / (kRowBytes8 / 16), piece = i % (kRowBytes8 / 16), row = at % (lo - first), h = at / (lo - first);
            reinterpret_cast<uint4*>(paged_append_smem + (h * rows + row) * kRowBytes8)[piece] =
                reinterpret_cast<const uint4*>(p.c.k.ptr + page * p.c.k.page + (h0 + h) * p.c.k.head + row * p.c.k.row)[piece];
        }
    for (int i = slot_row; i < hi - lo; i += slot_rows) {
        const int pos = lo + i;
        if (p.cos && pos >= p.rope_rows) {
            beyond = true;
            continue;
        }
        Turn turn;
        if (p.cos) turn = load_turn(p, pos, c);
        constexpr int kAhead = FP8 ? 1 : 2;      // an e4m3 head has its quotients to wait for
        for (int hb = h0 + slot_head; hb < h1; hb += kAhead * head_step) {
            uint4 ka[kAhead], kd[kAhead], va[kAhead], vd[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
                if (hb + u * head_step < h1) {
                    load_piece(p.key, token0 + pos, hb + u * head_step, c, ka[u], kd[u]);
                    load_piece(p.value, token0 + pos, hb + u * head_step, c, va[u], vd[u]);
                }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int h = hb + u * head_step;
                if (h >= h1) break;
                Piece k;
                unpack8(ka[u], k.lo);
                unpack8(kd[u], k.hi);
                if (p.cos) {
                    rotate(k, turn);
                    ka[u] = pack8(k.lo);
                    kd[u] = pack8(k.hi);
                }
                if (p.key_out.ptr) store_piece(p.key_out, token0 + pos, h, c, ka[u], kd[u]);
                if (page < 0) continue;
                uint8_t* k_row = p.c.k.ptr + page * p.c.k.page + h * p.c.k.head + (pos - first) * p.c.k.row;
                uint8_t* v_row = p.c.v.ptr + page * p.c.v.page + h * p.c.v.head + (pos - first) * p.c.v.row;
                uint8_t* s_row = paged_append_smem + ((h - h0) * rows + pos - first) * kRowBytes8;
                if (FP8) {
                    Piece v;
                    unpack8(va[u], v.lo);
                    unpack8(vd[u], v.hi);
                    const Divisor ks = divisor(p.c.k_scale[h]), vs = divisor(p.c.v_scale[h]);
                    const uint2 lo8 = pack8_e4m3(k.lo, ks), hi8 = pack8_e4m3(k.hi, ks);
                    reinterpret_cast<uint2*>(k_row)[c] = lo8;
                    reinterpret_cast<uint2*>(k_row)[c + 8] = hi8;
                    if (staged) {
                        reinterpret_cast<uint2*>(s_row)[c] = lo8;
                        reinterpret_cast<uint2*>(s_row)[c + 8] = hi8;
                    }
                    reinterpret_cast<uint2*>(v_row)[c] = pack8_e4m3(v.lo, vs);
                    reinterpret_cast<uint2*>(v_row)[c + 8] = pack8_e4m3(v.hi, vs);
                } else {
                    reinterpret_cast<uint4*>(k_row)[c] = ka[u];
                    reinterpret_cast<uint4*>(k_row)[c + 8] = kd[u];
                    if (staged) {
                        reinterpret_cast<uint4*>(s_row)[c] = ka[u];
                        reinterpret_cast<uint4*>(s_row)[c + 8] = kd[u];
                    }
                    reinterpret_cast<uint4*>(v_row)[c] = va[u];
                    reinterpret_cast<uint4*>(v_row)[c + 8] = vd[u];
                }
            }
        }
    }
    if (beyond) raise_status(p.c, kStatusTooLong);
    if (page < 0) {
        if (tid == 0) raise_status(p.c, in_table ? kStatusBadPage : kStatusTooLong);
        return;
    }
    if (fills) {
        __syncthreads();                            // the block's own rows are visible to all of it
        for (int h = h0; h < h1; ++h)
            if (staged)
                summarise_page<FP8, THREADS>(p, page, h, paged_append_smem + (h - h0) * rows * kRowBytes8, kRowBytes8);
            else
                summarise_page<FP8, THREADS>(p, page, h, p.c.k.ptr + page * p.c.k.page + h * p.c.k.head, p.c.k.row);
    }
}

}  // namespace paged
}  // namespace aa
