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
// d + 64 of a rotation.
#pragma once
#include <cuda_fp8.h>

#include "paged_common.cuh"

namespace aa {
namespace paged {

constexpr int kAppendThreads = 256;
constexpr int kRowsAtOnce = kAppendThreads / 8;

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
    int T, B, H, Hkv, Hg;
    int per_seq;                                    // cu == null: tokens of every sequence
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
__device__ __forceinline__ uint2 pack8_e4m3(const float (&f)[8], float scale) {
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        w[i >> 2] |= (uint32_t)__nv_cvt_float_to_fp8(__fdiv_rn(f[i], scale), __NV_SATFINITE, __NV_E4M3) << (8 * (i & 3));
    return make_uint2(w[0], w[1]);
}
__device__ __forceinline__ void load_piece(const Rows& r, int token, int head, int c, uint4& lo, uint4& hi) {
    const uint4* src = reinterpret_cast<const uint4*>(r.ptr + token * r.token + head * r.head);
    lo = src[c];
    hi = src[c + 8];
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

// Mean key of a complete page in 8 bits.  Every row of the page has been written and is visible to the block.
template <bool FP8>
__device__ void summarise_page(const AppendParams& p, int page, int h) {
    __shared__ double s_sum[kAppendThreads / 32][kD];                  // by warp
    __shared__ float s_max[kD / 32];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, c = tid & 7;
    const int rows = 1 << p.c.log2_page;
    const uint8_t* base = p.c.k.ptr + page * p.c.k.page + h * p.c.k.head;
    double sum[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) sum[i] = 0.0;
    for (int r = tid >> 3; r < rows; r += kRowsAtOnce) {
        float f[16];
        if (FP8) {
            // e4m3 codes through f16, exactly; a thread owns values 16 c .. 16 c + 15
            const uint4 x = __ldcg(reinterpret_cast<const uint4*>(base + r * p.c.k.row) + c);
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t y = e4m3x2_to_f16x2(w[i >> 1] >> (16 * (i & 1)));
                const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&y));
                f[2 * i] = v.x;
                f[2 * i + 1] = v.y;
            }
        } else {
            float lo[8], hi[8];
            unpack8(__ldcg(reinterpret_cast<const uint4*>(base + r * p.c.k.row) + 2 * c), lo);
            unpack8(__ldcg(reinterpret_cast<const uint4*>(base + r * p.c.k.row) + 2 * c + 1), hi);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                f[i] = lo[i];
                f[8 + i] = hi[i];
            }
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) sum[i] += (double)f[i];
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        sum[i] += __shfl_xor_sync(0xFFFFFFFFu, sum[i], 8);
        sum[i] += __shfl_xor_sync(0xFFFFFFFFu, sum[i], 16);
    }
    if (lane < 8)
#pragma unroll
        for (int i = 0; i < 16; ++i) s_sum[warp][16 * c + i] = sum[i];
    __syncthreads();
    float mean = 0.0f;
    if (tid < kD) {
        double x = 0.0;
#pragma unroll
        for (int w = 0; w < kAppendThreads / 32; ++w) x += s_sum[w][tid];
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

// grid (tasks, Hkv + (query ? Hkv : 0)): a task is one page a sequence writes to; y < Hkv: that KV head's keys and
// values, else the query heads of group y - Hkv.
template <bool FP8>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const __grid_constant__ AppendParams p) {
    const int tid = threadIdx.x, lane = tid & 31, c = tid & 7;
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
    const int lo = max(span.start, first), hi = min(span.end, first + rows);    // positions of this task
    const int token0 = span.token - span.start;                                // token of position x: token0 + x

    if ((int)blockIdx.y >= p.Hkv) {
        const int h0 = ((int)blockIdx.y - p.Hkv) * p.Hg;
        for (int pos = lo + (tid >> 3); pos < hi; pos += kRowsAtOnce) {
            if (p.cos && pos >= p.rope_rows) {
                raise_status(p.c, kStatusTooLong);
                continue;
            }
            Turn turn;
            if (p.cos) turn = load_turn(p, pos, c);
#pragma unroll 4
            for (int i = 0; i < p.Hg; ++i) {
                uint4 a, d;
                load_piece(p.query, token0 + pos, h0 + i, c, a, d);
                if (p.cos) {
                    Piece x;
                    unpack8(a, x.lo);
                    unpack8(d, x.hi);
                    rotate(x, turn);
                    a = pack8(x.lo);
                    d = pack8(x.hi);
                }
                store_piece(p.query_out, token0 + pos, h0 + i, c, a, d);
            }
        }
        return;
    }

    const int h = blockIdx.y;
    int page = -1;
    if (page_index < p.c.table_width) {
        page = pool_page(p.c, b, page_index);
        if (page < 0 && tid == 0) raise_status(p.c, kStatusBadPage);
    } else if (tid == 0) {
        raise_status(p.c, kStatusTooLong);
    }
    const float ks = FP8 ? p.c.k_scale[h] : 1.0f, vs = FP8 ? p.c.v_scale[h] : 1.0f;
    for (int pos = lo + (tid >> 3); pos < hi; pos += kRowsAtOnce) {
        if (p.cos && pos >= p.rope_rows) {
            raise_status(p.c, kStatusTooLong);
            continue;
        }
        uint4 ka, kd, va, vd;
        load_piece(p.key, token0 + pos, h, c, ka, kd);
        load_piece(p.value, token0 + pos, h, c, va, vd);
        Piece k;
        unpack8(ka, k.lo);
        unpack8(kd, k.hi);
        if (p.cos) {
            rotate(k, load_turn(p, pos, c));
            ka = pack8(k.lo);
            kd = pack8(k.hi);
        }
        if (p.key_out.ptr) store_piece(p.key_out, token0 + pos, h, c, ka, kd);
        if (page < 0) continue;
        uint8_t* k_row = p.c.k.ptr + page * p.c.k.page + h * p.c.k.head + (pos - first) * p.c.k.row;
        uint8_t* v_row = p.c.v.ptr + page * p.c.v.page + h * p.c.v.head + (pos - first) * p.c.v.row;
        if (FP8) {
            Piece v;
            unpack8(va, v.lo);
            unpack8(vd, v.hi);
            reinterpret_cast<uint2*>(k_row)[c] = pack8_e4m3(k.lo, ks);
            reinterpret_cast<uint2*>(k_row)[c + 8] = pack8_e4m3(k.hi, ks);
            reinterpret_cast<uint2*>(v_row)[c] = pack8_e4m3(v.lo, vs);
            reinterpret_cast<uint2*>(v_row)[c + 8] = pack8_e4m3(v.hi, vs);
        } else {
            reinterpret_cast<uint4*>(k_row)[c] = ka;
            reinterpret_cast<uint4*>(k_row)[c + 8] = kd;
            reinterpret_cast<uint4*>(v_row)[c] = va;
            reinterpret_cast<uint4*>(v_row)[c + 8] = vd;
        }
    }
    if (p.codes && page >= 0 && hi == first + rows && (!p.cos || hi <= p.rope_rows)) {
        __syncthreads();                            // the block's own rows are visible to all of it
        summarise_page<FP8>(p, page, h);
    }
}

}  // namespace paged
}  // namespace aa
