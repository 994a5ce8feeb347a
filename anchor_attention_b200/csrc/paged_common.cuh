// What the kernels of the paged key-value cache share: the view of the page pools, page lookups that
// never turn a bad page number into an address, the status word, and warp-level matrix instructions.
//
// The pools are [pages, Hkv, page_size, 128]: bf16, or e4m3 codes that stand for code * scale[head].  Any
// strides are accepted as long as the 128 values of a row are contiguous and rows start on 16-byte
// boundaries, so both [pages, Hkv, page_size, 128] and [pages, page_size, Hkv, 128] memory works.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

namespace aa {
namespace paged {

constexpr int kMaxNew = 16;              // new tokens a sequence brings to one attention call, at most
constexpr uint32_t kStatusBadPage = 1;   // a page number outside the pool, or a list entry outside the sequence
constexpr uint32_t kStatusTooLong = 2;   // a sequence longer than its row of the block table, or than the rotary tables
constexpr uint32_t kStatusTimeout = 4;   // a bounded wait gave up

// Clears bits that the host has read.  Other streams may set others meanwhile.
__global__ void clear_status_kernel(uint32_t* status, uint32_t bits) { atomicAnd(status, ~bits); }

// An 8-bit code's scale is the largest magnitude times this: the product, not a division, is the definition.
constexpr float kInv127 = 1.0f / 127.0f;

// Every kernel here starts in the shadow of the one before it on the stream and lets the next do the same
// (programmatic launch): nothing in global memory is touched before wait_for_kernels_before(), which returns when all earlier
// kernels are done and their writes visible.
__device__ __forceinline__ void start_next_kernel() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_kernels_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

struct Pool {
    uint8_t* ptr;
    int64_t page, head, row;             // strides in bytes
};

struct Cache {
    Pool k, v;
    const float *k_scale, *v_scale;      // [Hkv], e4m3 pools only
    const int32_t* table;                // [B, table_width] page numbers
    int64_t table_stride;
    int table_width;
    int pages;                           // pages of the pool
    int log2_page;                       // page_size is a power of two, 16 .. 256
    const int32_t* seq_lens;             // [B]
    uint32_t* status;
};

__device__ __forceinline__ void raise_status(const Cache& c, uint32_t bit) { atomicOr(c.status, bit); }

// Tokens of sequence b, between 0 and what its row of the block table can hold.
__device__ __forceinline__ int seq_len(const Cache& c, int b) {
    const int len = max(c.seq_lens[b], 0);
    const int64_t cap = (int64_t)c.table_width << c.log2_page;
    return len <= cap ? len : (int)cap;
}

// The pool page of a sequence's logical page (below table_width), -1 if the number is outside the pool.
__device__ __forceinline__ int pool_page(const Cache& c, int b, int logical) {
    const int p = c.table[b * c.table_stride + logical];
    return (uint32_t)p < (uint32_t)c.pages ? p : -1;
}

// ---- quotients
// Division by one number for many: q = x r with r = 1 / s rounded, then one step q - (q s - x) r.  The step gives the
// correctly rounded quotient (P. Markstein, Computation of elementary functions on the IBM RISC System/6000
// processor, 1990) as long as nothing overflows or vanishes; what is not in a safe range divides.  A remainder of 0 has the
// sign + , so it is q s - x that is formed: -0 less +0 stays -0, as in a division by a positive s.
struct Divisor {
    float s, r;
    bool plain;                                     // s in a range where r and the step's products are normal numbers
};
__device__ __forceinline__ Divisor divisor(float s) {
    return Divisor{s, __fdiv_rn(1.0f, s), s >= 0x1p-60f && s <= 0x1p60f && (__float_as_uint(s) & 0x7FFFFFu) != 0x7FFFFFu};
}
__device__ __forceinline__ float quotient(float x, const Divisor& d) {              // d.plain, |x| up to 2^60
    const float q = __fmul_rn(x, d.r);
    return __fmaf_rn(-__fmaf_rn(q, d.s, -x), d.r, q);
}
__device__ __forceinline__ float divide(float x, const Divisor& d) {
    // a quotient so small that the step's remainder vanishes has the code 0 whatever its last bit
    return d.plain && fabsf(x) <= 0x1p60f ? quotient(x, d) : __fdiv_rn(x, d.s);
}

// ---- matrix instructions of one warp ---------------------------------------------------------------------
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
// transpose of an 8x8 matrix of 16-bit values, one row pair per lane
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// two e4m3 codes (the low 16 bits) as two f16 values; every e4m3 value is exact in f16
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t x) {
    uint32_t y;
    asm("{\n\t.reg .b16 lo;\n\tcvt.u16.u32 lo, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}

}  // namespace paged
}  // namespace aa
