// C ABI of the paged key-value cache: argument checks and launches.  Declarations are in
// include/anchor_attn_b200.h.
#include "../../include/anchor_attn_b200.h"

#include <math.h>

#include <utility>

#include "page_select.cuh"
#include "paged_append.cuh"
#include "paged_attend.cuh"

namespace aa {
int record_cuda_error(cudaError_t e, const char* what);      // anchor_abi.cu
}

namespace {

using aa::record_cuda_error;

struct Device {
    int id = -1, sms = 0;
};

// The current device and its SM count; raises the shared-memory limit of the kernels on a thread's first call
// for a device.
template <typename F>
int current_device(Device& known, F&& configure) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return record_cuda_error(e, "cudaGetDevice");
    if (known.id != dev) {
        e = cudaDeviceGetAttribute(&known.sms, cudaDevAttrMultiProcessorCount, dev);
        if (e != cudaSuccess) return record_cuda_error(e, "cudaDeviceGetAttribute(SM count)");
        e = configure();
        if (e != cudaSuccess) return record_cuda_error(e, "cudaFuncSetAttribute(paged cache)");
        known.id = dev;
    }
    return AA_OK;
}

bool misaligned(const void* p) { return ((uintptr_t)p & 15) != 0; }
bool bad_stride(int64_t s, int elements = 8) { return s % elements != 0; }

// table, lengths and shapes; log2 of the page size
int check_table(const aa_paged_cache_t& c, int* log2_page) {
    if (c.B <= 0 || c.Hkv <= 0) return AA_ERR_SHAPE;
    if (c.D != 128) return AA_ERR_HEAD_DIM;
    if (c.pages <= 0 || c.table_width <= 0 || c.page_size < 16 || c.page_size > 256 || (c.page_size & (c.page_size - 1)))
        return AA_ERR_PAGE_SIZE;
    if (!c.block_table || !c.seq_lens || !c.status) return AA_ERR_NULL;
    if ((int64_t)c.table_width * c.page_size > (int64_t)1 << 30 || (int64_t)c.B * c.Hkv > 1 << 24) return AA_ERR_TOO_LARGE;
    *log2_page = 31 - __builtin_clz((unsigned)c.page_size);
    return AA_OK;
}

int check_pools(const aa_paged_cache_t& c) {
    if (!c.k_pages || !c.v_pages) return AA_ERR_NULL;
    if (c.cache_dtype != AA_BF16 && c.cache_dtype != AA_E4M3) return AA_ERR_DTYPE;
    if (c.cache_dtype == AA_E4M3 && (!c.k_scale || !c.v_scale)) return AA_ERR_NULL;
    const int unit = c.cache_dtype == AA_E4M3 ? 16 : 8;
    for (int64_t s : {c.k_stride_page, c.k_stride_head, c.k_stride_row, c.v_stride_page, c.v_stride_head, c.v_stride_row})
        if (bad_stride(s, unit)) return AA_ERR_STRIDE;
    if (misaligned(c.k_pages) || misaligned(c.v_pages)) return AA_ERR_STRIDE;
    return AA_OK;
}

aa::paged::Cache view(const aa_paged_cache_t& c, int log2_page) {
    const int64_t size = c.cache_dtype == AA_E4M3 ? 1 : 2;
    aa::paged::Cache v;
    v.k = {static_cast<uint8_t*>(c.k_pages), c.k_stride_page * size, c.k_stride_head * size, c.k_stride_row * size};
    v.v = {static_cast<uint8_t*>(c.v_pages), c.v_stride_page * size, c.v_stride_head * size, c.v_stride_row * size};
    v.k_scale = c.k_scale;
    v.v_scale = c.v_scale;
    v.table = c.block_table;
    v.table_stride = c.table_stride;
    v.table_width = c.table_width;
    v.pages = c.pages;
    v.log2_page = log2_page;
    v.seq_lens = c.seq_lens;
    v.status = c.status;
    return v;
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
size_t align256(size_t x) { return (x + 255) / 256 * 256; }

// Launches a kernel that waits for those before it on the device (wait_for_kernels_before): the launch itself and the
// kernel's start overlap their end.
template <typename... P, typename... A>
cudaError_t launch_after(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, int cluster, const A&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// ---- tensor maps: a pool [pages, Hkv, page_size, 128] as a 4-D map, dimension 0 the row, the others by increasing
// stride (a dimension of size 1 last, where its stride does not matter).  A copy takes 128 bytes of `box` rows.
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_tiled() {
    static const EncodeTiledFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
                        q == cudaDriverEntryPointSuccess;
        return reinterpret_cast<EncodeTiledFn>(ok ? p : nullptr);
    }();
    return fn;
}

int make_page_map(CUtensorMap* map, const aa::paged::Pool& pool, const aa_paged_cache_t& c, int box, aa::paged::MapOrder* order) {
    const EncodeTiledFn encode = encode_tiled();
    if (!encode) return record_cuda_error(cudaErrorNotSupported, "cuTensorMapEncodeTiled entry point");
    struct Dim {
        int64_t stride;                            // bytes
        cuuint64_t size;
        int* place;
    };
    Dim d[3] = {{pool.row, (cuuint64_t)c.page_size, &order->row}, {pool.head, (cuuint64_t)c.Hkv, &order->head},
                {pool.page, (cuuint64_t)c.pages, &order->page}};
    for (int i = 0; i < 3; ++i)
        for (int j = i + 1; j < 3; ++j)
            if ((d[j].size != 1 && d[j].stride < d[i].stride) || (d[i].size == 1 && d[j].size != 1)) {
                const Dim x = d[i];
                d[i] = d[j];
                d[j] = x;
            }
    const bool fp8 = c.cache_dtype == AA_E4M3;
    const cuuint64_t row_bytes = fp8 ? 128 : 256;
    const cuuint64_t sizes[4] = {128, d[0].size, d[1].size, d[2].size};
    cuuint64_t strides[3];
    cuuint32_t boxes[4] = {fp8 ? 128u : 64u, 1, 1, 1};
    const cuuint32_t steps[4] = {1, 1, 1, 1};
    for (int i = 0; i < 3; ++i) {
        strides[i] = d[i].size == 1 ? (i ? strides[i - 1] * sizes[i] : row_bytes) : (cuuint64_t)d[i].stride;
        *d[i].place = i;
        if (d[i].place == &order->row) boxes[i + 1] = (cuuint32_t)box;
    }
    const CUresult r = encode(map, fp8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, pool.ptr, sizes,
                              strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? AA_OK : record_cuda_error(cudaErrorInvalidValue, "cuTensorMapEncodeTiled (strides of the page pools)");
}

// ---- attention: how a call is cut up
struct AttendPlan {
    int log2_page, rows, row_tiles, tiles8;       // tiles8: tiles of 8 rows one CTA holds (1 .. 4)
    int ctas, unit_keys;
    bool whole;                                   // ranges of whole entries
    bool split;                                   // an entry can be cut, and parts may have to be added up
    size_t o_off, ml_off, cut_off, bytes;
};

template <bool FP8, int RW>
cudaError_t allow_smem() {
    return cudaFuncSetAttribute(aa::paged::paged_attend_kernel<FP8, RW>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                aa::paged::kSmemBytes);
}

int plan_attend(const aa_paged_attend_t* a, AttendPlan& pl) {
    if (!a) return AA_ERR_NULL;
    const aa_paged_cache_t& c = a->cache;
    int rc = check_table(c, &pl.log2_page);
    if (rc) return rc;
    if (a->H <= 0 || a->H % c.Hkv || a->Nq <= 0) return AA_ERR_SHAPE;
    if (a->Nq > aa::paged::kMaxNew) return AA_ERR_NEW_TOKENS;
    if (a->pages && (a->list_width <= 0 || !a->page_counts)) return a->page_counts ? AA_ERR_SHAPE : AA_ERR_NULL;
    if (a->pages && (int64_t)a->list_width * c.page_size > (int64_t)1 << 30) return AA_ERR_TOO_LARGE;
    static thread_local Device dev;
    rc = current_device(dev, [] {
        for (cudaError_t e : {allow_smem<false, 1>(), allow_smem<false, 2>(), allow_smem<false, 3>(), allow_smem<false, 4>(),
                              allow_smem<true, 1>(), allow_smem<true, 2>(), allow_smem<true, 3>(), allow_smem<true, 4>()})
            if (e != cudaSuccess) return e;
        return cudaSuccess;
    });
    if (rc) return rc;
    if ((int64_t)a->Nq * (a->H / c.Hkv) > 1 << 16) return AA_ERR_NEW_TOKENS;
    pl.rows = a->Nq * (a->H / c.Hkv);
    // rows in as few tiles of up to 32 as there can be (each reads the cache), the tiles alike
    pl.row_tiles = (int)ceil_div(pl.rows, 32);
    pl.tiles8 = (int)ceil_div(ceil_div(pl.rows, pl.row_tiles), 8);
    const int64_t entries = (int64_t)c.B * c.Hkv * pl.row_tiles;
    const int64_t keys = (int64_t)(a->pages ? a->list_width : c.table_width) * c.page_size;
    const bool fp8 = c.cache_dtype == AA_E4M3;
    static const int unit_keys[2][4] = {
        {aa::paged::Shape<false, 1>::kUnitKeys, aa::paged::Shape<false, 2>::kUnitKeys, aa::paged::Shape<false, 3>::kUnitKeys,
         aa::paged::Shape<false, 4>::kUnitKeys},
        {aa::paged::Shape<true, 1>::kUnitKeys, aa::paged::Shape<true, 2>::kUnitKeys, aa::paged::Shape<true, 3>::kUnitKeys,
         aa::paged::Shape<true, 4>::kUnitKeys}};
    pl.unit_keys = unit_keys[fp8][pl.tiles8 - 1];
    const int64_t units = ceil_div(keys, pl.unit_keys);
    if (entries * units > 0x7FFFFFFF) return AA_ERR_TOO_LARGE;
    const int64_t most = (int64_t)dev.sms * aa::paged::kCtasPerSm;
    // Entries of few units stay whole: a CTA takes about 1 us a unit of 8 rows, the second kernel that would add up their parts
    // 2.3 us.  One sequence of up to 120 tokens, 8 heads: 6.7 us whole, 8.9 us cut; 16 sequences of up to 250: 9.1 and 10.8; but
    // one of 380 tokens (6 units): 10.9 and 8.8.
    pl.whole = units <= (pl.tiles8 == 1 && 2 * entries >= dev.sms ? 4 : 2);
    const int64_t pieces = pl.whole ? entries : entries * units;
    pl.ctas = (int)(pieces < most ? pieces : most);
    if (pl.ctas > 512) pl.ctas = 512;             // the kernel's 32-bit ranges
    pl.split = !pl.whole && pl.ctas > 1;
    const size_t parts = pl.split ? (size_t)pl.ctas * 2 * 8 * pl.tiles8 : 0;
    pl.o_off = 0;
    pl.ml_off = align256(parts * aa::kD * sizeof(float));
    pl.cut_off = align256(pl.ml_off + parts * sizeof(float2));
    pl.bytes = align256(pl.cut_off + pl.ctas * sizeof(int2));
    return AA_OK;
}

template <bool FP8, int RW>
int launch_attend(const CUtensorMap& k_map, const CUtensorMap& v_map, const aa::paged::AttendParams& p, const AttendPlan& pl,
                  cudaStream_t st) {
    cudaError_t e = launch_after(aa::paged::paged_attend_kernel<FP8, RW>, dim3(pl.ctas), dim3(aa::paged::Shape<FP8, RW>::kThreads),
                                 aa::paged::kSmemBytes, st, 1, k_map, v_map, p);
    if (e != cudaSuccess) return record_cuda_error(e, "launch paged_attend");
    if (!pl.split) return AA_OK;
    e = launch_after(aa::paged::paged_join_kernel<FP8>, dim3(pl.ctas - 1, 8 * RW < pl.rows ? 8 * RW : pl.rows),
                     dim3(aa::paged::kJoinThreads), 0, st, 1, p, 8 * RW);
    if (e != cudaSuccess) return record_cuda_error(e, "launch paged_join");
    return AA_OK;
}

template <bool FP8>
int launch_attend_rows(const CUtensorMap& km, const CUtensorMap& vm, const aa::paged::AttendParams& p, const AttendPlan& pl,
                       cudaStream_t st) {
    switch (pl.tiles8) {
        case 1: return launch_attend<FP8, 1>(km, vm, p, pl, st);
        case 2: return launch_attend<FP8, 2>(km, vm, p, pl, st);
        case 3: return launch_attend<FP8, 3>(km, vm, p, pl, st);
        default: return launch_attend<FP8, 4>(km, vm, p, pl, st);
    }
}

// wait_polls: after which a computing warp gives up on a copy
int run_attend(const aa_paged_attend_t* a, uint32_t wait_polls, void* stream) {
    AttendPlan pl;
    int rc = plan_attend(a, pl);
    if (rc) return rc;
    const aa_paged_cache_t& c = a->cache;
    rc = check_pools(c);
    if (rc) return rc;
    if (!a->q || !a->out) return AA_ERR_NULL;
    for (int64_t s : {a->q_stride_b, a->q_stride_n, a->q_stride_h, a->o_stride_b, a->o_stride_n, a->o_stride_h})
        if (bad_stride(s)) return AA_ERR_STRIDE;
    if (misaligned(a->q) || misaligned(a->out)) return AA_ERR_STRIDE;
    if (!a->workspace || ((uintptr_t)a->workspace & 255) || a->workspace_bytes < pl.bytes) return AA_ERR_WORKSPACE;

    aa::paged::AttendParams p;
    p.c = view(c, pl.log2_page);
    p.q = static_cast<const __nv_bfloat16*>(a->q);
    p.q_sb = a->q_stride_b; p.q_sn = a->q_stride_n; p.q_sh = a->q_stride_h;
    p.out = static_cast<__nv_bfloat16*>(a->out);
    p.o_sb = a->o_stride_b; p.o_sn = a->o_stride_n; p.o_sh = a->o_stride_h;
    p.lse = a->lse;
    p.pages = a->pages;
    p.page_counts = a->page_counts;
    p.list_width = a->list_width;
    p.B = c.B; p.H = a->H; p.Hkv = c.Hkv; p.Hg = a->H / c.Hkv; p.nq = a->Nq;
    p.rows = pl.rows;
    p.row_tiles = pl.row_tiles;
    p.whole = pl.whole;
    const double scale = a->sm_scale != 0.0 ? a->sm_scale : 1.0 / sqrt((double)c.D);
    p.scale_log2 = (float)(scale * 1.4426950408889634);
    uint8_t* ws = static_cast<uint8_t*>(a->workspace);
    p.part_o = reinterpret_cast<float*>(ws + pl.o_off);
    p.part_ml = reinterpret_cast<float2*>(ws + pl.ml_off);
    p.cuts = reinterpret_cast<int2*>(ws + pl.cut_off);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int box = c.page_size < pl.unit_keys ? c.page_size : pl.unit_keys;
    p.log2_box = 31 - __builtin_clz((unsigned)box);
    p.wait_polls = wait_polls;
    CUtensorMap k_map, v_map;
    rc = make_page_map(&k_map, p.c.k, c, box, &p.k_order);
    if (!rc) rc = make_page_map(&v_map, p.c.v, c, box, &p.v_order);
    if (rc) return rc;
    return c.cache_dtype == AA_E4M3 ? launch_attend_rows<true>(k_map, v_map, p, pl, st)
                                    : launch_attend_rows<false>(k_map, v_map, p, pl, st);
}

}  // namespace

extern "C" {

int aa_paged_check_status(uint32_t* status, void* stream) {
    if (!status) return AA_ERR_NULL;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    uint32_t word = 0;
    cudaError_t e = cudaMemcpyAsync(&word, status, sizeof(word), cudaMemcpyDeviceToHost, st);
    if (e != cudaSuccess) return record_cuda_error(e, "cudaMemcpyAsync(status)");
    e = cudaStreamSynchronize(st);
    if (e != cudaSuccess) return record_cuda_error(e, "cudaStreamSynchronize");
    // one kind a call: the bit that is reported is cleared, and no other
    for (const auto& [bit, code] : {std::pair{aa::paged::kStatusTimeout, AA_ERR_DEVICE_TIMEOUT},
                                    std::pair{aa::paged::kStatusBadPage, AA_ERR_BAD_PAGE},
                                    std::pair{aa::paged::kStatusTooLong, AA_ERR_TOO_LONG}}) {
        if (!(word & bit)) continue;
        aa::paged::clear_status_kernel<<<1, 1, 0, st>>>(status, bit);
        e = cudaGetLastError();
        return e == cudaSuccess ? (int)code : record_cuda_error(e, "launch clear_status");
    }
    return AA_OK;
}

int aa_paged_append(const aa_paged_append_t* a, void* stream) {
    if (!a) return AA_ERR_NULL;
    const aa_paged_cache_t& c = a->cache;
    int log2_page = 0;
    int rc = check_table(c, &log2_page);
    if (rc) return rc;
    rc = check_pools(c);
    if (rc) return rc;
    if (a->T <= 0 || a->H < 0 || (a->query && (a->H <= 0 || a->H % c.Hkv))) return AA_ERR_SHAPE;
    if (!a->cu_seqlens && a->T % c.B) return AA_ERR_SHAPE;
    if (!a->key || !a->value || (a->query && !a->query_out)) return AA_ERR_NULL;
    if (!a->cos != !a->sin || !a->key_codes != !a->key_code_scales) return AA_ERR_NULL;
    if (a->cos && a->rope_rows <= 0) return AA_ERR_SHAPE;
    for (int64_t s : {a->key_stride_t, a->key_stride_h, a->value_stride_t, a->value_stride_h, a->query_stride_t, a->query_stride_h,
                      a->query_out_stride_t, a->query_out_stride_h, a->key_out_stride_t, a->key_out_stride_h})
        if (bad_stride(s)) return AA_ERR_STRIDE;
    for (const void* p : {a->key, a->value, a->query, (const void*)a->query_out, (const void*)a->key_out, (const void*)a->cos,
                          (const void*)a->sin})
        if (misaligned(p)) return AA_ERR_STRIDE;

    aa::paged::AppendParams p;
    p.c = view(c, log2_page);
    auto rows = [](const void* ptr, int64_t token, int64_t head) {
        return aa::paged::Rows{static_cast<__nv_bfloat16*>(const_cast<void*>(ptr)), token, head};
    };
    p.key = rows(a->key, a->key_stride_t, a->key_stride_h);
    p.value = rows(a->value, a->value_stride_t, a->value_stride_h);
    p.query = rows(a->query, a->query_stride_t, a->query_stride_h);
    p.query_out = rows(a->query_out, a->query_out_stride_t, a->query_out_stride_h);
    p.key_out = rows(a->key_out, a->key_out_stride_t, a->key_out_stride_h);
    p.cu = a->cu_seqlens;
    p.cos = a->cos;
    p.sin = a->sin;
    p.rope_rows = a->rope_rows;
    p.codes = a->key_codes;
    p.code_scales = a->key_code_scales;
    p.T = a->T;
    p.B = c.B;
    p.H = a->H;
    p.Hkv = c.Hkv;
    p.per_seq = a->cu_seqlens ? 0 : a->T / c.B;
    // n tokens touch at most (n - 1) / page_size + 2 pages, one token one page
    int64_t tasks;
    if (a->cu_seqlens)
        tasks = a->T / c.page_size + 2 * (int64_t)c.B;
    else
        tasks = p.per_seq == 1 ? c.B : c.B * ((p.per_seq - 1) / c.page_size + (int64_t)2);
    if (tasks > 0x7FFFFFFF) return AA_ERR_TOO_LARGE;
    // one token a sequence: a block for every KV head and for every 64 query heads; more tokens: see paged_append.cuh
    const bool single = !a->cu_seqlens && p.per_seq == 1;
    p.kv_heads = single ? 1 : c.page_size < aa::paged::kStagedRows ? aa::paged::kStagedRows / c.page_size : 1;
    p.q_heads = single ? (a->H < 64 ? a->H : 64) : 4 * p.kv_heads;
    p.kv_blocks = (int)ceil_div(c.Hkv, p.kv_heads);
    p.staged = !single && c.page_size <= aa::paged::kStagedRows;
    const int64_t q_blocks = a->query ? ceil_div(a->H, p.q_heads) : 0;
    if (p.kv_blocks + q_blocks > 65535) return AA_ERR_TOO_LARGE;
    const dim3 grid((unsigned)tasks, (unsigned)(p.kv_blocks + q_blocks));
    const bool fp8 = c.cache_dtype == AA_E4M3;
    const size_t smem = p.staged && p.codes ? (size_t)aa::paged::kStagedRows * (fp8 ? 128 : 256) : 0;
    static thread_local Device dev;
    rc = current_device(dev, [] {
        const int most = aa::paged::kStagedRows * 256;
        const cudaError_t e = cudaFuncSetAttribute(aa::paged::paged_append_kernel<true, aa::paged::kAppendThreads>,
                                                   cudaFuncAttributeMaxDynamicSharedMemorySize, most);
        return e != cudaSuccess ? e
                                : cudaFuncSetAttribute(aa::paged::paged_append_kernel<false, aa::paged::kAppendThreads>,
                                                       cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    });
    if (rc) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    constexpr int kMany = aa::paged::kAppendThreads, kOne = aa::paged::kSingleThreads;
    cudaError_t e;
    if (single && fp8)
        e = launch_after(aa::paged::paged_append_kernel<true, kOne>, grid, dim3(kOne), 0, st, 1, p);
    else if (single)
        e = launch_after(aa::paged::paged_append_kernel<false, kOne>, grid, dim3(kOne), 0, st, 1, p);
    else if (fp8)
        e = launch_after(aa::paged::paged_append_kernel<true, kMany>, grid, dim3(kMany), smem, st, 1, p);
    else
        e = launch_after(aa::paged::paged_append_kernel<false, kMany>, grid, dim3(kMany), smem, st, 1, p);
    return e == cudaSuccess ? AA_OK : record_cuda_error(e, "launch paged_append");
}

int aa_paged_attend_workspace_bytes(const aa_paged_attend_t* a, size_t* bytes) {
    if (!bytes) return AA_ERR_NULL;
    AttendPlan pl;
    int rc = plan_attend(a, pl);
    if (rc) return rc;
    *bytes = pl.bytes;
    return AA_OK;
}

int aa_paged_attend(const aa_paged_attend_t* a, void* stream) { return run_attend(a, aa::tc::kSpinLimit, stream); }

int aa_selftest_paged_wait(const aa_paged_attend_t* a, void* stream) { return run_attend(a, 0, stream); }

int aa_page_select(const aa_page_select_t* a, void* stream) {
    if (!a) return AA_ERR_NULL;
    const aa_paged_cache_t& c = a->cache;
    int log2_page = 0;
    int rc = check_table(c, &log2_page);
    if (rc) return rc;
    if (a->H <= 0 || a->H % c.Hkv || a->Nq <= 0 || a->top <= 0) return AA_ERR_SHAPE;
    if (a->keep_first < 0 || a->keep_last < 1 || (int64_t)a->keep_first + a->keep_last > a->top) return AA_ERR_SHAPE;
    if (a->Nq > aa::paged::kMaxNew || (int64_t)a->Nq * (a->H / c.Hkv) > aa::paged::kMaxSelectRows) return AA_ERR_NEW_TOKENS;
    if (c.table_width > aa::paged::kMaxSelectPages) return AA_ERR_TOO_LARGE;
    if (!a->q || !a->key_codes || !a->key_code_scales || !a->out || !a->counts) return AA_ERR_NULL;
    for (int64_t s : {a->q_stride_b, a->q_stride_n, a->q_stride_h})
        if (bad_stride(s)) return AA_ERR_STRIDE;
    if (misaligned(a->q) || misaligned(a->key_codes)) return AA_ERR_STRIDE;
    static thread_local Device dev;
    rc = current_device(dev, [] {
        return cudaFuncSetAttribute(aa::paged::page_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    (int)aa::paged::select_smem_bytes(aa::paged::kMaxSelectRows, aa::paged::kMaxSelectPages));
    });
    if (rc) return rc;

    aa::paged::SelectParams p;
    p.c = view(c, log2_page);
    p.q = static_cast<const __nv_bfloat16*>(a->q);
    p.q_sb = a->q_stride_b; p.q_sn = a->q_stride_n; p.q_sh = a->q_stride_h;
    p.codes = a->key_codes;
    p.code_scales = a->key_code_scales;
    p.out = a->out;
    p.counts = a->counts;
    p.B = c.B; p.H = a->H; p.Hkv = c.Hkv; p.Hg = a->H / c.Hkv; p.nq = a->Nq;
    p.rows = a->Nq * p.Hg;
    p.top = a->top;
    p.keep_first = a->keep_first;
    p.keep_last = a->keep_last;
    const size_t smem = aa::paged::select_smem_bytes(p.rows, c.table_width);
    // Blocks for a sequence and head: more as long as they leave SMs idle and have pages for their warps.
    int cluster = 1;
    while (cluster < aa::paged::kMaxSelectCluster && (int64_t)c.B * c.Hkv * cluster < 2 * dev.sms &&
           c.table_width > cluster * aa::paged::kSelectWarps * 16)
        cluster *= 2;
    const cudaError_t e = launch_after(aa::paged::page_select_kernel, dim3((unsigned)(c.B * c.Hkv * cluster)),
                                       dim3(aa::paged::kSelectThreads), smem, static_cast<cudaStream_t>(stream), cluster, p, cluster);
    return e == cudaSuccess ? AA_OK : record_cuda_error(e, "launch page_select");
}

}  // extern "C"
