// C-ABI entry points of the stand-alone attention operators: whole packed prompts, and a cache held in 4 bits with what writes it, reads
// it back, attends to it and makes it shorter.  Device pointers in and out, nothing synchronised or allocated; scratch comes from the
// caller and may hold anything.
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include "../../include/lpp_b200.h"
#include "common.cuh"
#include "kv4.cuh"
#include "op_launch.cuh"
#include "prompt_attention.cuh"
#include "tensor_map.h"

using namespace lpp;

void lpp_internal_set_error(const char* msg);  // engine.cu: text behind lpp_last_error()

namespace {

lpp_status refuse(const char* what, lpp_status s = LPP_ERR_INVALID_ARG) {
    lpp_internal_set_error(what);
    return s;
}
lpp_status launched(const char* what, lpp_status s) { return s == LPP_OK ? s : refuse(what, s); }

int sm_count() {  // of the current device; 0: none
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
        (void)cudaGetLastError();
        return 0;
    }
    return sms;
}

// Calls f with a constant for the groups of a row (1 - 4 or 8; 5 - 7 groups are held as 8).
int kv4_held_groups(int head_size) {
    const int g = kv4_groups(head_size);
    return g > 4 ? 8 : g;
}
template <int N>
struct Int {
    static constexpr int value = N;
};
template <typename F>
lpp_status with_groups(int groups, F f) {
    switch (groups) {
        case 1: return f(Int<1>());
        case 2: return f(Int<2>());
        case 3: return f(Int<3>());
        case 4: return f(Int<4>());
        default: return f(Int<8>());
    }
}
template <typename F>
lpp_status with_type(int dtype, F f) {
    if (dtype == LPP_F16) return f((__half*)nullptr);
    if (dtype == LPP_BF16) return f((__nv_bfloat16*)nullptr);
    return f((float*)nullptr);
}
// The factor of a score in base 2, scale * log2(e); 0 where the scale has none: the product, too, is positive and finite.
constexpr float kLog2e = 1.4426950408889634f;
float rate_of(float scale) {
    const float rate = scale * kLog2e;
    return rate > 0.f && rate <= 3.402823466e38f ? rate : 0.f;
}
bool is_dtype(int dtype) { return dtype == LPP_F32 || dtype == LPP_F16 || dtype == LPP_BF16; }

// What every call on a 4-bit cache wants of it; NULL = nothing wrong.
const char* size_fault(int batch, int kv_heads, int64_t capacity, int head_size) {
    if (batch <= 0 || kv_heads <= 0 || capacity <= 0 || batch > 65535 || kv_heads > 65535) return "4-bit cache: sizes out of range";
    if (capacity % 4 || capacity > (1 << 30)) return "4-bit cache: the capacity is a multiple of 4, at most 2^30";
    if (head_size <= 0 || head_size > 256) return "4-bit cache: head sizes are 1 to 256";
    return nullptr;
}
const char* cache_fault(const void* k, const void* v, int batch, int kv_heads, int64_t capacity, int head_size) {
    if (!k || !v) return "4-bit cache: null pointer";
    if (((uintptr_t)k | (uintptr_t)v) & 15) return "4-bit cache: the caches start on a 16-byte boundary";
    return size_fault(batch, kv_heads, capacity, head_size);
}

// Shared by writing and reading rows.
template <typename Launch>
lpp_status rows_op(const char* name, const void* k, const void* v, const int64_t* slots, const void* kc, const void* vc, int n, int batch, int kv_heads, int64_t capacity,
                   int head_size, int64_t k_stride, int64_t v_stride, int dtype, Launch launch) {
    if (const char* f = cache_fault(kc, vc, batch, kv_heads, capacity, head_size)) return refuse(f);
    if (!is_dtype(dtype)) return refuse("4-bit cache: rows are F32, F16 or BF16");
    if (n < 0 || (long long)n * kv_heads > (1 << 27)) return refuse("4-bit cache: too many rows");
    if (n == 0) return LPP_OK;
    if (!k || !v || !slots) return refuse("4-bit cache: null pointer");
    const int element = dtype == LPP_F32 ? 4 : 2;
    if (((uintptr_t)k | (uintptr_t)v) & (element - 1) || (uintptr_t)slots & 7) return refuse("4-bit cache: a pointer is not aligned to its type");
    const int64_t dense = (int64_t)kv_heads * head_size;
    if (k_stride < dense || v_stride < dense) return refuse("4-bit cache: a token's rows overlap the next one's");
    // 16 bytes at once where every thread's dimensions start on such a boundary
    const bool wide = head_size % 16 == 0 && !(((uintptr_t)k | (uintptr_t)v) & 15) && k_stride * element % 16 == 0 && v_stride * element % 16 == 0;
    auto by = [](uint32_t d) { return Kv4Div{d, d > 1 ? (uint32_t)((1ull << 32) / d) : 0u}; };
    Kv4Cache c = {(unsigned char*)kc, (unsigned char*)vc, capacity, (long long)batch * capacity, kv_heads, by((uint32_t)kv_heads), by((uint32_t)capacity)};
    const int groups = kv4_held_groups(head_size), rows = n * kv_heads;
    const long long ctas = ((long long)rows * 2 * groups + kKv4RowThreads - 1) / kKv4RowThreads;
    return launched(name, launch(c, groups, dim3((unsigned)ctas, 2), rows, wide));
}

// ---- attention over the 4-bit cache: how the work is dealt out, and the scratch
struct AttnPlan {
    int cluster;  // CTAs of a head; 0: runs of all heads' units, as many as the SMs hold CTAs
    int runs;
    size_t whole, ml, part, scores, total;  // places in the scratch
};
AttnPlan attn_plan(int batch, int n_heads, int n_kv_heads, int64_t capacity, int head_size, bool sums, int sms) {
    const int groups = kv4_held_groups(head_size), head_tiles = (n_heads / n_kv_heads + kKv4Heads - 1) / kKv4Heads;
    const long long ctas = (long long)sms * (groups > 4 ? kKv4Ctas<8> : kKv4Ctas<4>), heads = (long long)batch * n_kv_heads * head_tiles;
    const long long units = (capacity + kKv4Unit - 1) / kKv4Unit;
    AttnPlan P = {};
    auto up = [](size_t n) { return (n + 255) & ~(size_t)255; };
    // a cluster a head where the cache is short and the clusters run at once (with sums: where one has all query heads)
    int cluster = 1;
    while (cluster < kKv4Cluster && cluster < units && 2 * cluster * heads <= ctas) cluster *= 2;
    if (units <= (long long)kKv4ClusterUnits * cluster && heads * cluster <= ctas && !(sums && head_tiles > 1)) {
        P.cluster = cluster;
    } else {
        P.runs = (int)std::min(ctas, heads * units);
        P.ml = up(sums ? (size_t)batch * n_heads * 8 : 0);
        P.part = P.ml + up((size_t)P.runs * 2 * kKv4Heads * 8);
        P.scores = P.part + up((size_t)P.runs * 2 * kKv4Heads * groups * 32 * 4);
    }
    P.total = P.scores + up(sums ? (size_t)batch * n_heads * capacity * 4 : 0);
    return P;
}
const char* attn_fault(int batch, int n_heads, int n_kv_heads, int64_t capacity, int head_size) {
    if (const char* f = size_fault(batch, n_kv_heads, capacity, head_size)) return f;
    if ((long long)batch * n_heads * (capacity / kKv4Unit + 1 + kKv4Head) > 0x7fffffffll) return "4-bit attention: more than 2^31 pieces of work";
    if (n_heads <= 0 || n_heads % n_kv_heads || n_heads / n_kv_heads > 1024) return "4-bit attention: the key/value heads divide the heads, at most 1024 to one";
    return nullptr;
}

}  // namespace

extern "C" {

lpp_status lpp_op_prompt_attention(void* d_out, const void* d_q, const void* d_k, const void* d_v, const int* d_offsets, int n_sequences, int n_tokens, int n_heads,
                                   int n_kv_heads, int head_size, int64_t out_stride, int64_t q_stride, int64_t k_stride, int64_t v_stride, float scale, int dtype, void* stream) {
    if (n_sequences < 0 || n_tokens < 0 || n_tokens > (1 << 30)) return refuse("prompt attention: sizes out of range");
    if (n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads || n_heads > 65535) return refuse("prompt attention: the key/value heads divide the heads");
    if (head_size <= 0 || head_size % 8 || head_size > 128) return refuse("prompt attention: head sizes are multiples of 8 up to 128");
    if (dtype != LPP_F16 && dtype != LPP_BF16) return refuse("prompt attention: F16 or BF16");
    if (rate_of(scale) == 0.f) return refuse("prompt attention: the scale is positive, and finite with a factor of log2(e)");
    if (n_sequences == 0 || n_tokens == 0) return LPP_OK;
    if (!d_out || !d_q || !d_k || !d_v || !d_offsets) return refuse("prompt attention: null pointer");
    if (((uintptr_t)d_out | (uintptr_t)d_q | (uintptr_t)d_k | (uintptr_t)d_v) & 15 || (uintptr_t)d_offsets & 3)
        return refuse("prompt attention: queries, keys, values and results start on 16-byte boundaries");
    const int64_t rows = (int64_t)n_heads * head_size, kv_rows = (int64_t)n_kv_heads * head_size;
    if (out_stride < rows || q_stride < rows || k_stride < kv_rows || v_stride < kv_rows || (out_stride | q_stride | k_stride | v_stride) % 8 ||
        std::max(std::max(out_stride, q_stride), std::max(k_stride, v_stride)) > (1ll << 32))
        return refuse("prompt attention: a token's heads fit its stride, a multiple of 8 elements");
    const encode_tiled_fn encode = tensor_map_encoder();
    if (!encode) return refuse("prompt attention: no CUDA device, or cuTensorMapEncodeTiled is not available from this driver", LPP_ERR_NO_DEVICE);
    CUtensorMap q_map, k_map, v_map;
    auto make = [&](CUtensorMap* m, const void* p, int heads, int64_t stride) {  // 128 tokens x 64 dimensions of a head a copy
        const cuuint64_t dims[3] = {(cuuint64_t)head_size, (cuuint64_t)heads, (cuuint64_t)n_tokens};
        const cuuint64_t strides[2] = {(cuuint64_t)head_size * 2, (cuuint64_t)stride * 2};
        const cuuint32_t box[3] = {64u, 1u, (cuuint32_t)kPaRows}, estr[3] = {1, 1, 1};
        return encode(m, dtype == LPP_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(p), dims, strides, box, estr,
                      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    };
    if (!make(&q_map, d_q, n_heads, q_stride) || !make(&k_map, d_k, n_kv_heads, k_stride) || !make(&v_map, d_v, n_kv_heads, v_stride))
        return refuse("prompt attention: cuTensorMapEncodeTiled failed", LPP_ERR_CUDA);
    PromptAttnArgs a = {};
    a.out = d_out;
    a.v = d_v;
    a.offsets = d_offsets;
    a.out_stride = out_stride;
    a.v_stride = v_stride;
    a.n_sequences = n_sequences;
    a.n_tokens = n_tokens;
    a.heads = n_heads;
    a.gqa = n_heads / n_kv_heads;
    a.head_size = head_size;
    auto go = [&](auto shape, auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        constexpr int HS = shape.value;
        using Shape = PaShape<HS>;
        a.pair_heads = Shape::kTiles == 2 && a.gqa % 2 == 0;
        const int cta_rows = a.pair_heads ? kPaRows : Shape::kTiles * kPaRows, per_tile = a.pair_heads ? n_heads / 2 : n_heads;
        a.tiles = (n_tokens + cta_rows - 1) / cta_rows;
        a.rate = rate_of(scale);
        if ((long long)a.tiles * per_tile > 0x7fffffffll) return LPP_ERR_TOO_LARGE;
        if (!allow_smem<prompt_attention_kernel<HS, T>>(Shape::kSmem)) return LPP_ERR_CUDA;
        return launch_op(prompt_attention_kernel<HS, T>, dim3(a.tiles * per_tile), Shape::kThreads, Shape::kSmem, S(stream), q_map, k_map, v_map, a);
    };
    auto by_type = [&](auto shape) { return dtype == LPP_F16 ? go(shape, (__half*)nullptr) : go(shape, (__nv_bfloat16*)nullptr); };
    return launched("lpp_op_prompt_attention: too many tokens, or the launch failed", head_size <= 64 ? by_type(Int<64>()) : by_type(Int<128>()));
}

int64_t lpp_op_kv4_row_bytes(int head_size) { return head_size <= 0 || head_size > 256 ? -1 : kv4_row_bytes(kv4_held_groups(head_size)); }

lpp_status lpp_op_kv4_write(void* d_k_cache, void* d_v_cache, const void* d_k, const void* d_v, const int64_t* d_slots, int n_tokens, int batch, int n_kv_heads,
                            int64_t capacity, int head_size, int64_t k_stride, int64_t v_stride, int dtype, void* stream) {
    return rows_op("lpp_op_kv4_write: the launch failed", d_k, d_v, d_slots, d_k_cache, d_v_cache, n_tokens, batch, n_kv_heads, capacity, head_size, k_stride, v_stride, dtype,
                   [&](const Kv4Cache& c, int groups, dim3 grid, int rows, bool wide) {
                       return with_groups(groups, [&](auto ng) {
                           return with_type(dtype, [&](auto* t) {
                               using T = std::remove_pointer_t<decltype(t)>;
                               return launch_op(wide ? kv4_write_kernel<T, ng.value, true> : kv4_write_kernel<T, ng.value, false>, grid, kKv4RowThreads, 0, S(stream), c, (const T*)d_k, (const T*)d_v, (const long long*)d_slots,
                                                rows, head_size, (long long)k_stride, (long long)v_stride);
                           });
                       });
                   });
}

lpp_status lpp_op_kv4_read(void* d_k, void* d_v, const void* d_k_cache, const void* d_v_cache, const int64_t* d_slots, int n_tokens, int batch, int n_kv_heads,
                           int64_t capacity, int head_size, int64_t k_stride, int64_t v_stride, int dtype, void* stream) {
    return rows_op("lpp_op_kv4_read: the launch failed", d_k, d_v, d_slots, d_k_cache, d_v_cache, n_tokens, batch, n_kv_heads, capacity, head_size, k_stride, v_stride, dtype,
                   [&](const Kv4Cache& c, int groups, dim3 grid, int rows, bool wide) {
                       return with_groups(groups, [&](auto ng) {
                           return with_type(dtype, [&](auto* t) {
                               using T = std::remove_pointer_t<decltype(t)>;
                               return launch_op(wide ? kv4_read_kernel<T, ng.value, true> : kv4_read_kernel<T, ng.value, false>, grid, kKv4RowThreads, 0, S(stream), c, (T*)d_k, (T*)d_v, (const long long*)d_slots, rows, head_size,
                                                (long long)k_stride, (long long)v_stride);
                           });
                       });
                   });
}

int64_t lpp_op_kv4_attention_scratch_bytes(int batch, int n_heads, int n_kv_heads, int64_t capacity, int head_size, int with_sums) {
    const int sms = sm_count();
    if (sms <= 0 || attn_fault(batch, n_heads, n_kv_heads, capacity, head_size)) return -1;
    return (int64_t)attn_plan(batch, n_heads, n_kv_heads, capacity, head_size, with_sums != 0, sms).total;
}

lpp_status lpp_op_kv4_attention(void* scratch, int64_t scratch_bytes, void* d_out, const void* d_q, const void* d_k_cache, const void* d_v_cache, const int* d_lens,
                                const float* d_sums_in, float* d_sums_out, float scale, int batch, int n_heads, int n_kv_heads, int64_t capacity, int head_size,
                                int64_t out_stride, int64_t q_stride, int dtype, void* stream) {
    if (const char* f = cache_fault(d_k_cache, d_v_cache, batch, n_kv_heads, capacity, head_size)) return refuse(f);
    if (const char* f = attn_fault(batch, n_heads, n_kv_heads, capacity, head_size)) return refuse(f);
    if (((uintptr_t)scratch & 255) || !d_out || !d_q || !d_lens) return refuse("4-bit attention: null pointer, or scratch not on a 256-byte boundary");
    if (!is_dtype(dtype)) return refuse("4-bit attention: queries are F32, F16 or BF16");
    const int element = dtype == LPP_F32 ? 4 : 2;
    if (((uintptr_t)d_out | (uintptr_t)d_q) & (element - 1) || ((uintptr_t)d_lens | (uintptr_t)d_sums_in | (uintptr_t)d_sums_out) & 3)
        return refuse("4-bit attention: a pointer is not aligned to its type");
    if (out_stride < (int64_t)n_heads * head_size || q_stride < (int64_t)n_heads * head_size) return refuse("4-bit attention: a sequence's heads overlap the next one's");
    if (rate_of(scale) == 0.f) return refuse("4-bit attention: the scale is positive, and finite with a factor of log2(e)");
    if (d_sums_in && !d_sums_out) return refuse("4-bit attention: sums go in but not out");
    const int sms = sm_count();
    if (sms <= 0) return refuse("4-bit attention: no CUDA device", LPP_ERR_NO_DEVICE);
    const int groups = kv4_held_groups(head_size);
    const AttnPlan P = attn_plan(batch, n_heads, n_kv_heads, capacity, head_size, d_sums_out != nullptr, sms);
    if (scratch_bytes < (int64_t)P.total || (!scratch && P.total)) return refuse("4-bit attention: scratch is smaller than lpp_op_kv4_attention_scratch_bytes() says");
    char* w = (char*)scratch;
    Kv4AttnArgs a = {};
    a.k = (const unsigned char*)d_k_cache;
    a.v = (const unsigned char*)d_v_cache;
    a.q = d_q;
    a.out = d_out;
    a.lens = d_lens;
    a.sums_in = d_sums_in;
    a.sums_out = d_sums_out;
    a.scores = d_sums_out ? (float*)(w + P.scores) : nullptr;
    a.whole_ml = d_sums_out ? (float2*)(w + P.whole) : nullptr;
    a.part_ml = (float2*)(w + P.ml);
    a.part_o = (float*)(w + P.part);
    a.capacity = capacity;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.batch = batch;
    a.heads = n_heads;
    a.kv_heads = n_kv_heads;
    a.gqa = n_heads / n_kv_heads;
    a.head_size = head_size;
    a.head_tiles = (a.gqa + kKv4Heads - 1) / kKv4Heads;
    a.runs = P.runs;
    a.cluster = P.cluster;
    a.dtype = dtype;
    a.rate = rate_of(scale);
    return launched("lpp_op_kv4_attention: the launch failed", with_groups(groups, [&](auto ng) {
                        constexpr int NG = ng.value;
                        const int sums = kv4_sums_bytes<NG>(std::min(a.gqa, kKv4Heads));
                        // as many units in flight as the shared memory holds beside the warps' sums; a short cache has no more
                        auto go = [&](auto parts, auto clusters) {
                            constexpr bool split = parts.value == 2;
                            constexpr auto kernel = kv4_attn_kernel<NG, split, clusters.value == 1>;
                            constexpr int most = (227 * 1024) / kKv4Ctas<NG> - 1024 * (NG + 2) - (split ? 512 * NG : 0);  // shared memory of a CTA beside its fixed arrays
                            a.stages = std::min(clusters.value ? kKv4ClusterUnits : kKv4MaxStages, (most - sums) / kKv4StageBytes<NG>);
                            const int smem = a.stages * kKv4StageBytes<NG> + sums;
                            if (!allow_smem<kernel>(most)) return LPP_ERR_CUDA;
                            return launch_op_cluster(kernel, dim3(clusters.value ? P.cluster * batch * n_kv_heads * a.head_tiles : P.runs), kKv4Threads, smem,
                                                     clusters.value ? P.cluster : 1, false, S(stream), a);
                        };
                        if (P.cluster) return dtype == LPP_F32 ? go(Int<2>(), Int<1>()) : go(Int<1>(), Int<1>());
                        const lpp_status st = dtype == LPP_F32 ? go(Int<2>(), Int<0>()) : go(Int<1>(), Int<0>());
                        if (st != LPP_OK) return st;
                        const long long rows = d_sums_out ? (capacity + kKv4FinishRows - 1) / kKv4FinishRows : 0;
                        return launch_behind(kv4_finish_kernel<NG>, dim3((unsigned)(a.gqa + rows), n_kv_heads, batch), kKv4FinishThreads, (size_t)(2 * a.gqa + P.runs) * 4, S(stream), a);
                    }));
}

lpp_status lpp_op_kv4_evict(void* d_k_out, void* d_v_out, float* d_sums_out, int* d_kept, int* d_lens_out, const void* d_k_cache, const void* d_v_cache, const float* d_sums,
                            const int* d_lens, int batch, int n_kv_heads, int64_t capacity, int64_t capacity_out, int head_size, int keep, int recent, void* stream) {
    if (const char* f = cache_fault(d_k_cache, d_v_cache, batch, n_kv_heads, capacity, head_size)) return refuse(f);
    if (const char* f = cache_fault(d_k_out, d_v_out, batch, n_kv_heads, capacity_out, head_size)) return refuse(f);
    if (!d_sums_out || !d_kept || !d_lens_out || !d_sums || !d_lens) return refuse("eviction: null pointer");
    if (((uintptr_t)d_sums_out | (uintptr_t)d_kept | (uintptr_t)d_lens_out | (uintptr_t)d_sums | (uintptr_t)d_lens) & 3) return refuse("eviction: a pointer is not aligned to its type");
    if (keep <= 0 || keep > capacity_out || recent < 0 || recent > keep) return refuse("eviction: 0 <= recent <= keep <= capacity of the new cache, keep > 0");
    // rows move to other places, and are listed, while sums and other rows are read: what is written overlaps nothing else
    const int row = kv4_row_bytes(kv4_held_groups(head_size));
    const size_t heads = (size_t)batch * n_kv_heads, in = heads * capacity, out = heads * capacity_out;
    struct Range {
        const void* at;
        size_t bytes;
    };
    const Range ranges[] = {{d_k_out, out * row},  {d_v_out, out * row}, {d_sums_out, out * 4}, {d_kept, heads * keep * 4}, {d_lens_out, (size_t)batch * 4},  // written
                            {d_k_cache, in * row}, {d_v_cache, in * row}, {d_sums, in * 4},     {d_lens, (size_t)batch * 4}};
    for (int w = 0; w < 5; ++w)
        for (int r = w + 1; r < 9; ++r) {
            const uintptr_t x = (uintptr_t)ranges[w].at, y = (uintptr_t)ranges[r].at;
            if (x + ranges[w].bytes > y && y + ranges[r].bytes > x) return refuse("eviction: a result overlaps another one, or what is read");
        }
    const int sms = sm_count();
    if (sms <= 0) return refuse("eviction: no CUDA device", LPP_ERR_NO_DEVICE);
    Kv4EvictArgs a = {};
    a.k = (const unsigned char*)d_k_cache;
    a.v = (const unsigned char*)d_v_cache;
    a.k_out = (unsigned char*)d_k_out;
    a.v_out = (unsigned char*)d_v_out;
    a.sums = d_sums;
    a.sums_out = d_sums_out;
    a.kept = d_kept;
    a.lens_out = d_lens_out;
    a.lens = d_lens;
    a.capacity = capacity;
    a.capacity_out = capacity_out;
    a.kv_heads = n_kv_heads;
    a.keep = keep;
    a.recent = recent;
    a.row_bytes = row;
    // CTAs of a head: up to eight (a portable cluster), while they all run at once and have some hundred rows each
    a.cluster = 1;
    while (a.cluster < kKv4EvictCluster && 2ll * a.cluster * (long long)heads <= sms && capacity >= 1024ll * a.cluster) a.cluster *= 2;
    const bool few = keep <= kKv4EvictMove * a.cluster;
    lpp_status st = launch_op_cluster(few ? kv4_select_kernel<true> : kv4_select_kernel<false>, dim3(a.cluster, n_kv_heads, batch), kKv4EvictThreads, 0, a.cluster, false, S(stream), a);
    if (few || st != LPP_OK) return launched("lpp_op_kv4_evict: the launch failed", st);
    const dim3 grid(blocks(std::min<int64_t>(keep, capacity), kKv4MoveRows), n_kv_heads, batch);
    auto move = [&](auto kernel) { return launch_behind(kernel, grid, kKv4MoveRows, 0, S(stream), a); };
    switch (row / 20) {  // groups of a row
        case 1: st = move(kv4_move_kernel<uint32_t, 5>); break;
        case 2: st = move(kv4_move_kernel<uint2, 5>); break;
        case 3: st = move(kv4_move_kernel<uint32_t, 15>); break;
        case 4: st = move(kv4_move_kernel<uint4, 5>); break;
        default: st = move(kv4_move_kernel<uint4, 10>);
    }
    return launched("lpp_op_kv4_evict: the launch failed", st);
}

lpp_status lpp_op_call(int op, const void* words, int n_words, void* stream) {
    static const int count[] = {16, 13, 13, 18, 16};
    if (op < 0 || op > LPP_OP_KV4_EVICT || !words || n_words != count[op]) return refuse("lpp_op_call: no such operator, or another number of arguments");
    int64_t w[18];
    memcpy(w, words, (size_t)n_words * 8);
    auto ptr = [&](int i) { return (void*)(uintptr_t)w[i]; };
    bool fits = true;
    auto num = [&](int i) {
        fits = fits && w[i] >= INT32_MIN && w[i] <= INT32_MAX;
        return (int)w[i];
    };
    auto real = [&](int i) {
        double d;
        memcpy(&d, &w[i], 8);
        return (float)d;
    };
    // (the numbers are looked at before the call: arguments of one are evaluated in no order)
    static const unsigned numbers[] = {0x83e0u, 0x12e0u, 0x12e0u, 0x25c00u, 0xe600u};
    for (int i = 0; i < n_words; ++i)
        if (numbers[op] >> i & 1u) num(i);
    if (!fits) return refuse("lpp_op_call: a number does not fit 32 bits");
    switch (op) {
        case LPP_OP_PROMPT_ATTENTION:
            return lpp_op_prompt_attention(ptr(0), ptr(1), ptr(2), ptr(3), (const int*)ptr(4), num(5), num(6), num(7), num(8), num(9), w[10], w[11], w[12], w[13], real(14), num(15),
                                           stream);
        case LPP_OP_KV4_WRITE:
            return lpp_op_kv4_write(ptr(0), ptr(1), ptr(2), ptr(3), (const int64_t*)ptr(4), num(5), num(6), num(7), w[8], num(9), w[10], w[11], num(12), stream);
        case LPP_OP_KV4_READ:
            return lpp_op_kv4_read(ptr(0), ptr(1), ptr(2), ptr(3), (const int64_t*)ptr(4), num(5), num(6), num(7), w[8], num(9), w[10], w[11], num(12), stream);
        case LPP_OP_KV4_ATTENTION:
            return lpp_op_kv4_attention(ptr(0), w[1], ptr(2), ptr(3), ptr(4), ptr(5), (const int*)ptr(6), (const float*)ptr(7), (float*)ptr(8), real(9), num(10), num(11), num(12), w[13],
                                        num(14), w[15], w[16], num(17), stream);
        default:
            return lpp_op_kv4_evict(ptr(0), ptr(1), (float*)ptr(2), (int*)ptr(3), (int*)ptr(4), ptr(5), ptr(6), (const float*)ptr(7), (const int*)ptr(8), num(9), num(10), w[11], w[12],
                                    num(13), num(14), num(15), stream);
    }
}

}  // extern "C"
