// Causal attention of whole prompts, packed one behind the other, with grouped query heads (the reference runs a prompt token by token
// through src/model.cpp:178-199): out_i = sum_j softmax_j(scale q_i . k_j) v_j over the tokens j <= i of i's own sequence.
//
// A CTA takes two tiles of 128 query rows that read the same keys and values: the same 128 tokens of two heads that share a
// key/value head (or 256 tokens of one head where heads do not pair up).  Per tile of 128 keys and row tile one tcgen05.mma chain
// forms the scores S = Q . K^T in tensor memory; a warpgroup, one thread a row, takes the row into registers, forms the
// probabilities and writes them back over the scores as the 16-bit operand of the second chain, O += P . V, whose sums stay in tensor
// memory.  The two row tiles take turns: while one's rows are exponentiated the tensor cores work for the other.
//     tensor memory columns: S/P of tile 0 | S/P of tile 1 | O of tile 0 | O of tile 1, 128 each
// Sums O are rescaled only when a row's maximum has grown by more than 2^8 since it was last set: they are complete whenever the
// scores of the next key tile are (the tensor cores work in order), so the row's own thread does it.
//
// Sequences do not have to begin at tiles: row tiles cover the packed tokens whatever the borders, a row sees the keys from its
// sequence's start to itself, and a tile runs over the keys from its first row's sequence on.  Many short prompts share a tile.
//
// Keys of tokens that a row does not see are masked after the product; their values meet probabilities of 0, which hides everything but
// NaN and infinity.  So a warp looks through the value tiles that some row sees only in part, zeroes what is not finite, and the rows
// that do see it get it added to their results at the end.
#pragma once
#include "common.cuh"
#include "umma.cuh"

namespace lpp {

constexpr int kPaRows = 128, kPaKeys = 128, kPaSub = 128 * 128;  // kPaSub: bytes of 128 rows x 64 columns
constexpr int kPaSoftWarps = 8, kPaMmaWarp = 8, kPaLoadWarp = 9, kPaCheckWarp = 10, kPaCheckWarps = 2, kPaThreads = 12 * 32;
// Registers: 384 threads start with 168 each; the two softmax warpgroups take what the third gives back (2 x 128 x 56 = 128 x 112)
constexpr int kPaSoftRegs = 224, kPaOtherRegs = 56;
static_assert(2 * 128 * kPaSoftRegs + 128 * kPaOtherRegs <= 384 * 168, "a split must not ask for more registers than the block was launched with");
template <int HS>
constexpr int kPaTileBytes = HS / 64 * kPaSub;
template <int HS>
constexpr int kPaSmem = 1024 /*alignment*/ + 6 * kPaTileBytes<HS>;  // 2 x Q, 2 x K, 2 x V
constexpr float kPaGrowth = 8.f;  // of a row's maximum (base 2) before its sums are rescaled

struct PromptAttnArgs {
    void* out;
    const void* v;        // for rows that see a value that is not finite
    const int* offsets;   // [sequences + 1]
    long long out_stride, v_stride;
    int n_sequences, n_tokens, heads, gqa, head_size, pair_heads, tiles;
    float rate;           // scale * log2(e)
};

// Operand whose rows run along K (V as it lies in memory): 1024 bytes between groups of eight K rows, kPaSub between blocks of 64 columns
__device__ __forceinline__ uint64_t pa_desc_v(uint32_t smem_addr) {
    return (uint64_t)((smem_addr & 0x3ffffu) >> 4) | ((uint64_t)(kPaSub >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
template <typename T>
__host__ __device__ constexpr uint32_t pa_idesc(int n, bool b_mn_major) {  // FP32 sums, M = 128
    return (1u << 4) | (std::is_same<T, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u) | (b_mn_major ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(128 >> 4) << 24);
}
// D (tensor memory) += A (tensor memory, 16-bit pairs along K) . B (shared memory)
__device__ __forceinline__ void tc_mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d_tmem), "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// As tc_ld32 without the wait
__device__ __forceinline__ void tc_ld32_async(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// The registers of a load that has been waited for: nothing that uses them moves ahead of this
__device__ __forceinline__ void pin16(uint32_t* r) {
    asm volatile(""
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                   "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]));
}
__device__ __forceinline__ void tc_st32(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};"
        ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
        "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]),
        "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
        : "memory");
}
template <int N>
__device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// Two FP32 values in one instruction
__device__ __forceinline__ uint64_t f2_pack(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float2 f2_unpack(uint64_t x) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
    return r;
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// 2^x of two values on the FMA pipe, relative error 2^-13.7 (BF16 probabilities) or 2^-18.5 (FP16): x = n + f with n the nearest integer (by
// adding 1.5 2^23), a minimax polynomial for 2^f on [-1/2, 1/2] (Remez exchange for the relative error), n added to the exponent.  Below
// 2^-126: 2^-126.
template <typename T>
__device__ __forceinline__ float2 pa_exp2_poly(uint64_t x2) {
    float2 x = f2_unpack(x2);
    x2 = f2_pack(fmaxf(x.x, -126.f), fmaxf(x.y, -126.f));
    const uint64_t magic = f2_pack(12582912.f, 12582912.f), back = f2_pack(-12582912.f, -12582912.f), minus = f2_pack(-1.f, -1.f);
    const uint64_t t = f2_add(x2, magic), f = f2_fma(f2_add(t, back), minus, x2);
    uint64_t y;
    if constexpr (std::is_same<T, __half>::value) {
        y = f2_fma(f2_pack(0.009570102207362652f, 0.009570102207362652f), f, f2_pack(0.05591785907745361f, 0.05591785907745361f));
        y = f2_fma(y, f, f2_pack(0.240247443318367f, 0.240247443318367f));
        y = f2_fma(y, f, f2_pack(0.6931217908859253f, 0.6931217908859253f));
        y = f2_fma(y, f, f2_pack(0.9999992847442627f, 0.9999992847442627f));
    } else {
        y = f2_fma(f2_pack(0.0551716685295105f, 0.0551716685295105f), f, f2_pack(0.2426111251115799f, 0.2426111251115799f));
        y = f2_fma(y, f, f2_pack(0.6932609677314758f, 0.6932609677314758f));
        y = f2_fma(y, f, f2_pack(0.9999280571937561f, 0.9999280571937561f));
    }
    const float2 n = f2_unpack(t), v = f2_unpack(y);
    return make_float2(__int_as_float(__float_as_int(v.x) + (__float_as_int(n.x) << 23)), __int_as_float(__float_as_int(v.y) + (__float_as_int(n.y) << 23)));
}
__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float pa_exp2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// First token of the sequence that token i lies in (offsets[0] = 0 <= offsets[1] <= ...; equal ones are empty sequences)
__device__ __forceinline__ int pa_start(const int* offsets, int n, int i) {
    int lo = 0, hi = n;  // offsets[lo] <= i < offsets[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (offsets[mid] <= i)
            lo = mid;
        else
            hi = mid;
    }
    return max(0, min(offsets[lo], i));
}
constexpr int kPaOffsets = 1024;  // sequences whose offsets are searched in shared memory

template <int HS, typename T>
static __global__ void __launch_bounds__(kPaThreads, 1) prompt_attention_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                                                                                const __grid_constant__ CUtensorMap v_map, const PromptAttnArgs a) {
    constexpr int kPieces = HS / 64, kTile = kPaTileBytes<HS>;
    // FP16 probabilities stay clear of the subnormals: they are 2^(x - m + 6) at most 2^14
    constexpr float kLift = std::is_same<T, __half>::value ? 6.f : 0.f;
    constexpr int kPoly = HS == 64 ? 6 : 0;  // of 16 exponentials, how many on the FMA pipe
    // Head sizes up to 64 leave room for probabilities beside the scores: the next scores are formed while these are exponentiated.
    constexpr bool kApart = HS == 64;
    constexpr uint32_t kO = 256, kOWide = HS, kP = kApart ? 384 : 0, kPWide = kApart ? 64 : 128;  // columns of the sums and the probabilities
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], v_clean[2], s_full[2], s_read[2], p_ready[2], o_done[2];
    __shared__ uint32_t tmem_slot;
    __shared__ int s_fail, s_odd, s_start[2 * kPaRows], s_off[kPaOffsets + 1];
    const uint32_t base = (smem_u32(smem) + 1023u) & ~1023u;
    const uint32_t sq = base, sk = sq + 2 * kTile, sv = sk + 2 * kTile;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const int per_tile = a.pair_heads ? a.heads / 2 : a.heads;
    const int work = blockIdx.x, tile = a.tiles - 1 - work / per_tile, unit = work - (work / per_tile) * per_tile;
    const int cta_rows = a.pair_heads ? kPaRows : 2 * kPaRows, t0 = tile * cta_rows;
    const int head0 = a.pair_heads ? 2 * unit : unit, kvh = head0 / a.gqa;
    if (tid == 0) {
        tma_prefetch_map(&q_map);
        tma_prefetch_map(&k_map);
        tma_prefetch_map(&v_map);
    }
    pdl_wait();
    const bool few = a.n_sequences <= kPaOffsets;
    if (few)
        for (int i = tid; i <= a.n_sequences; i += kPaThreads) s_off[i] = a.offsets[i];
    const int total = min(a.offsets[a.n_sequences], a.n_tokens);
    if (t0 >= total) return;
    const int t_end = min(total, t0 + cta_rows);
    if (tid == 0) {
        s_fail = 0;
        s_odd = 0;
        mbar_init(&q_full, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&k_full[i], 1);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_full[i], 1);
            mbar_init(&v_empty[i], 1);
            mbar_init(&v_clean[i], kPaCheckWarps);
            mbar_init(&s_read[i], 4);
            mbar_init(&s_full[i], 1);
            mbar_init(&p_ready[i], 4);
            mbar_init(&o_done[i], 1);
        }
        mbar_fence_init();
    }
    if (warp == kPaMmaWarp) {
        tc_alloc(&tmem_slot, 512);
        tc_relinquish();
    }
    __syncthreads();
    if (tid < cta_rows) s_start[tid] = pa_start(few ? s_off : a.offsets, a.n_sequences, min(t0 + tid, t_end - 1));
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&tmem_slot);
    pdl_launch_dependents();
    const int k0 = s_start[0], n_tiles = (t_end - 1 - k0) / kPaKeys + 1, last_start = s_start[t_end - 1 - t0];
    // some row of the CTA sees only a part of key tile `it`
    auto partial = [&](int it) { return k0 + it * kPaKeys < last_start || k0 + it * kPaKeys + kPaKeys - 1 > t0; };

    if (warp >= kPaSoftWarps) {
    regs_down<kPaOtherRegs>();
    if (warp == kPaLoadWarp) {
        if (lane == 0) {
            bool ok = true;
            mbar_arrive_expect_tx(&q_full, 2 * kTile);
            for (int x = 0; x < 2; ++x)
                for (int p = 0; p < kPieces; ++p)
                    tma_load_3d(sq + x * kTile + p * kPaSub, &q_map, p * 64, a.pair_heads ? head0 + x : head0, t0 + (a.pair_heads ? 0 : x * kPaRows), smem_u32(&q_full));
            for (int it = 0; it < n_tiles && ok; ++it) {
                const int b = it & 1;
                const uint32_t par = (uint32_t)((it >> 1) - 1) & 1u;
                ok = it < 2 || mbar_wait_bounded(&k_empty[b], par, nullptr);
                if (!ok) break;
                mbar_arrive_expect_tx(&k_full[b], kTile);
                for (int p = 0; p < kPieces; ++p) tma_load_3d(sk + b * kTile + p * kPaSub, &k_map, p * 64, kvh, k0 + it * kPaKeys, smem_u32(&k_full[b]));
                ok = it < 2 || mbar_wait_bounded(&v_empty[b], par, nullptr);
                if (!ok) break;
                mbar_arrive_expect_tx(&v_full[b], kTile);
                for (int p = 0; p < kPieces; ++p) tma_load_3d(sv + b * kTile + p * kPaSub, &v_map, p * 64, kvh, k0 + it * kPaKeys, smem_u32(&v_full[b]));
            }
            if (!ok) s_fail = 1;
        }
    } else if (warp == kPaMmaWarp) {
        auto scores = [&](int x, int it) {
            if (elect_one()) {
#pragma unroll
                for (int ks = 0; ks < HS / 16; ++ks) {
                    const uint32_t off = (uint32_t)((ks >> 2) * kPaSub + (ks & 3) * 32);
                    tc_mma_f16(tmem + x * 128, umma_desc(sq + x * kTile + off), umma_desc(sk + (it & 1) * kTile + off), pa_idesc<T>(kPaKeys, false), ks > 0 ? 1u : 0u);
                }
                tc_commit(&s_full[x]);
                if (x == 1) tc_commit(&k_empty[it & 1]);
            }
            __syncwarp();
        };
        auto wait = [](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, nullptr)) != 0; };
        bool ok = wait(&q_full, 0) && wait(&k_full[0], 0);
        if (ok) {
            tc_fence_after();
            scores(0, 0);
            scores(1, 0);
        }
        for (int it = 0; it < n_tiles && ok; ++it) {
            const int b = it & 1;
            const bool more = it + 1 < n_tiles;
            if (more) ok = wait(&k_full[b ^ 1], (uint32_t)((it + 1) >> 1) & 1u);
            if constexpr (kApart) {
                for (int x = 0; x < 2 && ok && more; ++x) {  // these have been taken into registers: their place takes the next
                    ok = wait(&s_read[x], (uint32_t)it & 1u);
                    if (!ok) break;
                    tc_fence_after();
                    scores(x, it + 1);
                }
            }
            ok = ok && wait(&v_full[b], (uint32_t)(it >> 1) & 1u) && wait(&v_clean[b], (uint32_t)(it >> 1) & 1u);
            for (int x = 0; x < 2 && ok; ++x) {
                ok = wait(&p_ready[x], (uint32_t)it & 1u);
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) {
#pragma unroll
                    for (int ks = 0; ks < kPaKeys / 16; ++ks)
                        tc_mma_f16_ts(tmem + kO + x * kOWide, tmem + kP + x * kPWide + ks * 8, pa_desc_v(sv + b * kTile + ks * 2048), pa_idesc<T>(HS, true),
                                      it > 0 || ks > 0 ? 1u : 0u);
                    if (kApart || !more) tc_commit(&o_done[x]);
                    if (x == 1) tc_commit(&v_empty[b]);
                }
                __syncwarp();
                if (!kApart && more) scores(x, it + 1);  // over the probabilities, which the product before it reads first
            }
        }
        if (!ok) s_fail = 1;
    } else if (warp >= kPaCheckWarp) {
        constexpr uint32_t kExp = std::is_same<T, __nv_bfloat16>::value ? 0x7f807f80u : 0x7c007c00u, kOne = std::is_same<T, __nv_bfloat16>::value ? 0x00800080u : 0x04000400u;
        for (int it = 0; it < n_tiles; ++it) {
            // (every tile passes through here: a wait for a phase is only unambiguous where every phase is visited)
            const int b = it & 1;
            if (!__all_sync(0xffffffffu, mbar_wait_bounded(&v_full[b], (uint32_t)(it >> 1) & 1u, nullptr))) {
                s_fail = 1;
                break;
            }
            constexpr int kAhead = 8;
            for (int i0 = (warp - kPaCheckWarp) * 32 + lane; i0 < (partial(it) ? kTile / 16 : 0); i0 += kPaCheckWarps * 32 * kAhead) {
                uint32_t w[kAhead][4];
#pragma unroll
                for (int k = 0; k < kAhead; ++k)
                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                                 : "=r"(w[k][0]), "=r"(w[k][1]), "=r"(w[k][2]), "=r"(w[k][3])
                                 : "r"(sv + b * kTile + (i0 + k * kPaCheckWarps * 32) * 16));
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    uint32_t odd = 0;
#pragma unroll
                    for (int j = 0; j < 4; ++j) odd |= ((w[k][j] & kExp) + kOne) & 0x80008000u;  // an exponent of ones carries into the sign's place
                    if (odd) {
                        s_odd = 1;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const uint32_t o = ((w[k][j] & kExp) + kOne) & 0x80008000u;
                            if (o & 0x8000u) w[k][j] &= 0xffff0000u;
                            if (o & 0x80000000u) w[k][j] &= 0x0000ffffu;
                        }
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(sv + b * kTile + (i0 + k * kPaCheckWarps * 32) * 16), "r"(w[k][0]), "r"(w[k][1]), "r"(w[k][2]),
                                     "r"(w[k][3])
                                     : "memory");
                    }
                }
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&v_clean[b]);
        }
    }
    } else {
        regs_up<kPaSoftRegs>();
        const int x = warp >> 2, row = (warp & 3) * 32 + lane;
        const int r_cta = a.pair_heads ? row : x * kPaRows + row, token = t0 + r_cta, head = head0 + (a.pair_heads ? x : 0);
        const int i_row = min(token, t_end - 1), first = s_start[min(r_cta, t_end - 1 - t0)];
        // what all rows of the warp see in full: keys from the last row's sequence on, up to the first row
        const int w_first = __shfl_sync(0xffffffffu, first, 31), w_last = __shfl_sync(0xffffffffu, i_row, 0);
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, ts = tmem + lanes + x * 128, to = tmem + lanes + kO + x * kOWide, tp = tmem + lanes + kP + x * kPWide;
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        for (int it = 0; it < n_tiles && ok; ++it) {
            ok = __all_sync(0xffffffffu, mbar_wait_bounded(&s_full[x], (uint32_t)it & 1u, nullptr));
            if (!ok) break;
            tc_fence_after();
            uint32_t s[128];
#pragma unroll
            for (int c = 0; c < 4; ++c) tc_ld32_async(ts + c * 32, s + c * 32);
            tc_wait_ld();
#pragma unroll
            for (int c = 0; c < 8; ++c) pin16(s + c * 16);
            if constexpr (kApart) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&s_read[x]);
            }
            const int key = k0 + it * kPaKeys;
            if (key < w_first || key + kPaKeys - 1 > w_last) {
                const int lo = first - key, hi = i_row - key;
#pragma unroll
                for (int c = 0; c < 128; c += 32) {  // a bit a key
                    const uint32_t from = lo <= c ? ~0u : lo < c + 32 ? ~0u << (lo - c) : 0u, to_ = hi >= c + 31 ? ~0u : hi >= c ? ~0u >> (31 - (hi - c)) : 0u, seen = from & to_;
#pragma unroll
                    for (int i = 0; i < 32; ++i) s[c + i] = seen & (1u << i) ? s[c + i] : 0xff800000u;
                }
            }
            float mx[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) mx[c] = __uint_as_float(s[c]);
#pragma unroll
            for (int c = 4; c < 128; ++c) mx[c & 3] = max_nan(mx[c & 3], __uint_as_float(s[c]));
            const float top = max_nan(max_nan(mx[0], mx[1]), max_nan(mx[2], mx[3])) * a.rate;
            if (!(top < INFINITY)) l = NAN;  // a score that is not a number, or infinite
            const bool grows = top > m + kPaGrowth;
            bool summed = !kApart || it == 0;  // the sums, and the probabilities' place, are free: the product of the tile before has run
            auto wait_summed = [&]() {
                if (!summed) {
                    ok = __all_sync(0xffffffffu, mbar_wait_bounded(&o_done[x], (uint32_t)(it - 1) & 1u, nullptr));
                    tc_fence_after();
                    summed = true;
                }
            };
            if (__any_sync(0xffffffffu, grows)) {
                wait_summed();
                const float next = grows ? top : m, f = grows ? pa_exp2(m - next) : 1.f;  // (from -infinity: 0)
                m = next;
                l *= f;
                if (it > 0) {
#pragma unroll
                    for (int c = 0; c < HS / 32; ++c) {
                        uint32_t o[32];
                        tc_ld32_async(to + c * 32, o);
                        tc_wait_ld();
                        pin16(o);
                        pin16(o + 16);
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                        tc_st32(to + c * 32, o);
                    }
                }
            }
            const float u = m == -INFINITY ? 0.f : m - kLift;
            const uint64_t rate2 = f2_pack(a.rate, a.rate), u2 = f2_pack(-u, -u);
            uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                uint32_t p[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const uint64_t y = f2_fma(f2_pack(__uint_as_float(s[c * 64 + 2 * i]), __uint_as_float(s[c * 64 + 2 * i + 1])), rate2, u2);
                    float2 e;
                    if ((i % 16) * kPoly % 16 >= 16 - kPoly) {
                        e = pa_exp2_poly<T>(y);
                    } else {
                        e = f2_unpack(y);
                        e = make_float2(pa_exp2(e.x), pa_exp2(e.y));
                    }
                    sum[i & 1] = f2_add(sum[i & 1], f2_pack(e.x, e.y));
                    p[i] = pack2<T>(e.x, e.y);
                }
                if (c == 0) wait_summed();
                tc_st32(tp + c * 32, p);
            }
            const float2 total2 = f2_unpack(f2_add(sum[0], sum[1]));
            l += total2.x + total2.y;
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_ready[x]);
        }
        ok = ok && __all_sync(0xffffffffu, mbar_wait_bounded(&o_done[x], kApart ? (uint32_t)(n_tiles - 1) & 1u : 0u, nullptr));
        if (!ok) s_fail = 1;
        tc_fence_after();
        const bool mine = token < t_end;
        T* dst = reinterpret_cast<T*>(a.out) + (long long)token * a.out_stride + (long long)head * a.head_size;
        const float inv = ok ? __fdiv_rn(1.f, l) : NAN;
#pragma unroll
        for (int c = 0; c < HS / 32; ++c) {
            uint32_t o[32];
            tc_ld32_async(to + c * 32, o);
            tc_wait_ld();
            pin16(o);
            pin16(o + 16);
            if (mine)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (c * 32 + i * 8 < a.head_size) {
                        uint32_t w[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) w[j] = pack2<T>(__uint_as_float(o[i * 8 + 2 * j]) * inv, __uint_as_float(o[i * 8 + 2 * j + 1]) * inv);
                        *reinterpret_cast<uint4*>(dst + c * 32 + i * 8) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
        }
        if (ok && mine && *reinterpret_cast<volatile int*>(&s_odd)) {  // (set before the last product)
            for (int it = 0; it < n_tiles; ++it) {
                if (!partial(it)) continue;
                const int j1 = min(k0 + it * kPaKeys + kPaKeys - 1, i_row);
                for (int j = max(k0 + it * kPaKeys, first); j <= j1; ++j) {
                    const T* v = reinterpret_cast<const T*>(a.v) + (long long)j * a.v_stride + (long long)kvh * a.head_size;
                    for (int d = 0; d < a.head_size; ++d) {
                        const float y = to_float(v[d]);
                        if (!(fabsf(y) < INFINITY)) dst[d] = from_float<T>(to_float(dst[d]) + y);
                    }
                }
            }
        }
    }
    // ---------------- common exit
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    // after a wait that ran out, copies may still be in flight: give them a bounded time to land
    if (tid == 0 && *reinterpret_cast<volatile int*>(&s_fail) != 0) {
        const long long c0 = clock64();
        while (clock64() - c0 < (1 << 17)) __nanosleep(1000);
    }
    __syncthreads();
    if (warp == kPaMmaWarp) tc_dealloc(tmem, 512);
}

}  // namespace lpp
