// Causal attention of whole prompts, packed one behind the other, with grouped query heads (the reference runs a prompt token by token
// through src/model.cpp:178-199): out_i = sum_j softmax_j(scale q_i . k_j) v_j over the tokens j <= i of i's own sequence.
//
// Tiles of 128 query rows of a head against tiles of 128 keys.  One tcgen05.mma chain forms the scores S = Q . K^T in tensor memory; four
// warps, one thread a row, take them into registers, form the probabilities and write them to tensor memory as the 16-bit operand of
// the second chain, O += P . V, whose sums stay there.  While rows are exponentiated the tensor cores work on something else:
// * head sizes up to 64: a CTA has one row tile and half of an SM's tensor memory (S 128 columns, P 64, O 64).  The next scores are
//   formed while the present ones, already in registers, are exponentiated, and a second CTA on the SM fills what is left.
// * head sizes up to 128: a CTA has two row tiles that read the same keys and values (two heads that share them, or 256 tokens), and
//   all of the tensor memory: S 128 columns and O 128 for either.  P takes the place of S, and the row tiles take turns.
// Sums O are rescaled only when a row's maximum has grown by more than 2^8 since it was last set, by the row's own thread, when the
// product of the tile before is complete.
//
// Measured from graphs: 8192 tokens of 32 heads of 128 take 438 - 480 us (up to 1.25 PFLOP/s; 507 - 518 in calls without a pause, under the power
// cap).  The products are 475,000 clocks an SM of that, 242 us at the full clock; tensor cores and special functions are busy 60 % of the clocks
// each, and without any exponentials it is 435 us, so the rest is the hand-over between the row tiles and the clock under the cap, which have not been
// told apart.  1023 tokens of 32 heads of 64: 15.5 - 17 us, of which the longest row tiles' eight steps take 1.4 us each (exponentials of one
// warp a scheduler) and start and end 4.  201 tokens of 6 heads of 48: 6.8 us.
//
// Sequences do not have to begin at tiles: row tiles cover the packed tokens whatever the borders, a row sees the keys from its
// sequence's start to itself, and a tile runs over the keys from its first row's sequence on.  Many short prompts share a tile.
//
// Keys of tokens that a row does not see are masked after the product; their values meet probabilities of 0, which hides everything but
// NaN and infinity.  So two warps look through the value tiles that some row sees only in part, zero what is not finite, and the rows
// that do see it get it added to their results at the end.  In a tile that all rows see it goes through the product, where an infinity whose
// probability has become 0 leaves a NaN.  So a row whose sum is not finite looks for what it saw (at its end; other rows pay 0.1 us
// for the look at their sums): an infinity makes a result infinite, a NaN or infinities of both signs make it no number, wherever tiles are cut.
#pragma once
#include "common.cuh"
#include "umma.cuh"

namespace lpp {

constexpr int kPaRows = 128, kPaKeys = 128, kPaSub = 128 * 128;  // kPaSub: bytes of 128 rows x 64 columns
constexpr float kPaGrowth = 8.f;     // of a row's maximum (base 2) before its sums are rescaled
constexpr int kPaOffsets = 1024;     // sequences whose offsets are searched in shared memory
constexpr int kPaCheckWarps = 2;
template <int HS>
struct PaShape {
    static constexpr int kTiles = HS == 64 ? 1 : 2, kCtas = HS == 64 ? 2 : 1;  // row tiles of a CTA, CTAs of an SM
    static constexpr int kSoftWarps = 4 * kTiles, kMmaWarp = kSoftWarps, kLoadWarp = kSoftWarps + 1, kCheckWarp = kSoftWarps + 2, kThreads = (kSoftWarps + 4) * 32;
    // Registers: the threads start with kRegs each; the softmax warps take what the other four give back
    static constexpr int kRegs = HS == 64 ? 128 : 168, kSoftRegs = HS == 64 ? 200 : 224, kOtherRegs = 56;
    static_assert(kSoftWarps * 32 * kSoftRegs + 128 * kOtherRegs <= kThreads * kRegs && kThreads * kRegs * kCtas <= 65536,
                  "a split must not ask for more registers than the block was launched with");
    static constexpr int kTile = HS / 64 * kPaSub;                            // bytes of 128 rows
    static constexpr int kSmem = 1024 /*alignment*/ + (kTiles + 4) * kTile;  // Q, 2 x K, 2 x V
    static constexpr bool kApart = HS == 64;                                  // probabilities beside the scores, not over them
    static constexpr uint32_t kColumns = HS == 64 ? 256 : 512, kP = kApart ? 128 : 0, kO = HS == 64 ? 192 : 256;  // tensor memory; S at 0; 128 columns further for row tile 1
};

struct PromptAttnArgs {
    void* out;
    const void* v;        // for rows that see a value that is not finite
    const int* offsets;   // [sequences + 1]
    long long out_stride, v_stride;
    int n_sequences, n_tokens, heads, gqa, head_size, tiles;
    int pair_heads;       // two row tiles: 128 tokens of two heads; else 256 tokens of one
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
template <int HS, typename T>
static __global__ void __launch_bounds__(PaShape<HS>::kThreads, PaShape<HS>::kCtas) prompt_attention_kernel(const __grid_constant__ CUtensorMap q_map,
                                                                                                            const __grid_constant__ CUtensorMap k_map,
                                                                                                            const __grid_constant__ CUtensorMap v_map, const PromptAttnArgs a) {
    using Shape = PaShape<HS>;
    constexpr int kPieces = HS / 64, kTile = Shape::kTile, kTiles = Shape::kTiles;
    constexpr bool kApart = Shape::kApart;
    // FP16 probabilities stay clear of the subnormals: they are 2^(x - m + 6) at most 2^14
    constexpr float kLift = std::is_same<T, __half>::value ? 6.f : 0.f;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], v_clean[2], s_full[kTiles], s_read[kTiles], p_ready[kTiles], o_done[kTiles];
    __shared__ uint32_t tmem_slot;
    __shared__ int s_fail, s_odd, s_start[kTiles * kPaRows], s_off[kPaOffsets + 1];
    const uint32_t base = (smem_u32(smem) + 1023u) & ~1023u;
    const uint32_t sq = base, sk = sq + kTiles * kTile, sv = sk + 2 * kTile;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const bool pair = kTiles == 2 && a.pair_heads;
    // The last row tiles come first: of one sequence they are the longest.  (Several sequences' tiles sorted by length, so that long ones share
    // SMs: ten packed prompts of up to 1500 tokens 49 us against 47.)
    const int per_tile = pair ? a.heads / 2 : a.heads, rank = (int)blockIdx.x / per_tile, unit = (int)blockIdx.x - rank * per_tile;
    const int cta_rows = pair ? kPaRows : kTiles * kPaRows, t0 = (a.tiles - 1 - rank) * cta_rows;
    const int head0 = pair ? 2 * unit : unit, kvh = head0 / a.gqa;
    if (tid == 0) {
        tma_prefetch_map(&q_map);
        tma_prefetch_map(&k_map);
        tma_prefetch_map(&v_map);
        s_fail = 0;
        s_odd = 0;
        mbar_init(&q_full, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&k_full[i], 1);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_full[i], 1);
            mbar_init(&v_empty[i], 1);
            mbar_init(&v_clean[i], kPaCheckWarps);
        }
        for (int i = 0; i < kTiles; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&s_read[i], 4);
            mbar_init(&p_ready[i], 4);
            mbar_init(&o_done[i], 1);
        }
        mbar_fence_init();
    }
    pdl_wait();
    const bool few = a.n_sequences <= kPaOffsets;
    if (few)
        for (int i = tid; i <= a.n_sequences; i += Shape::kThreads) s_off[i] = a.offsets[i];
    const int total = min(a.offsets[a.n_sequences], a.n_tokens);
    if (t0 >= total) return;
    const int t_end = min(total, t0 + cta_rows);
    if (warp == Shape::kMmaWarp) {
        tc_alloc(&tmem_slot, Shape::kColumns);
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
    // the signs' places of the numbers of a pair that are not finite: an exponent of ones carries into them
    auto odd_of = [](uint32_t w) {
        constexpr bool bf16 = std::is_same<T, __nv_bfloat16>::value;
        return ((w & (bf16 ? 0x7f807f80u : 0x7c007c00u)) + (bf16 ? 0x00800080u : 0x04000400u)) & 0x80008000u;
    };
    auto wait = [](uint64_t* bar, int phase) { return __all_sync(0xffffffffu, mbar_wait_bounded(bar, (uint32_t)phase & 1u, nullptr)) != 0; };

    if (warp >= Shape::kSoftWarps) {
        regs_down<Shape::kOtherRegs>();
        if (warp == Shape::kLoadWarp) {
            // ---------------- queries, keys and values
            if (lane == 0) {
                auto load = [&](uint32_t to, const CUtensorMap* map, int head, int token, uint64_t* bar) {
                    for (int p = 0; p < kPieces; ++p) tma_load_3d(to + p * kPaSub, map, p * 64, head, token, smem_u32(bar));
                };
                mbar_arrive_expect_tx(&q_full, kTiles * kTile);
                for (int x = 0; x < kTiles; ++x) load(sq + x * kTile, &q_map, head0 + (pair ? x : 0), t0 + (pair ? 0 : x * kPaRows), &q_full);
                bool ok = true;
                for (int it = 0; it < n_tiles && ok; ++it) {
                    const int b = it & 1;
                    ok = it < 2 || mbar_wait_bounded(&k_empty[b], (uint32_t)((it >> 1) - 1) & 1u, nullptr);
                    if (!ok) break;
                    mbar_arrive_expect_tx(&k_full[b], kTile);
                    load(sk + b * kTile, &k_map, kvh, k0 + it * kPaKeys, &k_full[b]);
                    ok = it < 2 || mbar_wait_bounded(&v_empty[b], (uint32_t)((it >> 1) - 1) & 1u, nullptr);
                    if (!ok) break;
                    mbar_arrive_expect_tx(&v_full[b], kTile);
                    load(sv + b * kTile, &v_map, kvh, k0 + it * kPaKeys, &v_full[b]);
                }
                if (!ok) s_fail = 1;
            }
        } else if (warp == Shape::kMmaWarp) {
            // ---------------- products
            auto scores = [&](int x, int it) {
                if (elect_one()) {
#pragma unroll
                    for (int ks = 0; ks < HS / 16; ++ks) {
                        const uint32_t off = (uint32_t)((ks >> 2) * kPaSub + (ks & 3) * 32);
                        tc_mma_f16(tmem + x * 128, umma_desc(sq + x * kTile + off), umma_desc(sk + (it & 1) * kTile + off), pa_idesc<T>(kPaKeys, false), ks > 0 ? 1u : 0u);
                    }
                    tc_commit(&s_full[x]);
                    if (x == kTiles - 1) tc_commit(&k_empty[it & 1]);
                }
                __syncwarp();
            };
            bool ok = wait(&q_full, 0) && wait(&k_full[0], 0);
            if (ok) {
                tc_fence_after();
                for (int x = 0; x < kTiles; ++x) scores(x, 0);
            }
            for (int it = 0; it < n_tiles && ok; ++it) {
                const int b = it & 1;
                const bool more = it + 1 < n_tiles;
                if (more) ok = wait(&k_full[b ^ 1], (it + 1) >> 1);
                if (kApart && more && ok) {  // the scores have been taken into registers: their place takes the next
                    ok = wait(&s_read[0], it);
                    if (!ok) break;
                    tc_fence_after();
                    scores(0, it + 1);
                }
                ok = ok && wait(&v_full[b], it >> 1) && wait(&v_clean[b], it >> 1);
                for (int x = 0; x < kTiles && ok; ++x) {
                    ok = wait(&p_ready[x], it);
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one()) {
#pragma unroll
                        for (int ks = 0; ks < kPaKeys / 16; ++ks)
                            tc_mma_f16_ts(tmem + Shape::kO + x * 128, tmem + Shape::kP + x * 128 + ks * 8, pa_desc_v(sv + b * kTile + ks * 2048), pa_idesc<T>(HS, true),
                                          it > 0 || ks > 0 ? 1u : 0u);
                        if (kApart || !more) tc_commit(&o_done[x]);
                        if (x == kTiles - 1) tc_commit(&v_empty[b]);
                    }
                    __syncwarp();
                    if (!kApart && more) scores(x, it + 1);  // over the probabilities, which the product before it reads first
                }
            }
            if (!ok) s_fail = 1;
        } else {
            // ---------------- values that are not finite
            constexpr int kAhead = 8, kStep = kPaCheckWarps * 32;
            static_assert(kTile / 16 % (kAhead * kStep) == 0, "a tile is a whole number of rounds");
            for (int it = 0; it < n_tiles; ++it) {
                // (every tile passes through here: a wait for a phase is only unambiguous where every phase is visited)
                const int b = it & 1;
                if (!wait(&v_full[b], it >> 1)) {
                    s_fail = 1;
                    break;
                }
                for (int i0 = (warp - Shape::kCheckWarp) * 32 + lane; i0 < (partial(it) ? kTile / 16 : 0); i0 += kAhead * kStep) {
                    uint32_t w[kAhead][4];
#pragma unroll
                    for (int k = 0; k < kAhead; ++k)
                        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                                     : "=r"(w[k][0]), "=r"(w[k][1]), "=r"(w[k][2]), "=r"(w[k][3])
                                     : "r"(sv + b * kTile + (i0 + k * kStep) * 16));
#pragma unroll
                    for (int k = 0; k < kAhead; ++k) {
                        uint32_t odd = 0;
#pragma unroll
                        for (int j = 0; j < 4; ++j) odd |= odd_of(w[k][j]);
                        if (odd) {
                            s_odd = 1;
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const uint32_t o = odd_of(w[k][j]);
                                if (o & 0x8000u) w[k][j] &= 0xffff0000u;
                                if (o & 0x80000000u) w[k][j] &= 0x0000ffffu;
                            }
                            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(sv + b * kTile + (i0 + k * kStep) * 16), "r"(w[k][0]), "r"(w[k][1]), "r"(w[k][2]), "r"(w[k][3])
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
        // ---------------- probabilities and results: a thread a row
        regs_up<Shape::kSoftRegs>();
        const int x = warp >> 2, row = (warp & 3) * 32 + lane, r_cta = pair ? row : x * kPaRows + row;
        const int token = t0 + r_cta, head = head0 + (pair ? x : 0);
        const int i_row = min(token, t_end - 1), first = s_start[min(r_cta, t_end - 1 - t0)];
        // what all rows of the warp see: keys from the last row's sequence on, up to the first row
        const int w_first = __shfl_sync(0xffffffffu, first, 31), w_last = __shfl_sync(0xffffffffu, i_row, 0);
        const uint32_t tm = tmem + ((uint32_t)((warp & 3) * 32) << 16) + x * 128;
        const uint64_t rate2 = f2_pack(a.rate, a.rate);
        float m = -INFINITY, l = 0.f;  // reference of the exponentials (base 2), sum of the probabilities
        bool ok = true;
        for (int it = 0; it < n_tiles && ok; ++it) {
            ok = wait(&s_full[x], it);
            if (!ok) break;
            tc_fence_after();
            uint32_t s[128];
#pragma unroll
            for (int c = 0; c < 128; c += 32) tc_ld32_async(tm + c, s + c);
            tc_wait_ld();
#pragma unroll
            for (int c = 0; c < 128; c += 16) pin16(s + c);
            if constexpr (kApart) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&s_read[x]);
            }
            const int key = k0 + it * kPaKeys;
            uint32_t blank = 0;  // bit c: no row of the warp sees any of the keys 32 c .. 32 c + 31
            if (key < w_first || key + kPaKeys - 1 > w_last) {
                const int lo = first - key, hi = i_row - key;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int lo_c = lo - 32 * c, hi_c = hi - 32 * c;
                    const uint32_t seen = (lo_c <= 0 ? ~0u : lo_c < 32 ? ~0u << lo_c : 0u) & (hi_c >= 31 ? ~0u : hi_c >= 0 ? ~0u >> (31 - hi_c) : 0u);
                    if (kTiles == 1 && !__any_sync(0xffffffffu, seen != 0u)) blank |= 1u << c;
#pragma unroll
                    for (int i = 0; i < 32; ++i) s[c * 32 + i] = seen & (1u << i) ? s[c * 32 + i] : 0xff800000u;
                }
            }
            float mx[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) mx[c] = __uint_as_float(s[c]);
#pragma unroll
            for (int c = 4; c < 128; ++c) mx[c & 3] = max_nan(mx[c & 3], __uint_as_float(s[c]));
            const float top = max_nan(max_nan(mx[0], mx[1]), max_nan(mx[2], mx[3])) * a.rate;
            if (!(top < INFINITY)) l = NAN;  // a score that is not a number, or infinite
            bool summed = !kApart || it == 0;  // the product of the tile before has run: sums and the probabilities' place are free
            auto wait_summed = [&]() {
                if (!summed) {
                    ok = wait(&o_done[x], it - 1);
                    tc_fence_after();
                    summed = true;
                }
            };
            const bool grows = top > m + kPaGrowth;
            if (__any_sync(0xffffffffu, grows)) {
                const float next = grows ? top : m, f = grows ? pa_exp2(m - next) : 1.f;  // (from -infinity: 0)
                m = next;
                l *= f;
                if (it > 0) {
                    wait_summed();
#pragma unroll
                    for (int c = 0; c < HS; c += 32) {
                        uint32_t o[32];
                        tc_ld32_async(tm + Shape::kO + c, o);
                        tc_wait_ld();
                        pin16(o);
                        pin16(o + 16);
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                        tc_st32(tm + Shape::kO + c, o);
                    }
                }
            }
            const float u = m == -INFINITY ? 0.f : m - kLift;
            const uint64_t u2 = f2_pack(-u, -u);
            uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                uint32_t p[32];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (kTiles == 1 && (blank & (1u << (2 * c + h)))) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) p[h * 16 + i] = 0u;
                        continue;
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int at = c * 64 + h * 32 + 2 * i;
                        const uint64_t y = f2_fma(f2_pack(__uint_as_float(s[at]), __uint_as_float(s[at + 1])), rate2, u2);
                        const float2 z = f2_unpack(y);
                        const float e0 = pa_exp2(z.x), e1 = pa_exp2(z.y);
                        sum[i & 1] = f2_add(sum[i & 1], f2_pack(e0, e1));
                        p[h * 16 + i] = pack2<T>(e0, e1);
                    }
                }
                if (c == 0) wait_summed();
                tc_st32(tm + Shape::kP + c * 32, p);
            }
            const float2 both = f2_unpack(f2_add(sum[0], sum[1]));
            l += both.x + both.y;
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_ready[x]);
        }
        ok = ok && wait(&o_done[x], kApart ? n_tiles - 1 : 0);
        if (!ok) s_fail = 1;
        tc_fence_after();
        const bool mine = token < t_end;
        T* dst = reinterpret_cast<T*>(a.out) + (long long)token * a.out_stride + (long long)head * a.head_size;
        const float inv = ok ? __fdiv_rn(1.f, l) : NAN;
        float lost[4] = {};  // NaN: a sum is not finite
#pragma unroll
        for (int c = 0; c < HS; c += 32) {
            uint32_t o[32];
            tc_ld32_async(tm + Shape::kO + c, o);
            tc_wait_ld();
            pin16(o);
            pin16(o + 16);
#pragma unroll
            for (int i = 0; i < 32; ++i) lost[i & 3] = __fmaf_rn(__uint_as_float(o[i]), 0.f, lost[i & 3]);
#pragma unroll
            for (int i = 0; i < 32; i += 8)
                if (mine && c + i < a.head_size) {
                    uint32_t w[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) w[j] = pack2<T>(__uint_as_float(o[i + 2 * j]) * inv, __uint_as_float(o[i + 2 * j + 1]) * inv);
                    *reinterpret_cast<uint4*>(dst + c + i) = make_uint4(w[0], w[1], w[2], w[3]);
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
        // (no sum of probabilities: all is NaN).  The lanes look through 128 tokens at once, eight dimensions each, and hand what they find around.
        const bool search = ok && mine && l < INFINITY && !((lost[0] + lost[1]) + (lost[2] + lost[3]) == 0.f);
        if (__any_sync(0xffffffffu, search)) {
            const int j0 = __reduce_min_sync(0xffffffffu, search ? first : t_end), j1 = __reduce_max_sync(0xffffffffu, search ? i_row : 0);
            for (int d = 0; d < a.head_size; d += 8) {
                bool look = false;
                if (search)
#pragma unroll
                    for (int i = 0; i < 8; ++i) look = look || !(fabsf(to_float(dst[d + i])) < INFINITY);
                if (!__any_sync(0xffffffffu, look)) continue;
                const T* v = reinterpret_cast<const T*>(a.v) + (long long)kvh * a.head_size + d;
                float seen[8] = {};
                for (int j = j0; j <= j1; j += 128) {
                    uint4 y[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int at = j + 32 * k + lane;
                        y[k] = at <= j1 ? *reinterpret_cast<const uint4*>(v + (long long)at * a.v_stride) : make_uint4(0u, 0u, 0u, 0u);
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        unsigned odd = __ballot_sync(0xffffffffu, (odd_of(y[k].x) | odd_of(y[k].y) | odd_of(y[k].z) | odd_of(y[k].w)) != 0u);
                        for (; odd; odd &= odd - 1u) {
                            const int from = __ffs((int)odd) - 1, at = j + 32 * k + from;
                            const uint32_t w[4] = {__shfl_sync(0xffffffffu, y[k].x, from), __shfl_sync(0xffffffffu, y[k].y, from), __shfl_sync(0xffffffffu, y[k].z, from),
                                                   __shfl_sync(0xffffffffu, y[k].w, from)};
                            if (!look || at < first || at > i_row) continue;
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const float2 f = unpack2<T>(w[i]);
                                if (!(fabsf(f.x) < INFINITY)) seen[2 * i] += f.x;
                                if (!(fabsf(f.y) < INFINITY)) seen[2 * i + 1] += f.y;
                            }
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (seen[i] != 0.f) dst[d + i] = from_float<T>(seen[i]);  // (0: finite values whose sum is beyond the type)
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
    if (warp == Shape::kMmaWarp) tc_dealloc(tmem, Shape::kColumns);
}

}  // namespace lpp
