// A key/value cache held in 4 bits: writing rows into it, reading them back, attention of one token per sequence over it, and
// moving the rows that matter into a shorter cache.  No counterpart in the reference, whose cache is FP16 (src/model.h:108-109); the
// layout follows its order [kv head][position] (src/scatter_kv.cu:15-16) with one more dimension for the sequence.
//
// A row holds the keys (or values) of one head at one position in groups of 32 dimensions.  With lo and hi the least and the largest
// value of a group:
//     scale = fp16(fp32((hi - lo) / 15)),  zero = fp16(fp32(lo + 8 scale)),  code = clamp(round((x - zero) / scale) + 8, 0, 15)
// (exact quotients and sums rounded to FP32, then to FP16: of FP32 values a few groups in 100,000 get a neighbour of what one rounding
// would give, which its codes then go by; half to even; code 8 where scale is 0), and the code stands for zero + scale (code - 8).  The bytes of a row: 16 per group with two codes each (the lower
// dimension in the lower half), then 4 per group with scale and zero.  The dimensions that fill the last group up have code 8 and
// count neither for lo nor for hi.  A NaN is written as 0, values beyond the FP16 range as +-65504.
#pragma once
#include "common.cuh"

namespace lpp {

constexpr int kKv4Group = 32;
__host__ __device__ constexpr int kv4_groups(int head_size) { return (head_size + kKv4Group - 1) / kKv4Group; }
__host__ __device__ constexpr int kv4_row_bytes(int groups) { return groups * (kKv4Group / 2 + 4); }

// n / d for 32-bit numbers by the reciprocal floor(2^32 / d), which gives the quotient or one less
struct Kv4Div {
    uint32_t d, inv;
    __device__ __forceinline__ uint32_t operator()(uint32_t n) const {
        const uint32_t q = d == 1 ? n : __umulhi(n, inv);
        return q + (n - q * d >= d ? 1u : 0u);
    }
};
// The caches of one layer: [batch][kv_heads][capacity] rows.
struct Kv4Cache {
    unsigned char *k, *v;
    long long capacity, slots;  // slots: batch * capacity
    int kv_heads;
    Kv4Div by_heads, by_capacity;  // (the second where there are fewer than 2^32 slots)
    __device__ __forceinline__ long long row(long long slot, int head) const {
        const long long b = slots >> 32 ? slot / capacity : (long long)by_capacity((uint32_t)slot);
        return (b * kv_heads + head) * capacity + (slot - b * capacity);
    }
};

// ------------------------------------------------------------------ writing and reading rows
//
// Two threads a group, sixteen dimensions (two 32-bit words of codes) each.  Bound by the instructions on the way in (about 20 an element:
// 8001 tokens of 8 heads of 128, keys and values, 16 us, 2.7 TB/s; with eight elements a thread, conversions by the conversion unit and
// 64-bit divisions 34), by the bytes of the values and their latency on the way out (10 us, 4.2 TB/s).

constexpr int kKv4RowThreads = 256, kKv4Each = 16;  // kKv4Each: dimensions of a thread

// Sixteen consecutive values; `n` of them exist, the others are the first one again.  WIDE: all or none exist, on a 16-byte boundary.
template <typename T, bool WIDE>
__device__ __forceinline__ void kv4_load(const T* p, int n, float (&x)[kKv4Each]) {
    if constexpr (WIDE) {
        if constexpr (sizeof(T) == 4) {
            float4 a[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) a[i] = reinterpret_cast<const float4*>(p)[i];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[4 * i] = a[i].x, x[4 * i + 1] = a[i].y, x[4 * i + 2] = a[i].z, x[4 * i + 3] = a[i].w;
        } else {
            const uint4 a = reinterpret_cast<const uint4*>(p)[0], b = reinterpret_cast<const uint4*>(p)[1];
            const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float2 f = unpack2<T>(w[i]);
                x[2 * i] = f.x;
                x[2 * i + 1] = f.y;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < kKv4Each; ++i) x[i] = i < n ? to_float(p[i]) : i > 0 ? x[0] : 0.f;
    }
}

// a - b = d + e exactly (Knuth's two-sum)
__device__ __forceinline__ float exact_sub(float a, float b, float& e) {
    const float d = __fsub_rn(a, b), bb = __fsub_rn(d, a);
    e = __fsub_rn(__fsub_rn(a, __fsub_rn(d, bb)), __fadd_rn(b, bb));
    return d;
}

// The code of x where about `t` = (x - zero) / scale + 8, from 0 to 15, comes out next to a border between two codes: the exact remainder
// decides, so that the code is that of the exact quotient.
__device__ __forceinline__ uint32_t kv4_border(float x, float zero, float scale, float t) {
    float e;
    const float d = exact_sub(x, zero, e), border = floorf(t) + 0.5f;       // (border - 8) * scale: 5 + 11 bits, exact
    const float rest = __fadd_rn(__fsub_rn(d, (border - 8.f) * scale), e);  // the subtraction is exact so near the border
    return (uint32_t)(rest > 0.f ? border + 0.5f : rest < 0.f ? border - 0.5f : rintf(border));
}

template <typename T, int NG, bool WIDE>
static __global__ void __launch_bounds__(kKv4RowThreads, 5) kv4_write_kernel(const Kv4Cache c, const T* k, const T* v, const long long* slots, int n_rows,
                                                                          int head_size, long long k_stride, long long v_stride) {
    op_begin();
    constexpr int kLanes = 2 * NG;  // threads of a row
    const uint32_t i = blockIdx.x * kKv4RowThreads + threadIdx.x, row = i / kLanes, lane = i - row * kLanes;
    if ((i - (threadIdx.x & 31)) / kLanes >= (uint32_t)n_rows) return;  // (whole warps: the shuffles below need all lanes)
    const uint32_t known = min(row, (uint32_t)n_rows - 1), token = c.by_heads(known), head = known - token * c.kv_heads;
    const long long slot = slots[token];
    const int d0 = lane * kKv4Each, n = head_size - d0;
    float x[kKv4Each];
    const T* src = blockIdx.y ? v + token * v_stride : k + token * k_stride;
    kv4_load<T, WIDE>(src + (long long)head * head_size + (n > 0 ? d0 : 0), n, x);  // (where there is none: the first, which does not count)
    float lo, hi;
    auto ends = [&]() {  // NaN where there is one
        lo = hi = x[0];
#pragma unroll
        for (int j = 1; j < kKv4Each; ++j) {
            asm("min.NaN.f32 %0, %0, %1;" : "+f"(lo) : "f"(x[j]));
            asm("max.NaN.f32 %0, %0, %1;" : "+f"(hi) : "f"(x[j]));
        }
    };
    ends();
    if (!(lo >= -65504.f && hi <= 65504.f)) {
#pragma unroll
        for (int j = 0; j < kKv4Each; ++j) x[j] = x[j] == x[j] ? fminf(fmaxf(x[j], -65504.f), 65504.f) : 0.f;
        ends();
    }
    if (n <= 0) {  // no dimension of the head lies here
        lo = INFINITY;
        hi = -INFINITY;
    }
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, 1));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, 1));
    if (lo > hi) lo = hi = 0.f;  // nor in the whole group
    // (hi - lo) / 15: the exact difference's quotient rounded once to FP32, then to FP16
    float e;
    const float d = exact_sub(hi, lo, e), q = d * (1.f / 15.f), rest = __fadd_rn(__fmaf_rn(-15.f, q, d), e);
    const __half scale_h = __float2half_rn(__fmaf_rn(rest, 1.f / 15.f, q));
    const float scale = __half2float(scale_h);
    const __half zero_h = __float2half_rn(__fmaf_rn(8.f, scale, lo));
    const float zero = __half2float(zero_h);
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(scale));
    inv = scale == 0.f ? 0.f : inv * (1.f / 15.f);  // (0: every code 8)
    // Codes: a fifteenth of (quotient + 8), cut to 0 .. 1, times fifteen and rounded by adding 1.5 2^23.  The quotient is off by less than
    // 2^-17; where one came within twice that of a border the thread looks at its values again.
    uint32_t word[2] = {0u, 0u};
    float worst = 0.f;
#pragma unroll
    for (int j = 0; j < kKv4Each; ++j) {
        float t;
        asm("fma.rn.sat.f32 %0, %1, %2, %3;" : "=f"(t) : "f"(__fsub_rn(x[j], zero)), "f"(inv), "f"(8.f / 15.f));
        const float y = __fmaf_rn(t, 15.f, 12582912.f);
        worst = fmaxf(worst, fabsf(__fmaf_rn(t, 15.f, -__fsub_rn(y, 12582912.f))));
        word[j / 8] += __float_as_uint(y) << (4 * (j % 8));
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) word[w] -= 0x3f400000u;  // what 1.5 2^23 put there eight times, 4 bits apart
    if (worst > 0.499985f) {
        float from = zero;
        asm volatile("" : "+f"(from));  // (quotients are made again here, not kept from above)
#pragma unroll
        for (int j = 0; j < kKv4Each; ++j) {
            const float u = fminf(fmaxf(__fmaf_rn(__fsub_rn(x[j], from), inv * 15.f, 8.f), 0.f), 15.f);
            if (fabsf(u - rintf(u)) > 0.49996f) word[j / 8] = (word[j / 8] & ~(15u << (4 * (j % 8)))) | min(kv4_border(x[j], zero, scale, u), 15u) << (4 * (j % 8));
        }
    }
    if (n < (WIDE ? 1 : kKv4Each)) {  // dimensions that the head does not have: code 8
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const int have = n - 8 * w;
            const uint32_t there = have >= 8 ? ~0u : have <= 0 ? 0u : (1u << (4 * have)) - 1u;
            word[w] = (word[w] & there) | (0x88888888u & ~there);
        }
    }
    if (row >= (uint32_t)n_rows || slot < 0 || slot >= c.slots) return;
    unsigned char* dst = (blockIdx.y ? c.v : c.k) + c.row(slot, head) * kv4_row_bytes(NG);
    if constexpr (NG % 2 == 0) {
        *reinterpret_cast<uint2*>(dst + lane * 8) = make_uint2(word[0], word[1]);
    } else {
        reinterpret_cast<uint32_t*>(dst + lane * 8)[0] = word[0];
        reinterpret_cast<uint32_t*>(dst + lane * 8)[1] = word[1];
    }
    if ((lane & 1) == 0)
        *reinterpret_cast<uint32_t*>(dst + NG * 16 + lane * 2) = (uint32_t)__half_as_ushort(scale_h) | (uint32_t)__half_as_ushort(zero_h) << 16;
}

template <typename T, int NG, bool WIDE>
static __global__ void __launch_bounds__(kKv4RowThreads) kv4_read_kernel(const Kv4Cache c, T* k, T* v, const long long* slots, int n_rows, int head_size,
                                                                         long long k_stride, long long v_stride) {
    op_begin();
    constexpr int kLanes = 2 * NG;
    const uint32_t i = blockIdx.x * kKv4RowThreads + threadIdx.x, row = i / kLanes, lane = i - row * kLanes;
    if (row >= (uint32_t)n_rows) return;
    const uint32_t token = c.by_heads(row), head = row - token * c.kv_heads;
    const int d0 = lane * kKv4Each, n = head_size - d0;
    const long long slot = slots[token];
    if (n <= 0 || slot < 0 || slot >= c.slots) return;
    const unsigned char* src = (blockIdx.y ? c.v : c.k) + c.row(slot, head) * kv4_row_bytes(NG);
    uint32_t word[2];
    if constexpr (NG % 2 == 0) {
        const uint2 w = *reinterpret_cast<const uint2*>(src + lane * 8);
        word[0] = w.x;
        word[1] = w.y;
    } else {
        word[0] = reinterpret_cast<const uint32_t*>(src + lane * 8)[0];
        word[1] = reinterpret_cast<const uint32_t*>(src + lane * 8)[1];
    }
    const float2 sz = half2_bits_to_float2(*reinterpret_cast<const uint32_t*>(src + NG * 16 + (lane & ~1u) * 2));
    T* dst = (blockIdx.y ? v + token * v_stride : k + token * k_stride) + (long long)head * head_size + d0;
    __align__(16) T y[kKv4Each];
#pragma unroll
    for (int j = 0; j < kKv4Each; ++j) {  // 2^23 + code as a bit pattern; the product is exact
        const float code = __fsub_rn(__uint_as_float(0x4b000000u | (word[j / 8] >> (4 * (j % 8)) & 15u)), 8388616.f);
        y[j] = from_float<T>(__fmaf_rn(sz.x, code, sz.y));
    }
    if constexpr (WIDE) {
#pragma unroll
        for (int j = 0; j < (int)sizeof(T); ++j) reinterpret_cast<uint4*>(dst)[j] = reinterpret_cast<const uint4*>(y)[j];
    } else {
#pragma unroll
        for (int j = 0; j < kKv4Each; ++j)
            if (j < n) dst[j] = y[j];
    }
}

// ------------------------------------------------------------------ clusters

__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_map(uint32_t smem_addr, uint32_t cta) {  // the same place in another CTA of the cluster
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr), "r"(cta));
    return r;
}
__device__ __forceinline__ uint32_t kv4_cluster_load(uint32_t a) {
    uint32_t r;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(r) : "r"(a) : "memory");
    return r;
}

// ------------------------------------------------------------------ attention of one token per sequence
//
// out = sum_j p_j v_j, p = softmax(scale q . k_j) over the positions below the sequence's length.  Units of 128 positions of one
// key/value head, in the order [sequence][head][position], are dealt out to the CTAs in equal runs, whatever the lengths; the eight
// warps of a CTA take 16 positions of a unit each and keep running sums of their own, which are put together where a run goes on to
// the next head or ends.  Heads that lie in several runs are put together by the finishing kernel.
//
// Products on the tensor cores (mma.sync.m16n8k16, FP32 sums), cache rows as the 16-row operand and up to eight query heads of the
// key/value head as the 8-column one.  The codes themselves are the operand: as FP16 bit patterns, 0 .. 15 are the subnormals
// n 2^-24, and the same bits four places up are 16 n 2^-24, so a mask makes two elements of an operand register (the query elements of
// the second kind are divided by 16).  Sums are kept apart by group and multiplied with the group's scale in FP32:
//     q . k = sum_g scale_g sum_d q_d n_d + (zero_g - 8 scale_g) Q_g,  Q_g = sum_d q_d;
// the second part is one more product, of the (scale, zero) pairs as they lie in the row with (-8 Q_g, Q_g), Q_g as two FP16
// operands.  For the values the scale goes to the probability before that is rounded to FP16, the codes become n - 8 (rounding errors then
// are those of values around their middle), and sum_j p_j zero_jg is added in FP32.
//
// Reference of the exponentials: not the running maximum of the scores but a bound on the largest p * scale, which has to stay in the
// FP16 range: probabilities are 2^(x - M) with M far enough below the largest x + log2(scale) seen when M was set that they keep their
// bits, and M moves only when a product would leave the range.  So a tile needs no maximum over lanes, only a vote.
//
// Bound by the instructions around the products, about 400 a warp for 16 positions of 128 dimensions: 131071 positions of eight heads are
// 24 us of issue slots, their 168 MB 26 us.  Four warps a scheduler fill 63 % of the slots: 43.5 us (3.9 TB/s); 32769 positions with sums
// 23 us, of which starting and merging take 5 and the second kernel 4.  131071 positions of eight heads of 64, whose rows of 40 bytes are no
// multiple of 16 (no ldmatrix, see kv4_codes): 31 us for 84 MB.
//
// SPLIT, for FP32 queries and results, whose groups may differ in size: queries go in as two FP16 operands (hi + lo) with a power of two of
// every group, which scale_g's factor takes back; the keys' codes are n - 8 too, and zero_g Q_g is added in FP32 (sums of n and 8 Q_g that cancel
// would cost two bits of the scores).  Probabilities times scales go in as three BF16 operands, which are all of an FP32 number wherever it lies;
// two FP16 ones, under the one reference of all groups, lost bits of groups 2^-11 below the largest, and the low half of those 2^-22 below.
// About 610 instructions a warp for 16 positions: 131071 positions of eight heads of 128 66 us (with two FP16 operands 55), of heads of 64 40 us
// (35.5); 641 positions of 2048 6.65 us (6.4).
constexpr int kKv4Warps = 8, kKv4Threads = kKv4Warps * 32;
constexpr int kKv4Tile = 16;     // positions of a warp's tile
constexpr int kKv4Unit = kKv4Warps * kKv4Tile;
constexpr int kKv4Heads = 8;     // query heads of a CTA
constexpr float kKv4Limit = 32768.f;  // of p * scale
constexpr int kKv4MaxStages = 8;  // units in flight per CTA
template <int NG>
constexpr int kKv4Ctas = NG > 4 ? 1 : 2;    // of an SM

struct Kv4AttnArgs {
    const unsigned char *k, *v;
    const void* q;
    void* out;
    const int* lens;
    const float* sums_in;   // NULL = zeros
    float* sums_out;        // NULL = no sums
    float* scores;          // [batch][kv_heads][capacity][gqa], base-2 exponents (with sums)
    float2* whole_ml;       // [batch][heads]: reference and sum of heads that lie in one run (with sums)
    float2* part_ml;        // [runs][2][8]: the same of parts of a head: [0] one that began in an earlier run, [1] one that begins here
    float* part_o;          // [runs][2][8][NG * 32]
    long long capacity, q_stride, out_stride;
    int batch, heads, kv_heads, gqa, head_size, head_tiles, runs, stages;
    int cluster;            // short caches: CTAs of a head
    int dtype;
    float rate;             // scale * log2(e)
};

__device__ __forceinline__ int kv4_len(const Kv4AttnArgs& a, int b) { return (int)max(0ll, min((long long)a.lens[b], a.capacity)); }
__device__ __forceinline__ int kv4_units(int len) { return max(1, (len + kKv4Unit - 1) / kKv4Unit); }  // (an empty sequence has results to write)
// What a head weighs where work is dealt out: its units, and as many again as loading its queries and putting its warps together take.
// Point kKv4Head + u of a head stands for unit u, the points before for its beginning.
constexpr int kKv4Head = 4;
__device__ __forceinline__ int kv4_weight(int len) { return kv4_units(len) + kKv4Head; }
// The points of all heads cut into runs as even as they come (fewer than 2^31 points; no run is empty).
struct Kv4Runs {
    int runs, each, more;  // the first `more` runs have a point more
    __device__ __forceinline__ Kv4Runs(int most, int points) : runs(min(most, points)), each(points / runs), more(points - each * runs) {}
    __device__ __forceinline__ int begin(int i) const { return i * each + min(i, more); }
    __device__ __forceinline__ int of(int point) const {
        const int longer = more * (each + 1);
        return point < longer ? point / (each + 1) : more + (point - longer) / each;
    }
};
// Weight of all sequences for one head, by a warp.
__device__ __forceinline__ int kv4_total(const Kv4AttnArgs& a) {
    int n = 0;
    for (int b = threadIdx.x & 31; b < a.batch; b += 32) n += kv4_weight(kv4_len(a, b));
    return __reduce_add_sync(0xffffffffu, n);
}
// Sequence that holds point `at` of all, and its first point, by a warp; `heads` counts a key/value head once per eight query heads.
__device__ __forceinline__ int kv4_find(const Kv4AttnArgs& a, int heads, int at, int& first) {
    const int lane = threadIdx.x & 31;
    int base = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 32) {
        const int own = b0 + lane < a.batch ? kv4_weight(kv4_len(a, b0 + lane)) * heads : 0;
        int x = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        const unsigned there = __ballot_sync(0xffffffffu, base + x > at);
        if (there) {
            const int from = __ffs(there) - 1;
            first = base + __shfl_sync(0xffffffffu, x - own, from);
            return b0 + from;
        }
        base += __shfl_sync(0xffffffffu, x, 31);
    }
    first = base;
    return a.batch;
}

template <int NG>
constexpr int kKv4StageBytes = 2 * kKv4Unit * kv4_row_bytes(NG);  // keys, then values
template <int NG>
constexpr int kKv4Pitch = NG * 32 + 4;
template <int NG>
constexpr int kv4_sums_bytes(int heads) {  // of the warps, for up to eight heads
    return kKv4Warps * heads * kKv4Pitch<NG> * 4;
}

__device__ __forceinline__ float load_typed(const void* p, long long i, int dtype) {
    if (dtype == 1) return __half2float(reinterpret_cast<const __half*>(p)[i]);
    if (dtype == 2) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
    return reinterpret_cast<const float*>(p)[i];
}
__device__ __forceinline__ void store_typed(void* p, long long i, int dtype, float x) {
    if (dtype == 1)
        reinterpret_cast<__half*>(p)[i] = __float2half_rn(x);
    else if (dtype == 2)
        reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
    else
        reinterpret_cast<float*>(p)[i] = x;
}
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// d = a . b
__device__ __forceinline__ void kv4_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// d += a . b
__device__ __forceinline__ void kv4_mma_add(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// d += a . b in BF16
__device__ __forceinline__ void kv4_mma_add_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {  // 8 x 8 matrix of 16-bit elements spread over a warp
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
    uint32_t r;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(r) : "r"(a));
    return r;
}
__device__ __forceinline__ uint32_t lds16(uint32_t a) {
    uint16_t r;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(r) : "r"(a));
    return r;
}
// Scales and zeros of a row, a word a group
template <int NG>
__device__ __forceinline__ void kv4_params(uint32_t a, uint32_t (&w)[NG]) {
    if constexpr (NG % 4 == 0) {
#pragma unroll
        for (int i = 0; i < NG; i += 4) asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3]) : "r"(a + i * 4));
    } else if constexpr (NG == 2) {
        asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(a));
    } else {
#pragma unroll
        for (int i = 0; i < NG; ++i) w[i] = lds32(a + i * 4);
    }
}
template <bool TRANS>
__device__ __forceinline__ void ldmatrix4(uint32_t a, uint32_t (&r)[4]) {
    if constexpr (TRANS)
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
    else
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}
// Words of the codes of a tile, [group][half of the rows].  Keys: word t of rows g and g + 8.  Values: 16-bit piece g of rows 2 t (lower
// half) and 2 t + 1, and of the rows 8 further.
template <int NG, bool VALUES>
__device__ __forceinline__ void kv4_codes(uint32_t tile, int lane, uint32_t (&w)[NG][2]) {
    constexpr int kRow = kv4_row_bytes(NG);
    if constexpr (kRow % 16 == 0) {
        const uint32_t a = tile + ((lane & 7) + (lane & 8)) * kRow + (lane >> 4) * 16;
#pragma unroll
        for (int i = 0; i < NG; i += 2) {
            uint32_t r[4];
            ldmatrix4<VALUES>(a + i * 16, r);
            w[i][0] = r[0], w[i][1] = r[1], w[i + 1][0] = r[2], w[i + 1][1] = r[3];
        }
    } else {
        const int g = lane >> 2, t = lane & 3;
        const uint32_t a = VALUES ? tile + 2 * t * kRow + g * 2 : tile + g * kRow + t * 4;
#pragma unroll
        for (int i = 0; i < NG; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                w[i][h] = VALUES ? lds16(a + i * 16 + h * 8 * kRow) | lds16(a + i * 16 + (h * 8 + 1) * kRow) << 16 : lds32(a + i * 16 + h * 8 * kRow);
    }
}
// (n - 8) of the codes in bits 0-3 and 16-19, and in bits 4-7 and 20-23: 1024 + n - 1032, (1024 + 16 n) / 16 - 72, both exact.  The
// constants travel in registers of unknown content: as immediates mask and exponent would be two instructions.
struct Kv4Magic {
    uint32_t exponent = 0x64006400u, f = 0x2c002c00u /* 1/16 */, off = 0xd480d480u /* -72 */;
    __device__ __forceinline__ void hide() { asm volatile("" : "+r"(exponent), "+r"(f), "+r"(off)); }
};
__device__ __forceinline__ uint32_t kv4_low(uint32_t x, const Kv4Magic& c) {
    uint32_t b;
    asm("lop3.b32 %0, %1, 0x000f000f, %2, 0xea;" : "=r"(b) : "r"(x), "r"(c.exponent));  // (x & mask) | exponent
    const uint32_t off = 0x64086408u;
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&b), *reinterpret_cast<const __half2*>(&off));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t kv4_high(uint32_t x, const Kv4Magic& c) {
    uint32_t b;
    asm("lop3.b32 %0, %1, 0x00f000f0, %2, 0xea;" : "=r"(b) : "r"(x), "r"(c.exponent));
    const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&b), *reinterpret_cast<const __half2*>(&c.f), *reinterpret_cast<const __half2*>(&c.off));
    return *reinterpret_cast<const uint32_t*>(&r);
}
// (n - 8) in BF16 of the codes in bits 0-3 and 16-19: 128 + n - 136
__device__ __forceinline__ uint32_t kv4_bf16(uint32_t x, uint32_t exponent /* 0x43004300 */) {
    uint32_t b;
    asm("lop3.b32 %0, %1, 0x000f000f, %2, 0xea;" : "=r"(b) : "r"(x), "r"(exponent));
    const uint32_t off = 0x43084308u;
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&b), *reinterpret_cast<const __nv_bfloat162*>(&off));
    return *reinterpret_cast<const uint32_t*>(&r);
}
// The upper eight bits of the significands of x and y as a pair of BF16 numbers; x and y keep the rest.  Three times, and there is none.
__device__ __forceinline__ uint32_t kv4_part(float& x, float& y) {
    const uint32_t u = __float_as_uint(x), w = __float_as_uint(y);
    x = __fsub_rn(x, __uint_as_float(u & 0xffff0000u));
    y = __fsub_rn(y, __uint_as_float(w & 0xffff0000u));
    return __byte_perm(u, w, 0x7632);
}

// Barriers by address in shared memory (as pointers, their address is put together again at every use)
__device__ __forceinline__ bool kv4_try_wait(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return done != 0;
}
__device__ __forceinline__ bool kv4_wait(uint32_t bar, uint32_t parity) {  // bounded; the same answer for the whole warp
    if (__all_sync(0xffffffffu, kv4_try_wait(bar, parity))) return true;
    const long long t0 = clock64();
    bool done = false;
    while (!(done = kv4_try_wait(bar, parity)) && clock64() - t0 < kWaitCycles) {
    }
    return __all_sync(0xffffffffu, done);
}
__device__ __forceinline__ void kv4_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }

struct Kv4Ahead {
    int b, len, head, at, put;  // the next unit to be requested, and its place in the ring
};

// CLUSTER: the units of a head go to the CTAs of a cluster, which put their results together through distributed shared memory and
// need no second kernel.  For caches of up to two units a CTA: with more, the runs are the more even ones.  (One sequence at 641 positions of
// a cache of 2048, 1B shape: 6.5 us, in runs 8.1.)
constexpr int kKv4Cluster = 8, kKv4ClusterUnits = 2;
template <int NG, bool SPLIT, bool CLUSTER>
static __global__ void __launch_bounds__(kKv4Threads, kKv4Ctas<NG>) kv4_attn_kernel(const Kv4AttnArgs a) {
    constexpr int kRow = kv4_row_bytes(NG), kStage = kKv4StageBytes<NG>, kParts = SPLIT ? 2 : 1, kPitch = kKv4Pitch<NG>;
    constexpr float kUnit = SPLIT ? 1.f : 0x1p24f;  // of the keys' codes as operands
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float s_m[kKv4Warps][kKv4Heads], s_l[kKv4Warps][kKv4Heads];
    __shared__ uint64_t full[kKv4MaxStages], empty[kKv4MaxStages];
    __shared__ Kv4Ahead ahead;
    __shared__ int s_fail;
    // SPLIT: of every warp, group and pair of heads 2 t, 2 t + 1: factors of the group's scores, and sums Q of its queries
    __shared__ float4 s_q[SPLIT ? kKv4Warps : 1][SPLIT ? NG : 1][4];
    __shared__ float c_y[CLUSTER ? kKv4Heads * NG * 32 : 1], c_ml[kKv4Heads][2];                  // this CTA's sums, reference and sum of probabilities
    __shared__ float c_w[CLUSTER ? kKv4Heads : 1][kKv4Cluster + 2];                               // weights of the CTAs; reference, 1 / sum of all
    pdl_wait();
    pdl_launch_dependents();  // (after the wait: what the finishing kernel reads of the lengths is there when it starts)
    int lane = threadIdx.x & 31;
    asm volatile("" : "+r"(lane));  // (kept, not made again from the special register in every tile)
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), g = lane >> 2, t = lane & 3;
    const int heads8 = a.kv_heads * a.head_tiles;
    // (sequence, head, unit) of the first unit, and of the one behind the last
    struct Place {
        int b, len, head, unit;
    };
    Place p_begin, p_end;
    if constexpr (CLUSTER) {
        const int at = blockIdx.x / a.cluster, rank = blockIdx.x - at * a.cluster;
        p_begin.b = at / heads8;
        p_begin.head = at - p_begin.b * heads8;
        p_begin.len = kv4_len(a, p_begin.b);
        p_end = p_begin;
        p_begin.unit = kv4_units(p_begin.len) * rank / a.cluster;
        p_end.unit = kv4_units(p_begin.len) * (rank + 1) / a.cluster;
    } else {
        const Kv4Runs runs(a.runs, kv4_total(a) * heads8);
        if ((int)blockIdx.x >= runs.runs) return;
        auto place = [&](int at) {
            int first = 0;
            Place p;
            p.b = kv4_find(a, heads8, at, first);
            p.len = p.b < a.batch ? kv4_len(a, p.b) : 0;
            const int weight = kv4_weight(p.len);
            p.head = (at - first) / weight;
            p.unit = max(0, at - first - p.head * weight - kKv4Head);
            return p;
        };
        p_begin = place(runs.begin(blockIdx.x));
        p_end = place(runs.begin(blockIdx.x + 1));
        if (p_begin.b == p_end.b && p_begin.head == p_end.head && p_begin.unit == p_end.unit) return;
    }
    float* so = reinterpret_cast<float*>(smem + a.stages * kStage);
    if (tid == 0) {
        s_fail = 0;
        for (int i = 0; i < a.stages; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], kKv4Warps);
        }
        mbar_fence_init();
    }
    __syncthreads();
    int b = p_begin.b, len = p_begin.len, units = kv4_units(len), head = p_begin.head, unit = p_begin.unit;

    // one lane: requests the next unit that has positions.  The warps take turns (one that always did it would hold the others up); how far
    // the requests are stands in shared memory.
    auto request = [&]() {
        Kv4Ahead x = ahead;
        bool done = false;
        while (!done && (x.b < p_end.b || (x.b == p_end.b && (x.head < p_end.head || (x.head == p_end.head && x.at < p_end.unit * kKv4Unit))))) {
            if (x.at < x.len) {
                const long long from = (((long long)x.b * a.kv_heads + x.head / a.head_tiles) * a.capacity + x.at) * kRow;
                const uint32_t bytes = (uint32_t)(min(kKv4Unit, (x.len - x.at + 3) & ~3) * kRow);  // (the capacity is a multiple of four rows)
                unsigned char* to = smem + x.put * kStage;
                mbar_arrive_expect_tx(&full[x.put], 2 * bytes);
                bulk_g2s(to, a.k + from, bytes, &full[x.put]);
                bulk_g2s(to + kStage / 2, a.v + from, bytes, &full[x.put]);
                if (++x.put == a.stages) x.put = 0;
                done = true;
            }
            if ((x.at += kKv4Unit) >= x.len) {  // the next head
                x.at = 0;
                if (++x.head == heads8) {
                    x.head = 0;
                    if (++x.b < a.batch) x.len = kv4_len(a, x.b);
                }
            }
        }
        ahead = x;
    };
    uint32_t full_at = smem_u32(full), empty_at = smem_u32(empty), ring_at = smem_u32(smem) + warp * kKv4Tile * kRow;
    asm volatile("" : "+r"(full_at), "+r"(empty_at), "+r"(ring_at));
    if (tid == 0) {
        ahead = {b, len, head, unit * kKv4Unit, 0};
        for (int i = 0; i < a.stages; ++i) request();
    }
    bool ok = true;
    int stage = 0, stage_before = -1, turn = 0;
    uint32_t phase = 0, phase_before = 0;

    Kv4Magic magic;
    magic.hide();
    uint32_t magic_bf16 = 0x43004300u;
    asm volatile("" : "+r"(magic_bf16));

    while (CLUSTER || b < p_end.b || (b == p_end.b && (head < p_end.head || (head == p_end.head && unit < p_end.unit)))) {
        const int kvh = head / a.head_tiles, tile8 = head - kvh * a.head_tiles;
        const int h0 = kvh * a.gqa + tile8 * kKv4Heads, n_heads = min(kKv4Heads, a.gqa - tile8 * kKv4Heads);
        const long long row0 = ((long long)b * a.kv_heads + kvh) * a.capacity;
        const int mine = (b == p_end.b && head == p_end.head ? p_end.unit : units) - unit, p1 = len;
        // queries: head g of the tile, dimensions 8 t .. 8 t + 7 of every group, times a power of two that makes the largest (SPLIT: of the group)
        // 2^6 .. 2^7 (eight times their sums over a group stay in the FP16 range)
        uint32_t qf[kParts][NG][4];
        float rate[2];  // (not SPLIT) factor of the scores, heads 2 t and 2 t + 1
        uint32_t zf[NG > 4 ? 2 : 1][2];  // operand of (scale, zero), head g: (-8 Q, Q) of group t, and of the rest of Q after FP16 (more than 4 groups: group t + 4)
        {
            float x[NG][8], tops[NG], top = 0.f;
            const bool some = g < n_heads;
#pragma unroll
            for (int i = 0; i < NG; ++i) {
                tops[i] = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int d = i * 32 + t * 8 + j;
                    x[i][j] = some && d < a.head_size ? load_typed(a.q, (long long)b * a.q_stride + (long long)(h0 + g) * a.head_size + d, a.dtype) : 0.f;
                    tops[i] = fmaxf(tops[i], fabsf(x[i][j]));
                }
                if constexpr (SPLIT) {
                    tops[i] = fmaxf(tops[i], __shfl_xor_sync(0xffffffffu, tops[i], 1));
                    tops[i] = fmaxf(tops[i], __shfl_xor_sync(0xffffffffu, tops[i], 2));
                }
                top = fmaxf(top, tops[i]);
            }
            if constexpr (!SPLIT) {
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            }
            // exponents of 2 in two halves, either within the normal range
            auto exponent = [](float y) { return y > 0.f && y < INFINITY ? 6 - ilogbf(y) : 0; };
            auto power = [](int e) { return __int_as_float((127 + e) << 23); };
            // back from the operands' factors: 2^24 / 2^e (finite: beyond, scores are alike, or so far apart that one position wins)
            auto back_from = [&](int e) { return fminf(power(-(e / 2)) * a.rate * power(-(e - e / 2)) * kUnit, 3.402823466e38f); };
            const int e_all = exponent(top);
            float sums[NG];
#pragma unroll
            for (int i = 0; i < NG; ++i) {
                const int e = SPLIT ? exponent(tops[i]) : e_all;
                const float f0 = power(e / 2), f1 = power(e - e / 2);
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < 4; ++j) {  // register j: dimensions j and j + 4; odd ones meet codes times 16 (SPLIT: none)
                    const bool sixteenth = !SPLIT && (j & 1);
                    const float f = sixteenth ? 1.f / 16.f : 1.f;
                    const float u = x[i][j] * f0 * f1, w = x[i][j + 4] * f0 * f1;
                    const __half2 hi = __floats2half2_rn(u * f, w * f);
                    const float2 hf = __half22float2(hi);
                    qf[0][i][j] = *reinterpret_cast<const uint32_t*>(&hi);
                    if constexpr (SPLIT) {
                        const __half2 lo = __floats2half2_rn(u - hf.x, w - hf.y);
                        qf[1][i][j] = *reinterpret_cast<const uint32_t*>(&lo);
                        sum += u + w;
                    } else {
                        sum += (hf.x + hf.y) * (sixteenth ? 16.f : 1.f);
                    }
                }
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                sums[i] = sum;
                if constexpr (SPLIT)
                    if ((i & 3) == t) {
                        float* to = reinterpret_cast<float*>(&s_q[warp][i][g >> 1]) + (g & 1);
                        to[0] = back_from(e);
                        to[2] = sum;
                    }
            }
            if constexpr (SPLIT) {
                __syncwarp();
            } else {
                const float back = back_from(e_all);
#pragma unroll
                for (int j = 0; j < 2; ++j) rate[j] = __shfl_sync(0xffffffffu, back, (2 * t + j) * 4);
            }
            float own[NG > 4 ? 2 : 1] = {};
#pragma unroll
            for (int i = 0; i < NG; ++i)
                if ((i & 3) == t) own[i >> 2] = sums[i];
#pragma unroll
            for (int i = 0; i < (NG > 4 ? 2 : 1); ++i) {
                const __half hi = __float2half_rn(own[i]), lo = __float2half_rn(own[i] - __half2float(hi));
                const __half times = __float2half_rn(-8.f);
                const __half2 both = __halves2half2(__hmul(hi, times), hi), rest = __halves2half2(__hmul(lo, times), lo);
                zf[0][i] = *reinterpret_cast<const uint32_t*>(&both);
                zf[NG > 4 ? 1 : 0][NG > 4 ? i : 1] = *reinterpret_cast<const uint32_t*>(&rest);
            }
        }

        float o[2 * NG][4], z[NG][2], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 2 * NG; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
#pragma unroll
        for (int i = 0; i < NG; ++i) z[i][0] = z[i][1] = 0.f;

        float* scores = a.scores ? a.scores + (row0 + unit * kKv4Unit + warp * kKv4Tile + g) * a.gqa + tile8 * kKv4Heads + 2 * t : nullptr;
        auto tile = [&](auto whole, int at) {  // whole: every row lies below the length
            constexpr bool kWhole = decltype(whole)::value;
            const bool in0 = kWhole || at + g < p1, in1 = kWhole || at + g + 8 < p1;
            const uint32_t sk = ring_at + stage * kStage, sv = sk + kStage / 2;
            // ---- scores of rows g and g + 8
            float s[4];
            {
                uint32_t w[NG][2], p0[NG], p1w[NG];
                kv4_codes<NG, false>(sk, lane, w);
                const uint32_t r0 = sk + g * kRow + NG * 16, r1 = r0 + 8 * kRow;  // scales and zeros
                kv4_params<NG>(r0, p0);
                kv4_params<NG>(r1, p1w);
                float zacc[4], acc[NG][4];
                if constexpr (!SPLIT) {  // rows of (scale, zero) pairs as they lie there times (-8 Q, Q)
                    if constexpr (NG > 4) {
                        const uint32_t a0 = lds32(r0 + t * 4), a1 = lds32(r1 + t * 4), a2 = lds32(r0 + 16 + t * 4), a3 = lds32(r1 + 16 + t * 4);
                        kv4_mma(zacc, a0, a1, a2, a3, zf[0][0], zf[0][1]);
                        kv4_mma_add(zacc, a0, a1, a2, a3, zf[1][0], zf[1][1]);
                    } else {
                        const uint32_t a0 = t < NG ? lds32(r0 + t * 4) : 0u, a1 = t < NG ? lds32(r1 + t * 4) : 0u;
                        kv4_mma(zacc, a0, a1, a0, a1, zf[0][0], zf[0][1]);
                    }
                }
                // (the groups' chains of products side by side)
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int gr = 0; gr < NG; ++gr) {
                        const uint32_t x0 = w[gr][0] >> (8 * half), x1 = w[gr][1] >> (8 * half);
                        uint32_t a0, a1, a2, a3;
                        if constexpr (SPLIT)
                            a0 = kv4_low(x0, magic), a1 = kv4_low(x1, magic), a2 = kv4_high(x0, magic), a3 = kv4_high(x1, magic);
                        else
                            a0 = x0 & 0x000f000fu, a1 = x1 & 0x000f000fu, a2 = x0 & 0x00f000f0u, a3 = x1 & 0x00f000f0u;
                        if (half == 0)
                            kv4_mma(acc[gr], a0, a1, a2, a3, qf[0][gr][0], qf[0][gr][1]);
                        else
                            kv4_mma_add(acc[gr], a0, a1, a2, a3, qf[0][gr][2], qf[0][gr][3]);
                        if constexpr (SPLIT) kv4_mma_add(acc[gr], a0, a1, a2, a3, qf[1][gr][2 * half], qf[1][gr][2 * half + 1]);
                    }
#pragma unroll
                for (int j = 0; j < 4; ++j) s[j] = SPLIT ? 0.f : zacc[j] * (1.f / kUnit);
#pragma unroll
                for (int gr = 0; gr < NG; ++gr) {
                    const float2 u0 = half2_bits_to_float2(p0[gr]), u1 = half2_bits_to_float2(p1w[gr]);
                    if constexpr (SPLIT) {
                        const float4 f = s_q[warp][gr][t];
                        s[0] = fmaf(f.x, fmaf(u0.x, acc[gr][0], u0.y * f.z), s[0]);
                        s[1] = fmaf(f.y, fmaf(u0.x, acc[gr][1], u0.y * f.w), s[1]);
                        s[2] = fmaf(f.x, fmaf(u1.x, acc[gr][2], u1.y * f.z), s[2]);
                        s[3] = fmaf(f.y, fmaf(u1.x, acc[gr][3], u1.y * f.w), s[3]);
                    } else {
                        s[0] = fmaf(u0.x, acc[gr][0], s[0]);
                        s[1] = fmaf(u0.x, acc[gr][1], s[1]);
                        s[2] = fmaf(u1.x, acc[gr][2], s[2]);
                        s[3] = fmaf(u1.x, acc[gr][3], s[3]);
                    }
                }
            }
            if constexpr (!SPLIT) {
#pragma unroll
                for (int j = 0; j < 4; ++j) s[j] *= rate[j & 1];
            }
            if constexpr (!kWhole) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (!(j < 2 ? in0 : in1)) s[j] = -INFINITY;
            }
            if (a.scores) {
                if (2 * t + 1 < n_heads && a.gqa % 2 == 0) {
                    if (in0) *reinterpret_cast<float2*>(scores) = make_float2(s[0], s[1]);
                    if (in1) *reinterpret_cast<float2*>(scores + 8 * a.gqa) = make_float2(s[2], s[3]);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if ((j < 2 ? in0 : in1) && 2 * t + (j & 1) < n_heads) scores[(j >> 1) * 8 * a.gqa + (j & 1)] = s[j];
                }
                scores += (long long)kKv4Unit * a.gqa;
            }
            // ---- scales and zeros of the values of the same rows; beyond the end the rows may hold anything
            uint32_t vp[2][NG], codes[NG][2];
            kv4_codes<NG, true>(sv, lane, codes);
            float top[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                kv4_params<NG>(sv + (g + r * 8) * kRow + NG * 16, vp[r]);
                if (!(r ? in1 : in0)) {
#pragma unroll
                    for (int gr = 0; gr < NG; ++gr) vp[r][gr] = 0u;
                }
                __half2 most = *reinterpret_cast<const __half2*>(&vp[r][0]);
#pragma unroll
                for (int gr = 1; gr < NG; ++gr) most = __hmax2(most, *reinterpret_cast<const __half2*>(&vp[r][gr]));
                top[r] = fmaxf(__low2float(most), 0x1p-24f);
            }
            float p[4];  // (a row beyond the end: 0, or NaN while there is no reference, which the vote takes)
#pragma unroll
            for (int j = 0; j < 4; ++j) p[j] = exp2_fast(s[j] - m[j & 1]);
            if (__any_sync(0xffffffffu, !(fmaxf(p[0], p[1]) * top[0] <= kKv4Limit) || !(fmaxf(p[2], p[3]) * top[1] <= kKv4Limit))) {
                // move the reference: the largest product becomes 2^8 .. 2^9
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float x = fmaxf(s[j] + (float)(ilogbf(top[0]) - 8), s[j + 2] + (float)(ilogbf(top[1]) - 8));
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
                    const float next = fmaxf(m[j], x), f = m[j] == -INFINITY ? 0.f : exp2_fast(m[j] - next);
                    m[j] = next;
                    l[j] *= f;
#pragma unroll
                    for (int k = 0; k < 2 * NG; ++k) {
                        o[k][j] *= f;
                        o[k][j + 2] *= f;
                    }
#pragma unroll
                    for (int k = 0; k < NG; ++k) z[k][j] *= f;
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) p[j] = exp2_fast(s[j] - m[j & 1]);
            }
            l[0] += p[0] + p[2];
            l[1] += p[1] + p[3];
            // ---- values
            uint32_t pf[NG][2];  // probabilities times scales as operands: rows as the codes have them
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) {
                const float2 u = half2_bits_to_float2(vp[0][gr]), w = half2_bits_to_float2(vp[1][gr]);
                z[gr][0] = fmaf(p[2], w.y, fmaf(p[0], u.y, z[gr][0]));
                z[gr][1] = fmaf(p[3], w.y, fmaf(p[1], u.y, z[gr][1]));
                float y0 = p[0] * u.x, y1 = p[1] * u.x, y2 = p[2] * w.x, y3 = p[3] * w.x;
                if constexpr (SPLIT) {
                    uint32_t part[3][2];
#pragma unroll
                    for (int i = 0; i < 3; ++i) {
                        part[i][0] = transpose8(kv4_part(y0, y1));
                        part[i][1] = transpose8(kv4_part(y2, y3));
                    }
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const uint32_t xa = codes[gr][0] >> (8 * k), xb = codes[gr][1] >> (8 * k);
                        const uint32_t a0 = kv4_bf16(xa, magic_bf16), a1 = kv4_bf16(xa >> 4, magic_bf16), a2 = kv4_bf16(xb, magic_bf16), a3 = kv4_bf16(xb >> 4, magic_bf16);
#pragma unroll
                        for (int i = 0; i < 3; ++i) kv4_mma_add_bf16(o[2 * gr + k], a0, a1, a2, a3, part[i][0], part[i][1]);
                    }
                } else {
                    const __half2 ha = __floats2half2_rn(y0, y1), hb = __floats2half2_rn(y2, y3);
                    pf[gr][0] = transpose8(*reinterpret_cast<const uint32_t*>(&ha));
                    pf[gr][1] = transpose8(*reinterpret_cast<const uint32_t*>(&hb));
                }
            }
            if constexpr (!SPLIT) {
#pragma unroll
                for (int gr = 0; gr < NG; ++gr)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const uint32_t xa = codes[gr][0] >> (8 * k), xb = codes[gr][1] >> (8 * k);
                        const uint32_t a0 = kv4_low(xa, magic), a1 = kv4_high(xa, magic), a2 = kv4_low(xb, magic), a3 = kv4_high(xb, magic);
                        kv4_mma_add(o[2 * gr + k], a0, a1, a2, a3, pf[gr][0], pf[gr][1]);
                    }
            }
        };
        const int unit_end = min(p1, (unit + mine) * kKv4Unit);
        for (int unit_at = unit * kKv4Unit; unit_at < unit_end; unit_at += kKv4Unit) {
            const int at = unit_at + warp * kKv4Tile;
            ok = ok && kv4_wait(full_at + stage * 8, phase);
            if (!ok) {  // a copy that never came: the results of this run say so
                m[0] = m[1] = NAN;
                s_fail = 1;
                break;
            }
            if (at + kKv4Tile <= p1)
                tile(std::true_type(), at);
            else if (at < p1)
                tile(std::false_type(), at);
            __syncwarp();
            // the unit before has been read by all warps but late ones: its place takes the next
            if (turn == warp && stage_before >= 0) {
                ok = kv4_wait(empty_at + stage_before * 8, phase_before);
                if (lane == 0 && ok) request();
                __syncwarp();
            }
            if (lane == 0) kv4_arrive(empty_at + stage * 8);  // (after the request: who makes the next one sees how far it came)
            turn = (turn + 1) & (kKv4Warps - 1);
            stage_before = stage;
            phase_before = phase;
            if (++stage == a.stages) {
                stage = 0;
                phase ^= 1u;
            }
        }
        // ---- the warp's sums over its lanes, then the CTA's over its warps
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) l[j] += __shfl_xor_sync(0xffffffffu, l[j], d);
#pragma unroll
            for (int k = 0; k < NG; ++k)
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) z[k][j] += __shfl_xor_sync(0xffffffffu, z[k][j], d);
            if (g == 0) {
                s_m[warp][2 * t + j] = m[j];
                s_l[warp][2 * t + j] = l[j];
            }
        }
#pragma unroll
        for (int gr = 0; gr < NG; ++gr)
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int j = 0; j < 4; ++j)  // tile 2 gr + k: rows g and g + 8 are dimensions 4 g + 2 k and the one after
                    if (2 * t + (j & 1) < n_heads) so[(warp * n_heads + 2 * t + (j & 1)) * kPitch + gr * 32 + 4 * g + 2 * k + (j >> 1)] = o[2 * gr + k][j] + z[gr][j & 1];
        __syncthreads();
        const bool whole = unit == 0 && mine == units;  // the head lies in this run; else a part: [1] begins here, [0] began earlier
        const long long part = (long long)blockIdx.x * 2 + (unit == 0 ? 1 : 0);
        for (int i = tid; i < n_heads * NG * 32; i += kKv4Threads) {
            const int h = i / (NG * 32), d = i - h * (NG * 32);
            float top = -INFINITY, sum = 0.f, y = 0.f;
#pragma unroll
            for (int w = 0; w < kKv4Warps; ++w) top = fmaxf(top, s_m[w][h]);
#pragma unroll
            for (int w = 0; w < kKv4Warps; ++w) {
                const float f = s_m[w][h] == -INFINITY ? 0.f : exp2_fast(s_m[w][h] - top);
                sum = fmaf(f, s_l[w][h], sum);
                y = fmaf(f, so[(w * n_heads + h) * kPitch + d], y);
            }
            const long long bh = (long long)b * a.heads + h0 + h;
            if constexpr (CLUSTER) {
                c_y[i] = y;
                if (d == 0) {
                    c_ml[h][0] = top;
                    c_ml[h][1] = sum;
                }
            } else if (!whole) {
                a.part_o[(part * kKv4Heads + h) * (NG * 32) + d] = y;
                if (d == 0) a.part_ml[part * kKv4Heads + h] = make_float2(top, sum);
            } else {
                if (d < a.head_size) store_typed(a.out, (long long)b * a.out_stride + (long long)(h0 + h) * a.head_size + d, a.dtype, len > 0 ? __fdiv_rn(y, sum) : 0.f);
                if (d == 0 && a.whole_ml) a.whole_ml[bh] = make_float2(top, sum);
            }
        }
        if constexpr (CLUSTER) {
            cluster_barrier();  // every CTA's results are there
            const int rank = blockIdx.x % a.cluster;
            if (tid < n_heads) {
                float ml[kKv4Cluster][2], top = -INFINITY, sum = 0.f;
#pragma unroll
                for (int c = 0; c < kKv4Cluster; ++c)
                    if (c < a.cluster) {
                        const uint32_t at = cluster_map(smem_u32(&c_ml[tid][0]), c);
                        ml[c][0] = __uint_as_float(kv4_cluster_load(at));
                        ml[c][1] = __uint_as_float(kv4_cluster_load(at + 4));
                    }
#pragma unroll
                for (int c = 0; c < kKv4Cluster; ++c)
                    if (c < a.cluster) top = fmaxf(top, ml[c][0]);
#pragma unroll
                for (int c = 0; c < kKv4Cluster; ++c)
                    if (c < a.cluster) {
                        const float f = ml[c][0] == -INFINITY ? 0.f : exp2_fast(ml[c][0] - top);
                        c_w[tid][c] = f;
                        sum = fmaf(f, ml[c][1], sum);
                    }
                c_w[tid][kKv4Cluster] = top;
                c_w[tid][kKv4Cluster + 1] = __fdiv_rn(1.f, sum);
            }
            __syncthreads();
            for (int i = rank * kKv4Threads + tid; i < n_heads * NG * 32; i += a.cluster * kKv4Threads) {
                const int h = i / (NG * 32), d = i - h * (NG * 32);
                float y[kKv4Cluster], sum = 0.f;
#pragma unroll
                for (int c = 0; c < kKv4Cluster; ++c) y[c] = c < a.cluster ? __uint_as_float(kv4_cluster_load(cluster_map(smem_u32(&c_y[i]), c))) : 0.f;
#pragma unroll
                for (int c = 0; c < kKv4Cluster; ++c)
                    if (c < a.cluster) sum = fmaf(c_w[h][c], y[c], sum);
                if (d < a.head_size)
                    store_typed(a.out, (long long)b * a.out_stride + (long long)(h0 + h) * a.head_size + d, a.dtype, len > 0 ? sum * c_w[h][kKv4Cluster + 1] : 0.f);
            }
            if (a.sums_out) {  // (up to eight query heads: this CTA has all scores of its positions)
                for (int p = unit * kKv4Unit + tid; p < min(len, p_end.unit * kKv4Unit); p += kKv4Threads) {
                    const float* x = a.scores + (row0 + p) * a.gqa;
                    float sum = 0.f;
                    for (int h = 0; h < a.gqa; ++h) sum = fmaf(exp2_fast(x[h] - c_w[h][kKv4Cluster]), c_w[h][kKv4Cluster + 1], sum);
                    a.sums_out[row0 + p] = (a.sums_in ? a.sums_in[row0 + p] : 0.f) + sum;
                }
            }
            cluster_barrier();  // every CTA's shared memory stays until all have read it
            break;
        }
        __syncthreads();  // the sums have been read
        unit += mine;
        if (unit == units) {
            unit = 0;
            if (++head == heads8) {
                head = 0;
                if (++b < a.batch) len = kv4_len(a, b);
                units = kv4_units(len);
            }
        } else {
            break;
        }
    }
    if (s_fail) {  // copies may still be in flight: a bounded time to land
        const long long c0 = clock64();
        while (clock64() - c0 < (1 << 17)) __nanosleep(1000);
    }
}

// Puts the parts of heads together that lie in several runs (the first gqa blocks of a key/value head), and adds the probabilities of its
// queries to the sums of its positions (the others).  Grid (gqa + blocks of positions, kv_heads, batch).
constexpr int kKv4FinishThreads = 256, kKv4FinishRows = 512;
template <int NG>
static __global__ void __launch_bounds__(kKv4FinishThreads) kv4_finish_kernel(const Kv4AttnArgs a) {
    extern __shared__ float s_fin[];  // [gqa][2]: reference, 1 / sum; then [runs]: weights of the parts
    __shared__ float s_part[kKv4FinishThreads / 32][NG * 32];
    pdl_launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, kvh = blockIdx.y, b = blockIdx.z, heads8 = a.kv_heads * a.head_tiles;
    const int len = kv4_len(a, b), units = kv4_units(len), weight = kv4_weight(len), row_block = (int)blockIdx.x - a.gqa;
    if (row_block * kKv4FinishRows >= len && row_block >= 0) return;  // (others of the grid wait for the kernel before)
    const Kv4Runs runs(a.runs, kv4_total(a) * heads8);
    int before = 0;
    for (int i = lane; i < b; i += 32) before += kv4_weight(kv4_len(a, i));
    before = __reduce_add_sync(0xffffffffu, before);
    // runs that hold the first and the last unit of a head
    auto runs_of = [&](int tile8, int& r0, int& r1) {
        const int u0 = before * heads8 + (kvh * a.head_tiles + tile8) * weight + kKv4Head;
        r0 = runs.of(u0);
        r1 = runs.of(u0 + units - 1);
    };
    auto part_of = [&](int r, int r0, int h) { return ((long long)r * 2 + (r == r0 ? 1 : 0)) * kKv4Heads + h % kKv4Heads; };
    int r0, r1;
    if (row_block < 0) {
        runs_of((int)blockIdx.x / kKv4Heads, r0, r1);
        if (r0 == r1) {
            pdl_wait();
            return;  // written already
        }
    }
    pdl_wait();
    // rows of four scores are on their way while the references are put together
    constexpr int kRows = kKv4FinishRows / kKv4FinishThreads;
    const long long row0 = ((long long)b * a.kv_heads + kvh) * a.capacity;
    const bool four = a.gqa == 4;
    auto own = [&](int j) { return row_block * kKv4FinishRows + tid + j * kKv4FinishThreads; };
    float4 early[kRows];
    float before_in[kRows] = {};
    if (row_block >= 0 && four) {
#pragma unroll
        for (int j = 0; j < kRows; ++j)
            if (own(j) < len) {
                early[j] = *reinterpret_cast<const float4*>(a.scores + (row0 + own(j)) * 4);
                if (a.sums_in) before_in[j] = a.sums_in[row0 + own(j)];
            }
    }
    // reference and sum of the head, or of all heads where their probabilities are wanted
    for (int h = row_block < 0 ? (int)blockIdx.x + warp : warp; h < (row_block < 0 ? (int)blockIdx.x + 1 : a.gqa); h += kKv4FinishThreads / 32) {
        runs_of(h / kKv4Heads, r0, r1);
        float top = -INFINITY, sum = 0.f;
        if (r0 == r1) {
            if (a.whole_ml) {
                const float2 ml = a.whole_ml[(long long)b * a.heads + kvh * a.gqa + h];
                top = ml.x;
                sum = ml.y;
            }
        } else {
            float2 ml = make_float2(-INFINITY, 0.f);
            if (r0 + lane <= r1) ml = a.part_ml[part_of(r0 + lane, r0, h)];
            top = ml.x;
            for (int r = r0 + 32 + lane; r <= r1; r += 32) top = fmaxf(top, a.part_ml[part_of(r, r0, h)].x);
            top = warp_max(top);
            const float w = exp2_fast(ml.x - top);
            sum = w * ml.y;
            if (row_block < 0 && r0 + lane <= r1) s_fin[2 * a.gqa + lane] = w;
            for (int r = r0 + 32 + lane; r <= r1; r += 32) {
                const float2 more = a.part_ml[part_of(r, r0, h)];
                const float x = exp2_fast(more.x - top);
                sum = fmaf(x, more.y, sum);
                if (row_block < 0) s_fin[2 * a.gqa + r - r0] = x;
            }
            sum = warp_sum(sum);
        }
        if (lane == 0) {
            s_fin[2 * h] = top;
            s_fin[2 * h + 1] = __fdiv_rn(1.f, sum);
        }
    }
    __syncthreads();
    if (row_block < 0) {  // a warp takes every eighth part, a lane NG dimensions
        const int h = blockIdx.x;
        runs_of(h / kKv4Heads, r0, r1);
        float y[NG] = {};
#pragma unroll 4
        for (int r = r0 + warp; r <= r1; r += kKv4FinishThreads / 32) {
            const float w = s_fin[2 * a.gqa + r - r0];
            const float* po = a.part_o + part_of(r, r0, h) * (NG * 32) + lane;
#pragma unroll
            for (int k = 0; k < NG; ++k) y[k] = fmaf(w, po[k * 32], y[k]);
        }
#pragma unroll
        for (int k = 0; k < NG; ++k) s_part[warp][k * 32 + lane] = y[k];
        __syncthreads();
        for (int d = tid; d < a.head_size; d += kKv4FinishThreads) {
            float x = 0.f;
#pragma unroll
            for (int w = 0; w < kKv4FinishThreads / 32; ++w) x += s_part[w][d];
            store_typed(a.out, (long long)b * a.out_stride + (long long)(kvh * a.gqa + h) * a.head_size + d, a.dtype, x * s_fin[2 * h + 1]);
        }
        return;
    }
    if (four) {
#pragma unroll
        for (int j = 0; j < kRows; ++j)
            if (own(j) < len) {
                const float sum = fmaf(exp2_fast(early[j].x - s_fin[0]), s_fin[1], fmaf(exp2_fast(early[j].y - s_fin[2]), s_fin[3], fmaf(exp2_fast(early[j].z - s_fin[4]), s_fin[5],
                                       exp2_fast(early[j].w - s_fin[6]) * s_fin[7])));
                a.sums_out[row0 + own(j)] = before_in[j] + sum;
            }
        return;
    }
    for (int p = own(0); p < min(len, (row_block + 1) * kKv4FinishRows); p += kKv4FinishThreads) {
        const float* x = a.scores + (row0 + p) * a.gqa;
        float sum = 0.f;
        if (a.gqa % 4 == 0) {  // 16 bytes at once (F16, 32769 positions, groups of 8: 18.0 us, one by one 19.6; 131071, groups of 32: 69 and 106)
            for (int h = 0; h < a.gqa; h += 4) {
                const float4 v = *reinterpret_cast<const float4*>(x + h);
                sum = fmaf(exp2_fast(v.x - s_fin[2 * h]), s_fin[2 * h + 1], sum);
                sum = fmaf(exp2_fast(v.y - s_fin[2 * h + 2]), s_fin[2 * h + 3], sum);
                sum = fmaf(exp2_fast(v.z - s_fin[2 * h + 4]), s_fin[2 * h + 5], sum);
                sum = fmaf(exp2_fast(v.w - s_fin[2 * h + 6]), s_fin[2 * h + 7], sum);
            }
        } else {
            for (int h = 0; h < a.gqa; ++h) sum = fmaf(exp2_fast(x[h] - s_fin[2 * h]), s_fin[2 * h + 1], sum);
        }
        a.sums_out[row0 + p] = (a.sums_in ? a.sums_in[row0 + p] : 0.f) + sum;
    }
}

// ------------------------------------------------------------------ eviction
//
// Keeps the `recent` last rows of every head and, of the rows before them, those with the largest sums (the lowest position first among
// equals; a NaN counts as -infinity), in their order.  A cluster of CTAs takes a head, every CTA a run of its rows: the smallest sum that
// stays is found digit by digit (histograms of 8 bits of the sums' order, every CTA adding up all of the cluster's through distributed
// shared memory), then every CTA knows where its kept rows begin in the new cache and lists them.  A second kernel, of many small CTAs,
// moves many of them: bound by the rows' bytes where they are many, by the meetings of the cluster where they are few.  (Digits of 11 bits added
// up by remote atomics in one CTA: passes of 3 - 8 us each instead of 1.4.  Rows moved by the cluster that lists them, two sequences of
// 32768 and 20011 positions to 12000: 30 us, its SMs being too few for the bandwidth; now 26.)
// 512 threads: two CTAs fit an SM (of 1024, sixteen clusters of eight did not fit the GPU at once, and the last ran alone).
// A head has as many CTAs, up to eight, as give every CTA of the call an SM: of sequences of eight heads two get clusters of eight, four clusters of four,
// nine of two, more a CTA a head, whose sums beyond 4096 rows are read again in every pass.  1, 2, 3, 9 and 16 sequences of 32768 positions to
// 12000: 19.5, 27.6, 40.5, 94 and 152 us, their bytes 5 us a sequence.
constexpr int kKv4EvictThreads = 512, kKv4EvictCluster = 8;
constexpr int kKv4EvictKeep = 8;  // rows of a thread whose ranks stay in registers
constexpr int kKv4EvictMove = 256;  // new rows a CTA up to which one kernel does it all

struct Kv4EvictArgs {
    const unsigned char *k, *v;
    unsigned char *k_out, *v_out;
    const float* sums;
    float* sums_out;
    int *kept, *lens_out;
    const int* lens;
    long long capacity, capacity_out;
    int kv_heads, keep, recent, row_bytes, cluster;
};

// Order of the sums as unsigned integers
__device__ __forceinline__ uint32_t kv4_rank(float x) {
    const uint32_t u = x != x ? 0xff800000u : __float_as_uint(x + 0.f);  // (-0 becomes 0)
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
// Rows first .. first + n - 1 of the new cache, by one CTA
template <typename V, int UNITS>
__device__ __forceinline__ void kv4_move_rows(const Kv4EvictArgs& a, long long head, int first, int n) {
    const int* kept = a.kept + head * a.keep + first;
    const V *k = reinterpret_cast<const V*>(a.k) + head * a.capacity * UNITS, *v = reinterpret_cast<const V*>(a.v) + head * a.capacity * UNITS;
    V *ko = reinterpret_cast<V*>(a.k_out) + (head * a.capacity_out + first) * UNITS, *vo = reinterpret_cast<V*>(a.v_out) + (head * a.capacity_out + first) * UNITS;
#pragma unroll 4
    for (int i = threadIdx.x; i < n * UNITS; i += kKv4EvictThreads) {
        const int row = i / UNITS;
        const long long from = (long long)kept[row] * UNITS + (i - row * UNITS);
        const V x = k[from], y = v[from];
        ko[i] = x;
        vo[i] = y;
    }
    for (int i = threadIdx.x; i < n; i += kKv4EvictThreads) a.sums_out[head * a.capacity_out + first + i] = a.sums[head * a.capacity + kept[i]];
}
// MOVE: the CTAs also move the rows that they list, and there is no second kernel, whose launch takes the host 2.3 us.  For few rows.  (2048
// to 1024 positions, eight heads: calls behind one another 8.7 us, with two kernels 11; four sequences of 4096 to 1024 in a graph 9.4, 11.7;
// 32768 to 2048, as many as are moved so, 11.6 and 11.1.)
template <bool MOVE>
static __global__ void __launch_bounds__(kKv4EvictThreads, 2) kv4_select_kernel(const Kv4EvictArgs a) {
    __shared__ uint32_t hist[4][256], parts[2][256];  // hist: a pass each
    __shared__ uint32_t counts[kKv4EvictCluster][2], warp_sums[32], s_digit, s_left, s_all;
    pdl_wait();
    pdl_launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, cta = blockIdx.x % a.cluster, kvh = blockIdx.y, b = blockIdx.z;
    const int len = (int)max(0ll, min((long long)a.lens[b], a.capacity)), stay = min(len, a.keep), old = max(0, len - a.recent);
    const long long head = (long long)b * a.kv_heads + kvh;
    const float* sums = a.sums + head * a.capacity;
    int* kept = a.kept + head * a.keep;
    if (cta == 0 && kvh == 0 && tid == 0) a.lens_out[b] = stay;
    const int each = ((len + a.cluster - 1) / a.cluster + 31) & ~31, row0 = min(len, cta * each), row1 = min(len, row0 + each);
    uint32_t rank[kKv4EvictKeep];
#pragma unroll
    for (int j = 0; j < kKv4EvictKeep; ++j) {
        const int i = row0 + tid + j * kKv4EvictThreads;
        rank[j] = i < min(row1, old) ? kv4_rank(sums[i]) : 0u;
    }
    hist[tid >> 8][tid & 255] = hist[2 + (tid >> 8)][tid & 255] = 0;
    if (tid < 32) warp_sums[tid] = 0;
    __syncthreads();
    // the choose-th largest rank of the `old` first rows
    const uint32_t choose = (uint32_t)max(0, stay - (len - old));
    const bool every = choose >= (uint32_t)old, none = choose == 0;
    uint32_t prefix = 0, mask = 0, left = choose;
    if (!every && !none) {  // (the same for the whole cluster)
        const int end = min(row1, old);
#pragma unroll 1
        for (int pass = 0; pass < 4; ++pass) {
            const int shift = 24 - 8 * pass;
#pragma unroll
            for (int j = 0; j < kKv4EvictKeep; ++j)
                if (row0 + tid + j * kKv4EvictThreads < end && (rank[j] & mask) == prefix) atomicAdd(&hist[pass][rank[j] >> shift & 255u], 1u);
            for (int i = row0 + tid + kKv4EvictKeep * kKv4EvictThreads; i < end; i += kKv4EvictThreads) {
                const uint32_t r = kv4_rank(sums[i]);
                if ((r & mask) == prefix) atomicAdd(&hist[pass][r >> shift & 255u], 1u);
            }
            cluster_barrier();  // every CTA has started, and counted
            const int digit = 255 - (tid & 255);  // from the top
            uint32_t y[kKv4EvictCluster / 2], x = 0;
#pragma unroll
            for (int j = 0; j < kKv4EvictCluster / 2; ++j) {
                const int c = (tid >> 8) + 2 * j;
                y[j] = c < a.cluster ? kv4_cluster_load(cluster_map(smem_u32(&hist[pass][digit]), c)) : 0u;
            }
#pragma unroll
            for (int j = 0; j < kKv4EvictCluster / 2; ++j) x += y[j];
            parts[tid >> 8][tid & 255] = x;
            __syncthreads();
            uint32_t own = 0;
            if (tid < 256) {
                own = parts[0][tid] + parts[1][tid];
                x = own;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const uint32_t z = __shfl_up_sync(0xffffffffu, x, d);
                    if (lane >= d) x += z;
                }
                if (lane == 31) warp_sums[warp] = x;
            }
            __syncthreads();
            if (tid < 256) {
                x += __reduce_add_sync(0xffffffffu, lane < warp ? warp_sums[lane] : 0u);
                if (x - own < left && left <= x) {
                    s_digit = (uint32_t)digit;
                    s_left = left - (x - own);
                    s_all = s_left == own ? 1u : 0u;
                }
            }
            __syncthreads();
            prefix |= s_digit << shift;
            mask |= 255u << shift;
            left = s_left;
            if (s_all) break;  // all of these stay: further digits tell nothing apart
        }
    } else {
        cluster_barrier();  // every CTA has started
    }
    // rows with a larger rank stay, and the recent ones; of those that equal it the first `left`
    auto judge = [&](int i, uint32_t r, bool& more, bool& same) {
        const bool is_old = i < old;
        more = i < row1 && (!is_old || every || (!none && (r & mask) > prefix));
        same = i < row1 && is_old && !every && !none && (r & mask) == prefix;
    };
    auto rank_of = [&](int i) { return i < min(row1, old) ? kv4_rank(sums[i]) : 0u; };
    uint32_t n_more = 0, n_same = 0;
    auto count = [&](int i, uint32_t r) {
        bool more, same;
        judge(i, r, more, same);
        n_more += __popc(__ballot_sync(0xffffffffu, more));
        n_same += __popc(__ballot_sync(0xffffffffu, same));
    };
#pragma unroll
    for (int j = 0; j < kKv4EvictKeep; ++j) count(row0 + tid + j * kKv4EvictThreads, rank[j]);
    for (int i0 = row0 + kKv4EvictKeep * kKv4EvictThreads; i0 < row1; i0 += kKv4EvictThreads) count(i0 + tid, rank_of(i0 + tid));
    constexpr int kWarps = kKv4EvictThreads / 32;
    if (lane == 0) parts[0][warp] = n_more, parts[0][32 + warp] = n_same;
    __syncthreads();
    if (warp == 0) {
        n_more = __reduce_add_sync(0xffffffffu, lane < kWarps ? parts[0][lane] : 0u);
        n_same = __reduce_add_sync(0xffffffffu, lane < kWarps ? parts[0][32 + lane] : 0u);
        if (lane < a.cluster) {  // to every CTA of the cluster
            const uint32_t to = cluster_map(smem_u32(&counts[cta][0]), lane);
            asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to), "r"(n_more) : "memory");
            asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to + 4), "r"(n_same) : "memory");
        }
    }
    cluster_barrier();  // (also the last time that another CTA's shared memory is touched)
    uint32_t at = 0, equal = 0;
    for (int c = 0; c < cta; ++c) at += counts[c][0], equal += counts[c][1];
    at += min(equal, left);
    const int first = (int)at;
    auto place = [&](int i, uint32_t r) {
        bool more, same;
        judge(i, r, more, same);
        const uint32_t bm = __ballot_sync(0xffffffffu, more), bs = __ballot_sync(0xffffffffu, same), below = (1u << lane) - 1u;
        __syncthreads();
        if (lane == 0) warp_sums[warp] = (uint32_t)__popc(bm) | (uint32_t)__popc(bs) << 16;
        __syncthreads();
        const uint32_t w = lane < kWarps ? warp_sums[lane] : 0u, before = __reduce_add_sync(0xffffffffu, lane < warp ? w : 0u), total = __reduce_add_sync(0xffffffffu, w);
        const uint32_t eq = equal + (before >> 16) + __popc(bs & below);  // equals before this row
        const uint32_t to = at + (before & 0xffffu) + __popc(bm & below) + min(eq, left) - min(equal, left);
        if (more || (same && eq < left)) kept[to] = i;
        at += (total & 0xffffu) + min(equal + (total >> 16), left) - min(equal, left);
        equal += total >> 16;
    };
#pragma unroll
    for (int j = 0; j < kKv4EvictKeep; ++j)
        if (row0 + j * kKv4EvictThreads < row1) place(row0 + tid + j * kKv4EvictThreads, rank[j]);  // (the same for the whole CTA)
    for (int i0 = row0 + kKv4EvictKeep * kKv4EvictThreads; i0 < row1; i0 += kKv4EvictThreads) place(i0 + tid, rank_of(i0 + tid));
    if constexpr (MOVE) {
        __syncthreads();  // the list is there
        const int n = (int)at - first;
        switch (a.row_bytes) {
            case kv4_row_bytes(1): kv4_move_rows<uint32_t, 5>(a, head, first, n); break;
            case kv4_row_bytes(2): kv4_move_rows<uint2, 5>(a, head, first, n); break;
            case kv4_row_bytes(3): kv4_move_rows<uint32_t, 15>(a, head, first, n); break;
            case kv4_row_bytes(4): kv4_move_rows<uint4, 5>(a, head, first, n); break;
            default: kv4_move_rows<uint4, 10>(a, head, first, n);
        }
    }
}

// V: bytes a thread moves at once (16, 8 or 4, by the row's size), UNITS of them a row.  A CTA takes 256 rows, a thread UNITS pieces of the
// keys and of the values, all on their way at once.  Grid (blocks of rows, kv_heads, batch).
constexpr int kKv4MoveRows = 256;
template <typename V, int UNITS>
static __global__ void __launch_bounds__(kKv4MoveRows) kv4_move_kernel(const Kv4EvictArgs a) {
    pdl_launch_dependents();
    const int tid = threadIdx.x, kvh = blockIdx.y, b = blockIdx.z, row0 = blockIdx.x * kKv4MoveRows;
    const long long head = (long long)b * a.kv_heads + kvh;
    const int rows = (int)max(0ll, min(min((long long)a.lens[b], a.capacity), (long long)a.keep)) - row0;
    const int* kept = a.kept + head * a.keep + row0;
    const V *k = reinterpret_cast<const V*>(a.k) + head * a.capacity * UNITS, *v = reinterpret_cast<const V*>(a.v) + head * a.capacity * UNITS;
    V *ko = reinterpret_cast<V*>(a.k_out) + (head * a.capacity_out + row0) * UNITS, *vo = reinterpret_cast<V*>(a.v_out) + (head * a.capacity_out + row0) * UNITS;
    constexpr int kAhead = UNITS > 5 ? 5 : UNITS;
    pdl_wait();
    if (tid < rows) a.sums_out[head * a.capacity_out + row0 + tid] = a.sums[head * a.capacity + kept[tid]];
#pragma unroll
    for (int j0 = 0; j0 < UNITS; j0 += kAhead) {
        long long from[kAhead];
        V x[kAhead], y[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int i = tid + (j0 + j) * kKv4MoveRows, row = i / UNITS;
            from[j] = row < rows ? (long long)kept[row] * UNITS + (i - row * UNITS) : -1;
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            if (from[j] >= 0) {
                x[j] = k[from[j]];
                y[j] = v[from[j]];
            }
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            if (from[j] >= 0) {
                ko[tid + (j0 + j) * kKv4MoveRows] = x[j];
                vo[tid + (j0 + j) * kKv4MoveRows] = y[j];
            }
    }
}

}  // namespace lpp
