// tsrc_fa4_tc.cu -- attention over the q4_0 KV cache with many query rows on one stretch of cells (prompts), on the
// fifth-generation tensor cores. Layout of the cache: tsrc_kv4.cuh; the entry point and the rule that chooses
// between this kernel and the one for few rows: tsrc_fa4.cu.
//
// A CTA takes 128 query rows -- the (token, head) pairs of a group that share a KV head -- or two lots of 128 that share
// the dequantized tiles (bf16 outputs, where that fills the SMs), and passes over the cells they span in tiles of 64, its
// warps in three roles that hand over by mbarriers:
//   dequant (4 or 8 warps)  codes and scales from global memory (a tile ahead, in registers) to fp16 operands in
//                      shared memory: K as [8 values][cell][16 B], V transposed as [8 cells][value][16 B], the
//                      tensor cores' unswizzled layout, every 16-byte store of a quarter warp side by side. Two buffers
//                      each.
//   products (1 thread)  S(i + 1) = Q K^T while the softmax of tile i runs, then O += P(i) V; S twice and O in tensor
//                      memory, P written over its S.
//   softmax (4 warps for 128 rows)  a thread per row: scores from tensor memory, running sum, weights back as fp16.
// The reference that the weights' exponents are taken from follows the running maximum only when that has risen by
// 8 (in log2): outputs in tensor memory are then rescaled, seldom after the first tiles; up to there weights reach
// 2^8, which fp16 holds, and results do not depend on the reference.
//   Range: q is scaled by a power of two per row; K and V go in as 2^7 d (n - 8), which fills fp16 from scales of 32
// down (2^7 32 8 = 2^15) to the smallest that the cache can hold (2^-24: an operand of 2^-17, a normal number from 2^-21 on),
// so that no block's scale costs another block's digits, in its cell or elsewhere. A cell with a scale of 32 and above, which
// no row of ordinary size has, gets a power of two of its own, which its scores and weights make good: rows that do not
// see it keep their digits (beside one of 2^15, a block of the same cell keeps all of its own down to 2^-10). Precision:
// bf16 outputs take one fp16 term (11 bits) of q (exact), K, V and the weights. f32 and f16 outputs take two terms of each, 22
// bits (d (n - 8) has 15, so K and V are exact), and three products, the one of the two small terms left out: 2^-22 of the result.
#include <cfloat>
#include <type_traits>

#include "tsrc_fa4.cuh"

namespace tsrc {

namespace {

__device__ unsigned int g_fa4_error;                 // kKv4ErrWait once a wait ran out

constexpr uint32_t kTile = 64, kRows = 128;
constexpr long long kWaitCycles = 1ll << 31;         // a wait gives up after ~1 s of SM clock

template <class T, int D, bool MASK, uint32_t RG> struct TcShape {                        // RG: lots of 128 rows
    static constexpr bool PRECISE = !std::is_same_v<T, __nv_bfloat16>;              // two terms of K, V and the weights
    static constexpr bool TOTAL = std::is_same_v<T, float>;                         // two of q (fp16 is one), outputs in total
    static constexpr uint32_t NB = D / 32, TERMS = PRECISE ? 2 : 1;
    static constexpr uint32_t Q_TERM = kRows * D * 2, KV_TERM = kTile * D * 2;      // bytes of one term of an operand
    static constexpr uint32_t Q_ROWS = Q_TERM * (TOTAL ? 2 : 1), K_AT = Q_ROWS * RG, V_AT = K_AT + 2 * KV_TERM * TERMS;
    static constexpr uint32_t CTL_AT = V_AT + 2 * KV_TERM * TERMS;
    // two CTAs an SM at most, or one that takes all of tensor memory. Two lots of rows take four dequant warps: with eight
    // the registers a thread may have, 96, do not hold a row's scores (2048 tokens: 71.3 us, 68.6 with four).
    static constexpr uint32_t WANT = CTL_AT + 4096;
    static constexpr uint32_t MIN_CTAS = RG == 1 && !MASK && 2 * (WANT + 1024) <= 227 * 1024 ? 2 : 1;
    static constexpr uint32_t LEAST = MIN_CTAS == 2 ? 100 * 1024 : 116 * 1024, BYTES = WANT < LEAST ? LEAST : WANT;
    static constexpr uint32_t DW = MIN_CTAS == 1 && RG == 1 ? 8 : 4, SW = 4 * RG;              // dequant, softmax warps
    static constexpr uint32_t WARPS = SW + DW + 1, THREADS = 32 * WARPS;
    static constexpr uint32_t KU = 8 / DW, BV = 8 / DW;                             // a lane's cells of K, blocks of V
    // tensor-memory columns: score buffers (P over each) of each lot of rows, then the outputs. With four buffers S(i + 1)
    // need not wait for the products of P(i - 1), and the tensor cores never stop; two CTAs or two lots of rows have room
    // for two each.
    static constexpr uint32_t NS = MIN_CTAS == 1 && RG == 1 ? 4 : 2, O_COL = RG * NS * kTile, COLUMNS = MIN_CTAS == 1 ? 512 : 256;
    // The tensor cores cut every sum towards zero, about 2^-25 of it a product, so a row's output would shrink by 1e-5
    // over 60 tiles of twelve products. For f32 outputs FLUSH tiles are added up there, and then to the total, in tensor
    // memory too, by an ordinary f32 addition.
    static constexpr uint32_t FLUSH = 4, SUM_COL = O_COL + D;
    static_assert(O_COL + RG * D <= COLUMNS && SUM_COL + (TOTAL ? D : 0) <= COLUMNS && (RG == 1 || !TOTAL), "tensor memory");
};

constexpr int kOperandExp = 7;       // K and V operands are 2^7 of the values
// What the dequant warps tell of a tile: each of its own cells, 64 / DW in a row.
struct __align__(8) TileInfo {
    uint8_t flags[8];        // kBad, kFar
};
constexpr uint32_t kBad = 1;         // a scale of V that is no number or infinite is there (its block is 0 in the operand)
constexpr uint32_t kFar = 2;         // a scale above the common ones is there: the cells' own powers of two count
constexpr uint32_t kFarExp = 19;     // exponent field of scales of 16 to 32, the largest common ones

struct Control {                     // at most 4 KB
    uint64_t k_full[2], k_free[2], v_full[2], v_free[2];
    uint64_t s_full[2][4], p_full[2][4], o_done[2][2];    // of a lot of rows
    TileInfo info[4];
    // far tiles: what a cell's scores are times, and what the log2 of its weights is raised by. Of four tiles, as info:
    // the dequant warps are up to two tiles ahead of the softmax when they write these.
    float cell_k[4][kTile], cell_v[4][kTile];
    uint32_t tmem, abort;
    int32_t span[8][2];      // the softmax warps' first and last cell
    float q_unscale[2 * kRows];
    uint64_t drained;        // the products in flight when a wait ran out
    uint32_t never;          // stays 0
};

static_assert(sizeof(Control) <= 4096, "room behind the operands");

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint64_t* b, uint32_t n) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(b)), "r"(n) : "memory"); }
__device__ __forceinline__ void bar_arrive(uint64_t* b) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(b)) : "memory"); }
// Waits for the phase of that parity; false when about a second passed or another role gave up.
__device__ __forceinline__ bool bar_wait(uint64_t* b, uint32_t parity, volatile uint32_t* abort) {
    long long t0 = 0;
    for (uint32_t it = 0;; ++it) {
        uint32_t ok;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(ok) : "r"(smem_u32(b)), "r"(parity) : "memory");
        if (ok) return true;
        if ((it & 63u) != 0u) continue;
        if (*abort) return false;
        if (it == 0) t0 = clock64();
        else if (clock64() - t0 > kWaitCycles) break;
    }
    *abort = 1u;
    atomicOr(&g_fa4_error, kKv4ErrWait);
    return false;
}
__device__ __forceinline__ void commit(uint64_t* b) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(b)) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// operand of `rows` rows in shared memory, 16-byte chunks of a row `rows` x 16 bytes apart, eight rows 128 bytes
__device__ __forceinline__ uint64_t operand(uint32_t at, uint32_t rows) {
    return (uint64_t)((at >> 4) & 0x3FFFu) | ((uint64_t)rows << 16) | ((uint64_t)(128u >> 4) << 32) | (1ull << 46);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
}
// f32 sums of fp16 products, 128 x n
__host__ __device__ constexpr uint32_t instruction(uint32_t n) { return (1u << 4) | ((n >> 3) << 17) | ((kRows >> 4) << 24); }

#define TSRC_R8(v, o) "=r"((v)[o]), "=r"((v)[o + 1]), "=r"((v)[o + 2]), "=r"((v)[o + 3]), "=r"((v)[o + 4]), "=r"((v)[o + 5]), "=r"((v)[o + 6]), "=r"((v)[o + 7])
#define TSRC_I8(v, o) "r"((v)[o]), "r"((v)[o + 1]), "r"((v)[o + 2]), "r"((v)[o + 3]), "r"((v)[o + 4]), "r"((v)[o + 5]), "r"((v)[o + 6]), "r"((v)[o + 7])
__device__ __forceinline__ void tmem_ld32(uint32_t at, uint32_t* v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : TSRC_R8(v, 0), TSRC_R8(v, 8), TSRC_R8(v, 16), TSRC_R8(v, 24) : "r"(at));
}
__device__ __forceinline__ void tmem_ld8(uint32_t at, uint32_t* v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];" : TSRC_R8(v, 0) : "r"(at));
}
__device__ __forceinline__ void tmem_st8(uint32_t at, const uint32_t* v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::TSRC_I8(v, 0), "r"(at) : "memory");
}
// Waits for the thread's loads; the registers go through it, so that nothing uses them before.
#define TSRC_P8(v, o) "+r"((v)[o]), "+r"((v)[o + 1]), "+r"((v)[o + 2]), "+r"((v)[o + 3]), "+r"((v)[o + 4]), "+r"((v)[o + 5]), "+r"((v)[o + 6]), "+r"((v)[o + 7])
__device__ __forceinline__ void tmem_wait_ld(uint32_t* v) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : TSRC_P8(v, 0), TSRC_P8(v, 8) :: "memory");
    asm volatile("" : TSRC_P8(v, 16), TSRC_P8(v, 24));
}
__device__ __forceinline__ void tmem_wait_ld8(uint32_t* v) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : TSRC_P8(v, 0) :: "memory");
}
__device__ __forceinline__ void tmem_wait_ld64(uint32_t* v) {
    tmem_wait_ld(v);
    asm volatile("" : TSRC_P8(v, 32), TSRC_P8(v, 40), TSRC_P8(v, 48), TSRC_P8(v, 56));
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
__device__ __forceinline__ __half2 as_h2(uint32_t u) { return *reinterpret_cast<const __half2*>(&u); }
__device__ __forceinline__ uint32_t as_u32(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }
// What a cell's scales are times, e (kFarExp to 30) the exponent field of the largest: 2^7, or what takes that to below 2^12.
__device__ __forceinline__ __half2 operand_factor(uint32_t e) {
    return __half2half2(__ushort_as_half((unsigned short)((15u + kOperandExp + kFarExp - e) << 10)));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
// Two f32 side by side: a b + c, a + b
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 y;
    asm("{\n\t.reg .b64 a, b, c, y;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\tfma.rn.f32x2 y, a, b, c;\n\tmov.b64 {%0, %1}, y;\n\t}"
        : "=f"(y.x), "=f"(y.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return y;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 y;
    asm("{\n\t.reg .b64 a, b, y;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 y, a, b;\n\tmov.b64 {%0, %1}, y;\n\t}"
        : "=f"(y.x), "=f"(y.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return y;
}
// the largest finite magnitude among the four halves of two words
__device__ __forceinline__ uint32_t finite_most(uint32_t u) {
    u &= 0x7FFF7FFFu;
    const uint32_t a = u & 0xFFFFu, b = u >> 16;
    return max(a < 0x7C00u ? a : 0u, b < 0x7C00u ? b : 0u);
}
__device__ __forceinline__ uint32_t finite_only(uint32_t u) {
    return ((u & 0x7C00u) == 0x7C00u ? 0u : u & 0xFFFFu) | ((u & 0x7C000000u) == 0x7C000000u ? 0u : u & 0xFFFF0000u);
}
// Codes i = 0..3 of two halves side by side (four bits each) times d, that is d (n - 8), as operand words: n - 8 without
// rounding from the fp16 whose last bits are n (1024 + n, or 1024 + 16 n with the code in the next four bits), then the rounded
// product and, of two terms, what it lacks.
template <bool PRECISE>
__device__ __forceinline__ void scaled(__half2 d, uint32_t x, uint32_t (&h)[4], uint32_t (&l)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t y = j & 2 ? x >> 8 : x;
        const __half2 n = j & 1 ? __hfma2(as_h2((y & 0x00F000F0u) | 0x64006400u), __float2half2_rn(0.0625f), __float2half2_rn(-72.0f))
                                : __hsub2(as_h2((y & 0x000F000Fu) | 0x64006400u), __float2half2_rn(1032.0f));
        const __half2 w = __hmul2(n, d);
        h[j] = as_u32(w);
        if (PRECISE) l[j] = as_u32(__hfma2(n, d, __hneg2(w)));
    }
}

// Eight cells of a row's mask from `cell` on, -inf where `seen` lacks the cell's bit (the mask there may hold anything).
// wide: the row holds all of the tile in aligned memory, and the load stands outside any branch, so that a tile's eight are
// under way together; every: no bit lacks.
__device__ __forceinline__ uint4 mask_of(const __half* row, int32_t cell, uint32_t seen, bool wide, bool every) {
    uint32_t w[4];
    if (wide) {
        const uint4 h = *reinterpret_cast<const uint4*>(row + cell);
        w[0] = h.x; w[1] = h.y; w[2] = h.z; w[3] = h.w;
    } else {
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            w[j] = seen >> (2 * j) & 1u ? __half_as_ushort(row[cell + 2 * (int32_t)j]) : 0u;
            if (seen >> (2 * j) & 2u) w[j] |= (uint32_t)__half_as_ushort(row[cell + 2 * (int32_t)j + 1]) << 16;
        }
    }
    if (!every) {
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            const uint32_t keep = (seen >> (2 * j) & 1u ? 0x0000FFFFu : 0u) | (seen >> (2 * j) & 2u ? 0xFFFF0000u : 0u);
            w[j] = (w[j] & keep) | (0xFC00FC00u & ~keep);
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// O times f
template <int D>
__device__ __forceinline__ void rescale(uint32_t o_at, float f) {
#pragma unroll 1
    for (uint32_t k = 0; k < D; k += 16) {
        uint32_t o[16];
        tmem_ld8(o_at + k, o);
        tmem_ld8(o_at + k + 8u, o + 8);
        tmem_wait_ld8(o);
        tmem_wait_ld8(o + 8);
#pragma unroll
        for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
        tmem_st8(o_at + k, o);
        tmem_st8(o_at + k + 8u, o + 8);
    }
}
// The total (none before the first) and O times f; flush: O goes into the total.
template <int D>
__device__ __forceinline__ void settle(uint32_t o_at, uint32_t sum_at, float f, bool none, bool flush) {
    if (none && !flush) return rescale<D>(o_at, f);
#pragma unroll 1
    for (uint32_t k = 0; k < D; k += 16) {
        uint32_t o[16], t[16];
        tmem_ld8(o_at + k, o);
        tmem_ld8(o_at + k + 8u, o + 8);
        tmem_ld8(sum_at + k, t);
        tmem_ld8(sum_at + k + 8u, t + 8);
        tmem_wait_ld8(o);
        tmem_wait_ld8(o + 8);
        tmem_wait_ld8(t);
        tmem_wait_ld8(t + 8);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const float x = __uint_as_float(o[j]), y = none ? 0.0f : __uint_as_float(t[j]);
            t[j] = __float_as_uint((flush ? x + y : y) * f);
            o[j] = __float_as_uint(x * f);
        }
        tmem_st8(sum_at + k, t);
        tmem_st8(sum_at + k + 8u, t + 8);
        if (!flush) {
            tmem_st8(o_at + k, o);
            tmem_st8(o_at + k + 8u, o + 8);
        }
    }
}

template <class T, int D, bool MASK, uint32_t RG>
__global__ void __launch_bounds__(TcShape<T, D, MASK, RG>::THREADS, TcShape<T, D, MASK, RG>::MIN_CTAS) fa4_tc_kernel(Fa4Args a) {
    using S = TcShape<T, D, MASK, RG>;
    constexpr bool PRECISE = S::PRECISE, TOTAL = S::TOTAL;
    constexpr uint32_t NB = S::NB;
    extern __shared__ __align__(1024) uint8_t sm[];
    Control& c = *reinterpret_cast<Control*>(sm + S::CTL_AT);
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    // the last rows first: in a causal prompt they see the most cells
    const uint32_t split = blockIdx.x % a.splits, place = blockIdx.x / a.splits;
    const uint32_t hk = place % a.n_head_kv, rest = place / a.n_head_kv;
    const uint32_t rt = a.row_tiles - 1u - rest % a.row_tiles, grp = rest / a.row_tiles;
    const uint32_t rows = a.group * a.G, row = rt * kRows * RG + tid;
    const uint32_t tok = grp * a.group + row / a.G, head = hk * a.G + row % a.G;

    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&c.tmem)), "n"(S::COLUMNS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        if (lane == 0) {
            c.abort = c.never = 0;
            for (int i = 0; i < 2; ++i) {
                bar_init(&c.k_full[i], S::DW);
                bar_init(&c.k_free[i], 1);
                bar_init(&c.v_full[i], S::DW);
                bar_init(&c.v_free[i], 1);
            }
            for (uint32_t i = 0; i < 4 * RG; ++i) {
                bar_init(&c.s_full[i / 4][i % 4], 2);      // the tensor cores, and the issuing thread for what it has seen
                bar_init(&c.p_full[i / 4][i % 4], 4);
            }
            for (uint32_t i = 0; i < 2 * RG; ++i) bar_init(&c.o_done[i / 2][i % 2], 1);
            bar_init(&c.drained, 1);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
    }
    int32_t lo = 0, hi = 0;
    if (warp < S::SW) {
        if (row < rows) {
            hi = (int32_t)a.n_kv;
            if (a.ranges) {
                lo = max(a.ranges[2u * (size_t)tok], 0);
                hi = min(a.ranges[2u * (size_t)tok + 1u], hi);
            }
            if (lo >= hi) lo = hi = 0;
        }
        const int32_t first = __reduce_min_sync(0xFFFFFFFFu, lo < hi ? lo : 0x7FFFFFFF), last = __reduce_max_sync(0xFFFFFFFFu, hi);
        if (lane == 0) {
            c.span[warp][0] = first;
            c.span[warp][1] = last;
        }
    }
    // q, eight rows at a time by a warp: the row's largest value to [2^12, 2^13), chunks of eight values in the order
    // 0 4 1 5 2 6 3 7 that K has
    for (uint32_t r0 = 8u * warp; warp < S::SW + S::DW && r0 < kRows * RG; r0 += 8u * (S::SW + S::DW)) {
        const uint32_t r = r0 + (lane & 7u), row_r = rt * kRows * RG + r;
        const uint32_t tok_r = grp * a.group + row_r / a.G, head_r = hk * a.G + row_r % a.G;
        const T* q = static_cast<const T*>(a.q) + (size_t)tok_r * a.q_stride + (size_t)head_r * D + 8u * (lane >> 3);
        float x[D / 32][8], top = 0.0f;
#pragma unroll
        for (uint32_t j = 0; j < D / 32; ++j) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[j][i] = 0.0f;
            if (row_r < rows) {
                if (a.q_wide) load8<T, true>(q + 32u * j, x[j]);
                else load8<T, false>(q + 32u * j, x[j]);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[j][i]));
        }
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 8));
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 16));
        const int e2 = min(12 - ((int)(__float_as_uint(top) >> 23) - 127), 100);
        const float f = copysignf(pow2(e2), a.scale);        // the factor that scores get is positive
        // cut to the largest finite factor: scores of 0 stay 0, and others are as far apart as any exponential can tell
        if (lane < 8) c.q_unscale[r] = fminf(fabsf(a.scale) * pow2(-e2) * (1.4426950408889634f / (1 << kOperandExp)), FLT_MAX);
#pragma unroll
        for (uint32_t j = 0; j < D / 32; ++j) {
            uint32_t h[4], l[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float u = x[j][i] * f, v = x[j][i + 4] * f;
                const __half2 w = __floats2half2_rn(u, v);
                h[i] = as_u32(w);
                if (TOTAL) {
                    const float2 back = __half22float2(w);
                    l[i] = as_u32(__floats2half2_rn(u - back.x, v - back.y));
                }
            }
            uint8_t* p = sm + r / kRows * S::Q_ROWS + (4u * j + (lane >> 3)) * (kRows * 16u) + r % kRows * 16u;
            *reinterpret_cast<uint4*>(p) = make_uint4(h[0], h[1], h[2], h[3]);
            if (TOTAL) *reinterpret_cast<uint4*>(p + S::Q_TERM) = make_uint4(l[0], l[1], l[2], l[3]);
        }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = c.tmem;
    int32_t first = c.span[0][0], last = c.span[0][1];
#pragma unroll
    for (uint32_t w = 1; w < S::SW; ++w) {
        first = min(first, c.span[w][0]);
        last = max(last, c.span[w][1]);
    }
    const uint32_t from = last > first ? (uint32_t)first / kTile : 0u;
    const uint32_t span = last > first ? ((uint32_t)last + kTile - 1u) / kTile - from : 0u;
    const uint32_t tile0 = from + (uint32_t)((uint64_t)span * split / a.splits);             // this split's tiles
    const uint32_t tiles = from + (uint32_t)((uint64_t)span * (split + 1u) / a.splits) - tile0;

    if (warp == S::SW + S::DW) {
        // ---- products, issued by one thread. Descriptors are made once and advanced by constants: made anew for every
        // product they cost the issuing thread 90 cycles each, more than a 128 x 64 x 16 product takes (48).
        uint32_t one;
        asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
        if (one) {
            const uint64_t q_op = operand(smem_u32(sm), kRows), k_op = operand(smem_u32(sm) + S::K_AT, kTile), v_op = operand(smem_u32(sm) + S::V_AT, D);
            auto scores = [&](uint32_t i, uint32_t rg) {   // S(i) of a lot of rows
                const uint32_t buf = i & 1u, sb = i % S::NS;
                // it takes the place of P(i - 2), or of P(i - 4): then the products of P(i - 3), the latest whose phase is
                // still the barrier's last, are waited for
                constexpr uint32_t BACK = S::NS == 2 ? 2 : 3;
                if (i >= BACK && !bar_wait(&c.o_done[rg][(i - BACK) & 1u], ((i - BACK) >> 1) & 1u, &c.abort)) return false;
                if (!bar_wait(&c.k_full[buf], (i >> 1) & 1u, &c.abort)) return false;
                fence_after();
                const uint64_t kb = k_op + buf * (S::KV_TERM * S::TERMS >> 4), qa = q_op + rg * (S::Q_ROWS >> 4);
                const uint32_t to = tmem + (rg * S::NS + sb) * kTile;
#pragma unroll
                for (uint32_t k = PRECISE ? 3 : 1; k-- > 0;) {         // q k_lo, q_lo k, q k: the small ones first, so that
                    if (k == 1 && !TOTAL) continue;                    // what is cut from them is small
#pragma unroll
                    for (uint32_t s = 0; s < D / 16; ++s)
                        mma_ss(to, qa + ((k == 1 ? S::Q_TERM : 0u) + s * 2u * kRows * 16u >> 4), kb + ((k == 2 ? S::KV_TERM : 0u) + s * 2u * kTile * 16u >> 4),
                               instruction(kTile), k != (PRECISE ? 2u : 0u) || s != 0u);
                }
                if (rg + 1u == RG) commit(&c.k_free[buf]);
                commit(&c.s_full[rg][sb]);
                bar_arrive(&c.s_full[rg][sb]);
                return true;
            };
            auto outputs = [&](uint32_t i, uint32_t rg) {  // O += P(i) V
                const uint32_t buf = i & 1u, sb = i % S::NS;
                if (!bar_wait(&c.v_full[buf], (i >> 1) & 1u, &c.abort) || !bar_wait(&c.p_full[rg][sb], (i / S::NS) & 1u, &c.abort)) return false;
                fence_after();
                const uint64_t vb = v_op + buf * (S::KV_TERM * S::TERMS >> 4);
                const uint32_t pa = tmem + (rg * S::NS + sb) * kTile;
#pragma unroll
                for (uint32_t k = PRECISE ? 3 : 1; k-- > 0;)           // p v_lo, p_lo v, p v
#pragma unroll
                    for (uint32_t s = 0; s < kTile / 16; ++s)
                        mma_ts(tmem + S::O_COL + rg * D, pa + (k == 1 ? kTile / 2u : 0u) + 8u * s, vb + ((k == 2 ? S::KV_TERM : 0u) + s * 2u * D * 16u >> 4),
                               instruction(D), k == (PRECISE ? 2u : 0u) && s == 0u ? (TOTAL ? i % S::FLUSH : i) : 1u);
                commit(&c.o_done[rg][buf]);
                if (rg + 1u == RG) commit(&c.v_free[buf]);
                return true;
            };
            bool ok = true;
            for (uint32_t rg = 0; ok && tiles && rg < RG; ++rg) ok = scores(0, rg);
            for (uint32_t i = 0; ok && i < tiles; ++i)
                for (uint32_t rg = 0; ok && rg < RG; ++rg) ok = (i + 1u == tiles || scores(i + 1u, rg)) && outputs(i, rg);
            if (!ok) {                                       // given up: what is in flight ends before the CTA leaves
                commit(&c.drained);
                bar_wait(&c.drained, 0, &c.never);
            }
        }
        __syncwarp();
    } else if (warp >= S::SW) {
        // ---- dequant
        constexpr uint32_t KU = S::KU, BV = S::BV;
        const uint32_t dw = warp - S::SW;
        // K: unit u is cell kc + 8 u, values 8t .. 8t + 7 of every block, t = lane / 8
        const uint32_t kt = lane >> 3, kc = 8u * KU * dw + (lane & 7u);
        const size_t plane = (size_t)hk * a.n_alloc + (size_t)tile0 * kTile;
        // V: cells 8 vg .. + 7, chunk g, BV blocks from vb on
        const uint32_t vg = BV == 2 ? 2u * dw + (lane >> 4) : dw, g = lane & 7u, vb = BV == 2 ? (lane >> 3 & 1u) * 2u : lane >> 3;
        const bool v_live = vb < NB;
        const uint8_t* kq = a.kq + (plane + kc) * (D / 2) + kv4_place(2u * kt, kc) * (NB * 2u);
        const __half* kd = a.kd + (plane + kc) * NB;
        const uint8_t* vq = a.vq + (plane + 8u * vg) * (D / 2) + 2u * (v_live ? vb : 0u);
        const __half* vd = a.vd + (plane + 8u * vg) * NB + (v_live ? vb : 0u);
        uint32_t kw[KU][NB], ks[KU][NB / 2], vw[8], vs[8];
        auto load_k = [&](uint32_t i) {
            const size_t o = (size_t)i * kTile;
#pragma unroll
            for (uint32_t u = 0; u < KU; ++u) {
                const uint8_t* p = kq + (o + 8u * u) * (D / 2);
                const __half* d = kd + (o + 8u * u) * NB;
                if constexpr (NB == 4) {
                    const uint4 x = *reinterpret_cast<const uint4*>(p);
                    const uint2 y = *reinterpret_cast<const uint2*>(d);
                    kw[u][0] = x.x; kw[u][1] = x.y; kw[u][2] = x.z; kw[u][3] = x.w;
                    ks[u][0] = y.x; ks[u][1] = y.y;
                } else {
                    const uint2 x = *reinterpret_cast<const uint2*>(p);
                    kw[u][0] = x.x; kw[u][1] = x.y;
                    ks[u][0] = *reinterpret_cast<const uint32_t*>(d);
                }
            }
        };
        auto load_v = [&](uint32_t i) {
            const size_t o = (size_t)i * kTile;
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k) {
                const uint8_t* p = vq + (o + k) * (D / 2) + kv4_place(g, k) * (NB * 2u);
                const __half* d = vd + (o + k) * NB;
                if constexpr (BV == 2) {
                    vw[k] = *reinterpret_cast<const uint32_t*>(p);
                    vs[k] = *reinterpret_cast<const uint32_t*>(d);
                } else {
                    vw[k] = *reinterpret_cast<const uint16_t*>(p);
                    vs[k] = *reinterpret_cast<const uint16_t*>(d);
                }
            }
        };
        bool ok = true;
        if (tiles) {
            load_k(0);
            load_v(0);
        }
#pragma unroll 1
        for (uint32_t i = 0; i < tiles; ++i) {
            const uint32_t buf = i & 1u, round = i >> 1;
            // the largest scales among the warp's cells
            __half2 mk = __float2half2_rn(0.0f), mv = mk;
#pragma unroll
            for (uint32_t u = 0; u < KU; ++u)
#pragma unroll
                for (uint32_t b = 0; b < NB / 2; ++b) mk = __hmax2_nan(mk, __habs2(as_h2(ks[u][b])));
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k) mv = __hmax2_nan(mv, __habs2(as_h2(vs[k])));
            const __half2 both = __hmax2_nan(mk, mv);
            bool bad = false, far = false;
            __half2 k_one[KU], v_one[4];             // powers of two that the scales are times
#pragma unroll
            for (uint32_t u = 0; u < KU; ++u) k_one[u] = operand_factor(kFarExp);
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) v_one[k] = operand_factor(kFarExp);
            if (__any_sync(0xFFFFFFFFu, max(as_u32(both) & 0xFFFFu, as_u32(both) >> 16) >= (kFarExp + 1u) << 10)) {        // seldom
                uint32_t x = 0, odd = 0;
#pragma unroll
                for (uint32_t u = 0; u < KU; ++u)
#pragma unroll
                    for (uint32_t b = 0; b < NB / 2; ++b) x = max(x, finite_most(ks[u][b]));
#pragma unroll
                for (uint32_t k = 0; k < 8; ++k) {
                    x = max(x, finite_most(vs[k]));
                    odd |= vs[k] ^ finite_only(vs[k]);
                }
                far = __any_sync(0xFFFFFFFFu, x >> 10 > kFarExp);
                bad = __any_sync(0xFFFFFFFFu, odd != 0);
            }
            if (lane == 0) c.info[i & 3u].flags[dw] = (uint8_t)((bad ? kBad : 0u) | (far ? kFar : 0u));
            if (far) {
#pragma unroll
                for (uint32_t u = 0; u < KU; ++u) {
                    uint32_t own = kFarExp;
#pragma unroll
                    for (uint32_t b = 0; b < NB / 2; ++b) own = max(own, finite_most(ks[u][b]) >> 10);
                    k_one[u] = operand_factor(own);
                    if (kt == 0) c.cell_k[i & 3u][kc + 8u * u] = pow2((int)(own - kFarExp));
                }
#pragma unroll
                for (uint32_t k = 0; k < 8; ++k) {
                    uint32_t x = finite_most(vs[k]);
#pragma unroll
                    for (uint32_t o = 8; o < (BV == 2 ? 16u : 32u); o <<= 1) x = max(x, __shfl_xor_sync(0xFFFFFFFFu, x, o));
                    const uint32_t own = max(kFarExp, x >> 10);
                    if (g == 0 && vb == 0) c.cell_v[i & 3u][8u * vg + k] = (float)(own - kFarExp);
                    const __half2 one = operand_factor(own);
                    v_one[k / 2] = k & 1u ? __lows2half2(v_one[k / 2], one) : __lows2half2(one, one);
                }
            }
            if (bad) {
#pragma unroll
                for (uint32_t k = 0; k < 8; ++k) vs[k] = finite_only(vs[k]);
            }
            // K
            if (i >= 2) ok = __all_sync(0xFFFFFFFFu, bar_wait(&c.k_free[buf], (round - 1u) & 1u, &c.abort));
            if (!ok) break;
            uint8_t* kb = sm + S::K_AT + buf * S::KV_TERM * S::TERMS;
#pragma unroll
            for (uint32_t u = 0; u < KU; ++u)
#pragma unroll
                for (uint32_t b = 0; b < NB; ++b) {
                    const uint32_t x = __byte_perm(kw[u][b / 2], kw[u][NB / 2 + b / 2], b & 1u ? 0x7632 : 0x5410);
                    const uint32_t s = ks[u][b / 2];
                    const __half2 d = __hmul2(as_h2(__byte_perm(s, s, b & 1u ? 0x3232 : 0x1010)), k_one[u]);
                    uint32_t h[4], l[4];
                    scaled<PRECISE>(d, x, h, l);
                    uint8_t* p = kb + (4u * b + kt) * (kTile * 16u) + (kc + 8u * u) * 16u;
                    *reinterpret_cast<uint4*>(p) = make_uint4(h[0], h[1], h[2], h[3]);
                    if (PRECISE) *reinterpret_cast<uint4*>(p + S::KV_TERM) = make_uint4(l[0], l[1], l[2], l[3]);
                }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) bar_arrive(&c.k_full[buf]);
            if (i + 1u < tiles) load_k(i + 1u);
            // V
            if (i >= 2) ok = __all_sync(0xFFFFFFFFu, bar_wait(&c.v_free[buf], (round - 1u) & 1u, &c.abort));
            if (!ok) break;
            uint32_t cw[8], cs[8];
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k) {
                cw[k] = vw[k];
                cs[k] = vs[k];
            }
            if (i + 1u < tiles) load_v(i + 1u);
            if (v_live) {
                uint8_t* vo = sm + S::V_AT + buf * S::KV_TERM * S::TERMS + vg * (D * 16u);
#pragma unroll
                for (uint32_t b = 0; b < BV; ++b) {
                    uint32_t h[4][4], l[4][4];       // [cell pair][value]
#pragma unroll
                    for (uint32_t k = 0; k < 4; ++k) {
                        const uint32_t x = __byte_perm(cw[2 * k], cw[2 * k + 1], b ? 0x7632 : 0x5410);
                        const __half2 d = __hmul2(as_h2(__byte_perm(cs[2 * k], cs[2 * k + 1], b ? 0x7632 : 0x5410)), v_one[k]);
                        scaled<PRECISE>(d, x, h[k], l[k]);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        // row j D / 4 + 8 (block) + g holds value 32 (block) + 4 g + j
                        uint8_t* p = vo + ((uint32_t)j * (D / 4) + 8u * (vb + b) + g) * 16u;
                        *reinterpret_cast<uint4*>(p) = make_uint4(h[0][j], h[1][j], h[2][j], h[3][j]);
                        if (PRECISE) *reinterpret_cast<uint4*>(p + S::KV_TERM) = make_uint4(l[0][j], l[1][j], l[2][j], l[3][j]);
                    }
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) bar_arrive(&c.v_full[buf]);
        }
        // the last tiles' buffers come free too before the CTA leaves, so that no arrival comes after it
        for (uint32_t b = 0; ok && dw == 0 && b < 2; ++b) {
            const uint32_t n = (tiles + 1u - b) >> 1;            // phases of buffer b
            if (n) ok = bar_wait(&c.k_free[b], (n - 1u) & 1u, &c.abort) && bar_wait(&c.v_free[b], (n - 1u) & 1u, &c.abort);
        }
        __syncwarp();
    } else {
        // ---- softmax: this thread's row
        const uint32_t rg = warp / 4u, mine = tmem + ((warp % 4u * 32u) << 16), o_at = mine + S::O_COL + rg * D;
        const float qs = c.q_unscale[tid];           // this row's scale, for scores in log2
        float m = -INFINITY, l = 0.0f;               // reference of the weights' exponents; running sum, both in units of 2^6 p
        float off = MASK ? -INFINITY : 0.0f;         // the mask's maximum so far: scores and m are relative to it
        // a thread without a row may load the last token's, and sees nothing of it
        const __half* mrow = MASK ? a.mask + (size_t)min(tok, a.T - 1u) * a.mask_stride : nullptr;
        uint32_t lost = 0;                           // blocks of V in which the row sees a scale that is no number
        bool ok = true;
        // the cells that all rows of the warp see; rows behind the group's last lose nothing
        const int32_t all_lo = __reduce_max_sync(0xFFFFFFFFu, row < rows ? lo : 0), all_hi = __reduce_min_sync(0xFFFFFFFFu, row < rows ? hi : 0x7FFFFFFF);
#pragma unroll 1
        for (uint32_t i = 0; ok && i < tiles; ++i) {
            const uint32_t buf = i & 1u, sb = i % S::NS, at = mine + (rg * S::NS + sb) * kTile;
            const int32_t c0 = (int32_t)((tile0 + i) * kTile);
            if (MASK && c0 + 2 * (int32_t)kTile <= (int32_t)a.n_kv)      // the next tile's mask, a line or two of this row
                asm volatile("prefetch.global.L1 [%0];" ::"l"(mrow + c0 + (int32_t)kTile));
            ok = __all_sync(0xFFFFFFFFu, bar_wait(&c.s_full[rg][sb], (i / S::NS) & 1u, &c.abort));
            if (!ok) break;
            fence_after();
            constexpr uint32_t GC = kTile / S::DW;   // cells of a dequant warp
            const TileInfo& info = c.info[i & 3u];
            float f = qs;                            // what scores are times
            uint32_t flags = 0;
#pragma unroll
            for (uint32_t w = 0; w < S::DW; w += 4) flags |= *reinterpret_cast<const uint32_t*>(info.flags + w);
            const bool open = c0 >= all_lo && c0 + (int32_t)kTile <= all_hi, far = flags & kFar * 0x01010101u, bad = flags & kBad * 0x01010101u;
            if (far) {                               // seldom: scores with the cells' own powers of two, put back for what follows
#pragma unroll 1
                for (uint32_t k = 0; k < kTile; k += 8) {
                    const bool own = info.flags[k / GC] & kFar;
                    uint32_t x[8];
                    tmem_ld8(at + k, x);
                    tmem_wait_ld8(x);
#pragma unroll
                    for (uint32_t j = 0; j < 8; ++j) {
                        const float z = __uint_as_float(x[j]) * qs;
                        x[j] = __float_as_uint(own ? fmaf(z, c.cell_k[i & 3u][k + j], c.cell_v[i & 3u][k + j]) : z);
                    }
                    tmem_st8(at + k, x);
                }
                tmem_wait_st();
            }
            uint32_t raw[64];
            tmem_ld32(at, raw);
            tmem_ld32(at + 32u, raw + 32);
            tmem_wait_ld64(raw);
            // bit j of the words: the row's range holds cell c0 + j; a thread without a row sees none (and has no mask)
            uint32_t w0 = row < rows ? ~0u : 0u, w1 = w0;
            if (MASK || !open || far) {              // then these are the scores, elsewhere their factors wait for the exponent
                if (!far) {
#pragma unroll
                    for (int j = 0; j < 64; ++j) raw[j] = __float_as_uint(__uint_as_float(raw[j]) * qs);
                }
                f = 1.0f;
            }
            if (!open) {
                const int32_t from = min(max(lo - c0, 0), 64), to = min(max(hi - c0, from), 64);
                const unsigned long long bits = (to >= 64 ? ~0ull : (1ull << to) - 1ull) & ~(from >= 64 ? ~0ull : (1ull << from) - 1ull);
                w0 = (uint32_t)bits;
                w1 = (uint32_t)(bits >> 32);
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    raw[j] = w0 >> j & 1u ? raw[j] : 0xFF800000u;
                    raw[32 + j] = w1 >> j & 1u ? raw[32 + j] : 0xFF800000u;
                }
            }
            if constexpr (MASK) {
                // the mask's running maximum is taken out first: a row of the type's lowest value keeps its scores' digits
                const bool every = __all_sync(0xFFFFFFFFu, (w0 & w1) == ~0u);
                auto pass = [&](auto whole) {        // two forms, so that no branch stands before the loads
                    constexpr bool WIDE = decltype(whole)::value;
                    __half2 most2 = __half2half2(__ushort_as_half((unsigned short)0xFC00u));
#pragma unroll
                    for (uint32_t k = 0; k < 8; ++k) {
                        const uint4 h = mask_of(mrow, c0 + 8 * (int32_t)k, (k < 4 ? w0 >> 8u * k : w1 >> (8u * k - 32u)) & 0xFFu, WIDE, WIDE && every);
                        most2 = __hmax2(most2, __hmax2(__hmax2(as_h2(h.x), as_h2(h.y)), __hmax2(as_h2(h.z), as_h2(h.w))));
                    }
                    const float now = fmaxf(off, fmaxf(__low2float(most2), __high2float(most2))), base = now == -INFINITY ? 0.0f : now;
                    if (off != -INFINITY && off != now) m += (off - base) * 1.4426950408889634f;
                    off = now;
#pragma unroll
                    for (uint32_t k = 0; k < 8; ++k) {
                        const uint4 h = mask_of(mrow, c0 + 8 * (int32_t)k, (k < 4 ? w0 >> 8u * k : w1 >> (8u * k - 32u)) & 0xFFu, WIDE, WIDE && every);
                        const uint32_t w[4] = {h.x, h.y, h.z, h.w};
#pragma unroll
                        for (uint32_t j = 0; j < 8; ++j) {
                            const float x = __half2float(__ushort_as_half((unsigned short)(w[j / 2] >> (j & 1u ? 16 : 0))));
                            const float z = fmaf(x - base, 1.4426950408889634f, __uint_as_float(raw[8 * k + j]));
                            raw[8 * k + j] = __float_as_uint(x == -INFINITY ? -INFINITY : z);
                        }
                    }
                };
                if (a.mask_wide && c0 + (int32_t)kTile <= (int32_t)a.n_kv) pass(std::true_type{});
                else pass(std::false_type{});
            }
            float most = -INFINITY;
#pragma unroll
            for (uint32_t w = 0; w < 4; ++w) {
                float top = max3(__uint_as_float(raw[16 * w]), __uint_as_float(raw[16 * w + 1]), __uint_as_float(raw[16 * w + 2]));
#pragma unroll
                for (uint32_t j = 3; j + 1 < 16; j += 2) top = max3(top, __uint_as_float(raw[16 * w + j]), __uint_as_float(raw[16 * w + j + 1]));
                most = max3(most, top, __uint_as_float(raw[16 * w + 15]));
            }
            most *= f;
            const bool raise = __any_sync(0xFFFFFFFFu, most > m + 8.0f);
            const bool flush = TOTAL && i > 0 && i % S::FLUSH == 0u;
            if (raise || flush) {
                float both = 1.0f;
                if (raise) {
                    const float now = fmaxf(m, most), base = now == -INFINITY ? 0.0f : now, down = ex2(m - base);
                    l *= down;
                    m = now;
                    both = down;
                }
                if (i > 0) {
                    // the products so far have to be there
                    ok = __all_sync(0xFFFFFFFFu, bar_wait(&c.o_done[rg][buf ^ 1u], ((i - 1u) >> 1) & 1u, &c.abort));
                    if (!ok) break;
                    fence_after();
                    if constexpr (TOTAL) settle<D>(o_at, mine + S::SUM_COL, both, i <= S::FLUSH, flush);
                    else rescale<D>(o_at, both);
                }
            }
            const float up = m == -INFINITY ? 0.0f : 6.0f - m;
            float far_sum = 0.0f;
            if (MASK && far) {                       // the sum takes the weights without V's powers of two
#pragma unroll
                for (int j = 0; j < 64; ++j)
                    far_sum += ex2(__uint_as_float(raw[j]) - (info.flags[j / GC] & kFar ? c.cell_v[i & 3u][j] : 0.0f) + up);
            } else if (far) {
#pragma unroll 1
                for (uint32_t k = 0; k < kTile; k += 8) {
                    const bool own = info.flags[k / GC] & kFar;
                    uint32_t x[8];
                    tmem_ld8(at + k, x);
                    tmem_wait_ld8(x);
#pragma unroll
                    for (uint32_t j = 0; j < 8; ++j) {
                        const int32_t cell = c0 + (int32_t)(k + j);
                        if (cell >= lo && cell < hi) far_sum += ex2(__uint_as_float(x[j]) - (own ? c.cell_v[i & 3u][k + j] : 0.0f) + up);
                    }
                    __syncwarp();
                }
            }
            float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
            for (int k = 0; k < 4; ++k) {            // sixteen cells at a time: eight words of each term
                uint32_t hw[8], lw[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint32_t e = 16 * k + 2 * j;
                    const float2 z = fma2(make_float2(__uint_as_float(raw[e]), __uint_as_float(raw[e + 1])), make_float2(f, f), make_float2(up, up));
                    const float2 p = make_float2(ex2(z.x), ex2(z.y));
                    sum[j & 1] = add2(sum[j & 1], p);
                    const __half2 h = __floats2half2_rn(p.x, p.y);
                    hw[j] = as_u32(h);
                    if (PRECISE) {
                        const float2 back = __half22float2(h);
                        lw[j] = as_u32(__floats2half2_rn(p.x - back.x, p.y - back.y));
                    }
                }
                tmem_st8(at + 8u * k, hw);
                if (PRECISE) tmem_st8(at + kTile / 2u + 8u * k, lw);
            }
            const float2 total = add2(sum[0], sum[1]);
            l += far ? far_sum : total.x + total.y;
            tmem_wait_st();
            fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(&c.p_full[rg][sb]);
            if (bad) {                          // seldom: which of the blocks left out of V this row would have met
#pragma unroll 1
                for (uint32_t j = 0; j < kTile; ++j) {
                    if (c0 + (int32_t)j < lo || c0 + (int32_t)j >= hi || (MASK && __half2float(mrow[c0 + (int32_t)j]) == -INFINITY)) continue;
                    const __half* d = a.vd + ((size_t)hk * a.n_alloc + (uint32_t)c0 + j) * NB;
                    for (uint32_t b = 0; b < NB; ++b)
                        if ((__half_as_ushort(d[b]) & 0x7C00u) == 0x7C00u) lost |= 1u << b;
                }
            }
        }
        // every product has ended: the outputs are there, and the tensor memory may go
        if (ok && tiles) ok = bar_wait(&c.o_done[rg][(tiles - 1u) & 1u], ((tiles - 1u) >> 1) & 1u, &c.abort);
        ok = __all_sync(0xFFFFFFFFu, ok);
        if (ok) {
            fence_after();
            // l and O are in units of 2^6 p: a split's share names 2^-6 of its reference
            const float unit = pow2(-kOperandExp), f = a.splits > 1u ? unit : l == 0.0f ? 0.0f : unit / l;
            T* out = static_cast<T*>(a.out) + (size_t)tok * a.out_stride + (size_t)head * D;
            const size_t part = ((((size_t)grp * a.row_tiles + rt) * a.n_head_kv + hk) * a.splits + split) * (kRows * RG) + tid;
            if (a.splits > 1u && row < rows) *reinterpret_cast<float4*>(a.part_ml + part * 4u) = make_float4(off, m - 6.0f, l, 0.0f);
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b) {
                uint32_t o[32] = {};
                if (tiles) {
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j) tmem_ld8(o_at + j * (D / 4) + 8u * b, o + 8 * j);
                    tmem_wait_ld(o);
                    if (TOTAL && tiles > S::FLUSH) {
                        uint32_t t[32];
#pragma unroll
                        for (uint32_t j = 0; j < 4; ++j) tmem_ld8(mine + S::SUM_COL + j * (D / 4) + 8u * b, t + 8 * j);
                        tmem_wait_ld(t);
#pragma unroll
                        for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) + __uint_as_float(t[j]));
                    }
                }
                if (row < rows) {
#pragma unroll
                    for (uint32_t g = 0; g < 8; ++g) {
                        float x[4];
#pragma unroll
                        for (uint32_t j = 0; j < 4; ++j) {
                            x[j] = l == 0.0f ? 0.0f : __uint_as_float(o[8 * j + g]) * f;
                            if (lost >> b & 1u) x[j] = __int_as_float(0x7FC00000);
                        }
                        if (a.splits > 1u) store4<float>(a.part_o + part * D + 32u * b + 4u * g, x, true);
                        else store4<T>(out + 32u * b + 4u * g, x, a.out_wide);
                    }
                }
                __syncwarp();
            }
        }
    }
    fence_before();
    __syncthreads();
    if (warp == 0) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(S::COLUMNS));
    }
}

template <class T, int D, bool MASK, uint32_t RG>
cudaError_t launch_m(const Fa4Args& a, uint32_t units, cudaStream_t st) {
    using S = TcShape<T, D, MASK, RG>;
    static bool done[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !done[dev]) {
        e = cudaFuncSetAttribute(fa4_tc_kernel<T, D, MASK, RG>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::BYTES);
        if (e != cudaSuccess) return e;
        if (dev < 64) done[dev] = true;
    }
    fa4_tc_kernel<T, D, MASK, RG><<<units * a.splits, S::THREADS, S::BYTES, st>>>(a);
    return cudaGetLastError();
}

template <class T, int D, uint32_t RG>
cudaError_t launch_g(const Fa4Args& a, uint32_t units, cudaStream_t st) {
    return a.mask ? launch_m<T, D, true, RG>(a, units, st) : launch_m<T, D, false, RG>(a, units, st);
}
template <class T, int D>
cudaError_t launch(const Fa4Args& a, uint32_t units, cudaStream_t st) {
    if constexpr (std::is_same_v<T, __nv_bfloat16>)
        if (a.tile_rows == 2u * kFa4TcRows) return launch_g<T, D, 2>(a, units, st);
    return launch_g<T, D, 1>(a, units, st);
}

}  // namespace

cudaError_t launch_fa4_tc(uint32_t type, uint32_t D, const Fa4Args& a, uint32_t units, cudaStream_t st) {
    if (type == TSRC_TYPE_F32) return D == 64u ? launch<float, 64>(a, units, st) : launch<float, 128>(a, units, st);
    if (type == TSRC_TYPE_F16) return D == 64u ? launch<__half, 64>(a, units, st) : launch<__half, 128>(a, units, st);
    return D == 64u ? launch<__nv_bfloat16, 64>(a, units, st) : launch<__nv_bfloat16, 128>(a, units, st);
}

cudaError_t fa4_error(uint32_t* code, bool clear) {
    cudaError_t e = cudaMemcpyFromSymbol(code, g_fa4_error, sizeof(uint32_t));
    if (e == cudaSuccess && clear && *code) {
        const uint32_t zero = 0;
        e = cudaMemcpyToSymbol(g_fa4_error, &zero, sizeof(uint32_t));
    }
    return e;
}

}  // namespace tsrc
