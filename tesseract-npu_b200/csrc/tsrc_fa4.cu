// tsrc_fa4.cu -- attention over the q4_0 KV cache (tsrc_flash_attn_q4). Cache layout: tsrc_kv4.cuh.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "tsrc_fa4.cuh"

namespace tsrc {

namespace {

constexpr uint32_t kDecWarps = 4, kDecTile = 32, kDecStages = 3;
constexpr uint32_t kSms = 148;
constexpr uint32_t kMaxCluster = 16;

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp8(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// d = a b + c of a 16 x 16 by 16 x 8 tile
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1,
                                         float c0, float c1, float c2, float c3) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {      // of an 8 x 8 tile of fp16, two neighbours a lane
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ __half2 as_h2(uint32_t u) { return *reinterpret_cast<const __half2*>(&u); }
__device__ __forceinline__ uint32_t as_u32(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }
__device__ __forceinline__ uint32_t pack2(float lo, float hi) { return as_u32(__floats2half2_rn(lo, hi)); }
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 remote_f32x4(const float4* p, uint32_t rank) {
    uint32_t at;
    float4 v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at));
    return v;
}

// how a warp's columns of eight query rows are used
enum : int {
    kRows8Split = 0,       // eight rows; q and the weights in two fp16 terms each
    kRows8 = 1,            // eight rows, one term (bf16 outputs)
    kRows16 = 2,           // sixteen rows, one term (bf16 outputs)
    kRows128 = 3,          // the kernel for many rows
};
template <int MODE> constexpr uint32_t kRowsOf = MODE == kRows16 ? 16u : 8u;

template <int D> struct DecShape {
    static constexpr uint32_t WARPS = kDecWarps;
    static constexpr uint32_t NB = D == 64 ? 2 : 4;            // blocks of a warp's group of values
    static constexpr uint32_t W = NB * 32;                      // values of a group: a warp's share of the head
    static constexpr uint32_t NG = D / W;                       // warps of a team: they share a tile's scores
    static constexpr uint32_t TEAMS = WARPS / NG;
    static constexpr uint32_t ROW = W / 2, DS = NB * 2;         // bytes of a cell's codes and scales in a group
    static constexpr uint32_t V_AT = kDecTile * ROW, KD_AT = 2 * kDecTile * ROW, VD_AT = KD_AT + kDecTile * DS;
    static constexpr uint32_t STAGE = VD_AT + kDecTile * DS;
    static constexpr uint32_t RING = STAGE * kDecStages;
};
// ring (later the warps' results), the warps' and the CTA's maxima and sums, the score exchange of teams (two turns)
// or the factors of a cluster's CTAs
template <int D, int MODE> __host__ __device__ constexpr uint32_t dec_smem() {
    using S = DecShape<D>;
    constexpr uint32_t WARPS = kDecWarps;
    return WARPS * S::RING + (WARPS + 1u) * 16u * 16u + (S::NG > 1 ? 2u * WARPS * 32u : kMaxCluster + 4u) * kRowsOf<MODE> * 4u;
}

// Weights go in as 2^10 p dV: below 2^15 for scales of V below 32, with digits down to fp16's last, 2^-24. Where all scales
// that a warp has met are below 2^-10, they are taken times 2^10. A cell with a scale of 32 and above (no row of ordinary
// size has one) has its scales divided by 2^x, x that scale's exponent field above kFarExp, and x added to its scores for the
// weights (not for their sum): the rows that see it follow by their running maximum, those that do not keep their digits.
constexpr float kWeightUp = 10.0f;
constexpr int kTinyUp = 10;
constexpr uint32_t kFarExp = 19;           // exponent field of scales of 16 to 32
constexpr uint32_t kTinyExp = 5;           // ... and of 2^-10 to 2^-9
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

// Decode attention, one pass over the cells.
//   A CTA takes up to 8 (16) query rows -- the (token, head) pairs of a group that share a KV head -- and one split
// of the cells they span; its warps take tiles of 32 cells in turn (D > 128: teams of D / 128 warps, each with 128
// values of the head, which add up their partial scores through shared memory). Tiles come by cp.async, three deep.
// The splits of a row are the CTAs of one cluster, which join their results through shared memory, or, where more
// than sixteen are wanted, separate CTAs and a merge kernel.
//   Both products run transposed, scores = K q^T and outputs = V^T w^T, so that the eight columns of an mma are the
// query rows and its sixteen rows are cells (values): with few query rows nothing of a tile is idle, and an output
// takes half the registers. The weights change from the first product's layout to the second's by movmatrix.
//   Codes go to the tensor cores as they are: a code n in the low four bits of an fp16 is the subnormal number
// n 2^-24, in the next four n 2^-20 (q's values that meet those carry 2^-4; outputs from those are scaled at the
// end), so an operand register of two codes is one AND of a word of eight, and a shift for every second pair. What
// is missing, sum q (n - 8) = sum q n - 8 sum q, is the accumulator's start value for K; for V the weights' sum
// comes from one more mma per block with 8 2^-24 in every row. The blocks' scales stay out of the products: K's
// multiply the four (two) partial sums of a score in f32; V's multiply the weights: w = p dV, a set for each block.
//   Precision: q and w are two fp16 terms each, 22 bits (q scaled by a power of two per row); for bf16 outputs one
// term, 11 bits. Running maximum, sum and outputs are f32. The tensor cores align a subnormal operand's products as
// if it were 2^-14, so up to seven of the sum's 24 bits are lost that way (measured: 2^-17 of the largest product at
// worst, 1.4e-5 of an output row): enough for 16-bit outputs; f32 outputs take n - 8 as an ordinary fp16, one fused
// step more for two codes, and need neither start value nor weights' sum (1e-6).
template <class T, int D, int MODE, bool MASK>
__global__ void __launch_bounds__(kDecWarps * 32, MODE == kRows16 ? 3 : 4) fa4_dec_kernel(Fa4Args a) {
    using S = DecShape<D>;
    constexpr uint32_t WARPS = kDecWarps;
    constexpr uint32_t NB = S::NB, R = kRowsOf<MODE>, NT = R / 8;        // NT: columns of eight rows
    constexpr bool SPLIT = MODE == kRows8Split, WHOLE = std::is_same_v<T, float>;     // WHOLE: operands are n - 8
    // a word's codes as operands: those in the low four bits, those in the next four
    auto even = [](uint32_t x) {
        x &= 0x000F000Fu;
        return WHOLE ? as_u32(__hsub2(as_h2(x | 0x64006400u), __float2half2_rn(1032.0f))) : x;
    };
    auto odd = [](uint32_t x) {
        x &= 0x00F000F0u;
        return WHOLE ? as_u32(__hfma2(as_h2(x | 0x64006400u), __float2half2_rn(0.0625f), __float2half2_rn(-72.0f))) : x;
    };
    constexpr float kOdd = WHOLE ? 1.0f : 0.0625f;               // makes up for the odd codes' place
    extern __shared__ __align__(128) uint8_t sm[];
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, g = lane >> 2, t = lane & 3u;
    const uint32_t team = warp / S::NG, sub = warp % S::NG;
    const uint32_t unit = blockIdx.x / a.splits, split = blockIdx.x - unit * a.splits;
    const uint32_t hk = unit % a.n_head_kv, rt = unit / a.n_head_kv % a.row_tiles, grp = unit / (a.n_head_kv * a.row_tiles);
    const uint32_t rows = a.group * a.G;
    uint8_t* ringp = sm + warp * S::RING;
    const uint32_t ring = smem_u32(ringp);
    float4* red = reinterpret_cast<float4*>(sm + WARPS * S::RING);       // [warps + 1][16]: mask reference, maximum, sum; then factors
    float* xch = reinterpret_cast<float*>(red + (WARPS + 1u) * 16u);

    // the cells of this lane's rows (8 n + 2 t + i), and the hull of all rows
    int32_t lo[NT][2], hi[NT][2], first = 0x7FFFFFFF, last = 0, all_lo = 0, all_hi = 0x7FFFFFFF;
    const __half* mrow[NT][2];
#pragma unroll
    for (uint32_t n = 0; n < NT; ++n)
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) {
            const uint32_t row = rt * R + 8u * n + 2u * t + i;
            lo[n][i] = hi[n][i] = 0;
            mrow[n][i] = a.mask;
            if (row < rows) {
                const uint32_t tok = grp * a.group + row / a.G;
                int32_t x = 0, y = (int32_t)a.n_kv;
                if (a.ranges) {
                    x = max(a.ranges[2u * (size_t)tok], 0);
                    y = min(a.ranges[2u * (size_t)tok + 1u], y);
                }
                if (x < y) {
                    lo[n][i] = x;
                    hi[n][i] = y;
                    first = min(first, x);
                    last = max(last, y);
                }
                // the cells that every row sees; a column without a row has nothing to lose
                all_lo = max(all_lo, lo[n][i]);
                all_hi = min(all_hi, hi[n][i]);
                if (MASK) mrow[n][i] = a.mask + (size_t)tok * a.mask_stride;
            }
        }
    first = __reduce_min_sync(0xFFFFFFFFu, first);
    last = __reduce_max_sync(0xFFFFFFFFu, last);
    all_lo = __reduce_max_sync(0xFFFFFFFFu, all_lo);
    all_hi = __reduce_min_sync(0xFFFFFFFFu, all_hi);
    const uint32_t tile0 = (uint32_t)min(first, last) / kDecTile, tiles = last > first ? ((uint32_t)last + kDecTile - 1u) / kDecTile - tile0 : 0u;
    const uint32_t from = tile0 + (uint32_t)((uint64_t)tiles * split / a.splits) + team;
    const uint32_t to = tile0 + (uint32_t)((uint64_t)tiles * (split + 1u) / a.splits);

    // this lane's pieces of a tile: codes at rows lane / PER + 32 / PER i, the scales as one run or cell by cell
    constexpr uint32_t PER = S::ROW / 16;                       // 16-byte pieces of a cell's codes
    const size_t plane = (size_t)hk * a.n_alloc;
    const uint8_t* kq = a.kq + (plane + lane / PER) * (D / 2) + sub * S::ROW + 16u * (lane % PER);
    const uint8_t* vq = a.vq + (plane + lane / PER) * (D / 2) + sub * S::ROW + 16u * (lane % PER);
    constexpr uint32_t DP = kDecTile * S::DS / 16;              // 16-byte pieces of a tile's scales
    const uint8_t* ds = S::NG > 1 ? reinterpret_cast<const uint8_t*>(a.kd + (plane + lane) * (D / 32) + sub * NB)
                                  : reinterpret_cast<const uint8_t*>((lane < DP ? a.kd : a.vd) + plane * NB) + 16u * (lane % DP);
    const uint8_t* ds2 = S::NG > 1 ? reinterpret_cast<const uint8_t*>(a.vd + (plane + lane) * (D / 32) + sub * NB) : nullptr;
    auto fetch = [&](uint32_t tile, uint32_t stage) {
        const size_t c0 = (size_t)tile * kDecTile;
        const uint32_t at = ring + stage * S::STAGE + 16u * lane;
        const uint8_t *k = kq + c0 * (D / 2), *v = vq + c0 * (D / 2);
#pragma unroll
        for (uint32_t i = 0; i < PER; ++i) {
            cp16(at + 512u * i, k + i * (32u / PER) * (D / 2));
            cp16(at + S::V_AT + 512u * i, v + i * (32u / PER) * (D / 2));
        }
        if constexpr (S::NG == 1) {
            if (lane < 2u * DP) cp16(at + S::KD_AT, ds + c0 * S::DS);
        } else {
            cp8(at + S::KD_AT - 8u * lane, ds + c0 * (D / 16));
            cp8(at + S::VD_AT - 8u * lane, ds2 + c0 * (D / 16));
        }
    };
#pragma unroll
    for (uint32_t s = 0; s < kDecStages - 1; ++s) {
        if (from + s * S::TEAMS < to) fetch(from + s * S::TEAMS, s);
        cp_commit();
    }

    // q's fragments: lane (g, t) owns values 8t .. 8t + 7 of each block of row g (8 n + g)
    uint32_t qb[NT][SPLIT ? 2 : 1][NB][2][2];
    float start[NT][NB][2], rs[NT][2];
#pragma unroll
    for (uint32_t n = 0; n < NT; ++n) {
        const uint32_t row = rt * R + 8u * n + g;
        float x[NB][8], top = 0.0f;
        if (row < rows) {
            const T* q = static_cast<const T*>(a.q) + (size_t)(grp * a.group + row / a.G) * a.q_stride +
                         (size_t)(hk * a.G + row % a.G) * D + sub * S::W + 8u * t;
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b) {
                if (a.q_wide) load8<T, true>(q + 32u * b, x[b]);
                else load8<T, false>(q + 32u * b, x[b]);
            }
        } else {
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b)
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) x[b][i] = 0.0f;
        }
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b)
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[b][i]));
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
        // the row's largest value to [2^12, 2^13); rows of tiny values by 2^100 at most
        const int e = min(12 - ((int)(__float_as_uint(top) >> 23) - 127), 100);
        // Step by step, so that only a factor that leaves f32 itself does; cut to the largest finite one, scores of 0 stay 0, and
        // others are as far apart from each other as any exponential can tell (the smallest is 2^-48 of the factor).
        const float f = pow2(e), mine = fminf(fmaxf(a.scale * pow2(-e) * (kLog2e * (WHOLE ? 1.0f : 16777216.0f)), -FLT_MAX), FLT_MAX);
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) rs[n][i] = __shfl_sync(0xFFFFFFFFu, mine, 8u * t + 4u * i);
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b) {
            float sum = 0.0f;
#pragma unroll
            for (uint32_t k = 0; k < (SPLIT ? 2u : 1u); ++k) {
                float y[8];
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) {
                    if (k == 0) x[b][i] *= f;
                    y[i] = __half2float(__float2half_rn(x[b][i]));
                    x[b][i] -= y[i];
                    sum += y[i];
                }
#pragma unroll
                for (uint32_t j = 0; j < 2; ++j) {
                    qb[n][k][b][j][0] = pack2(y[2 * j], y[2 * j + 4]);
                    qb[n][k][b][j][1] = pack2(y[2 * j + 1] * kOdd, y[2 * j + 5] * kOdd);
                }
            }
            sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 1);
            sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 2);
            sum *= WHOLE ? 0.0f : -8.0f / 16777216.0f;
#pragma unroll
            for (uint32_t i = 0; i < 2; ++i) start[n][b][i] = __shfl_sync(0xFFFFFFFFu, sum, 8u * t + 4u * i);
        }
    }

    float o[NT][NB][2][4] = {}, wsum[NT][NB][2] = {}, m[NT][2], l[NT][2], off[NT][2];
    bool tiny = true;        // no scale of V of 2^-10 and above was met
    uint32_t lost = 0;       // bit 4 (2 n + i) + b: the row sees a scale of V in block b that is infinite or no number
#pragma unroll
    for (uint32_t n = 0; n < NT; ++n)
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) {
            m[n][i] = off[n][i] = -INFINITY;
            l[n][i] = 0.0f;
        }
    // Cells of an eight in the order 0 1 3 2 4 5 7 6: with kv4_place, the four cells that the lanes of a column
    // meet in V then lie in different banks, and so do the two of a K load.
    const uint32_t pg = g ^ ((g >> 1) & 1u);                      // the cell of this lane's row of K's operand
    const uint32_t c_a = (2u * t) ^ (t & 1u), c_b = c_a ^ 1u;     // the cells of the pair 2t, 2t + 1
    const uint32_t k_at = pg * S::ROW + (t ^ ((pg >> 1) & 2u)) * (S::ROW / 4);
    const uint32_t v_at = S::V_AT + c_a * S::ROW + (g ^ ((t >> 1) * 4u)) * (S::ROW / 8);
    const int32_t v_step = c_b > c_a ? (int32_t)S::ROW : -(int32_t)S::ROW;

    uint32_t stage = 0, turn = 0;
    for (uint32_t tile = from; tile < to; tile += S::TEAMS) {
        {
            const uint32_t next = tile + (kDecStages - 1) * S::TEAMS;
            if (next < to) fetch(next, stage == 0 ? kDecStages - 1 : stage - 1);
            cp_commit();
        }
        const uint32_t c0 = tile * kDecTile;
        const bool open = !MASK && (int32_t)c0 >= all_lo && (int32_t)(c0 + kDecTile) <= all_hi;
        // scores: index j of a lane's four cells pg + 8 j
        float mk[NT][2][4];
        if (MASK) {
#pragma unroll
            for (uint32_t n = 0; n < NT; ++n)
#pragma unroll
                for (uint32_t i = 0; i < 2; ++i)
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j) {
                        const int32_t c = (int32_t)(c0 + pg + 8u * j);
                        mk[n][i][j] = c >= lo[n][i] && c < hi[n][i] ? __half2float(mrow[n][i][c]) : -INFINITY;
                    }
        }
        cp_wait<kDecStages - 1>();
        __syncwarp();
        const uint8_t* sk = ringp + stage * S::STAGE;
        float s[NT][2][4];
#pragma unroll
        for (uint32_t mt = 0; mt < 2; ++mt) {
            uint32_t w[2][NB], d[2][NB / 2];
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h) {
                const uint8_t* p = sk + k_at + (16u * mt + 8u * h) * S::ROW;
                const uint8_t* pd = sk + S::KD_AT + (16u * mt + 8u * h + pg) * S::DS;
                if constexpr (NB == 4) {
                    const uint4 v = *reinterpret_cast<const uint4*>(p);
                    w[h][0] = __byte_perm(v.x, v.z, 0x5410);
                    w[h][1] = __byte_perm(v.x, v.z, 0x7632);
                    w[h][2] = __byte_perm(v.y, v.w, 0x5410);
                    w[h][3] = __byte_perm(v.y, v.w, 0x7632);
                    const uint2 u = *reinterpret_cast<const uint2*>(pd);
                    d[h][0] = u.x;
                    d[h][1] = u.y;
                } else {
                    const uint2 v = *reinterpret_cast<const uint2*>(p);
                    w[h][0] = __byte_perm(v.x, v.y, 0x5410);
                    w[h][1] = __byte_perm(v.x, v.y, 0x7632);
                    d[h][0] = *reinterpret_cast<const uint32_t*>(pd);
                }
            }
            float acc[NT][4] = {};
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b) {
                const uint32_t x0 = w[0][b], x1 = w[1][b], y0 = x0 >> 8, y1 = x1 >> 8;
                const uint32_t e0 = even(x0), e1 = even(x1), o0 = odd(x0), o1 = odd(x1);
                const uint32_t f0 = even(y0), f1 = even(y1), p0 = odd(y0), p1 = odd(y1);
                const float2 g0 = __half22float2(as_h2(d[0][b / 2])), g1 = __half22float2(as_h2(d[1][b / 2]));
                const float d0 = b & 1u ? g0.y : g0.x, d1 = b & 1u ? g1.y : g1.x;
#pragma unroll
                for (uint32_t n = 0; n < NT; ++n) {
                    // the small term first: its roundings are then relative to it alone
                    float c[4] = {start[n][b][0], start[n][b][1], start[n][b][0], start[n][b][1]};
#pragma unroll
                    for (uint32_t k = SPLIT ? 2 : 1; k-- > 0;) {
                        mma16816(c, e0, e1, o0, o1, qb[n][k][b][0][0], qb[n][k][b][0][1], c[0], c[1], c[2], c[3]);
                        mma16816(c, f0, f1, p0, p1, qb[n][k][b][1][0], qb[n][k][b][1][1], c[0], c[1], c[2], c[3]);
                    }
                    acc[n][0] = fmaf(c[0], d0, acc[n][0]);
                    acc[n][1] = fmaf(c[1], d0, acc[n][1]);
                    acc[n][2] = fmaf(c[2], d1, acc[n][2]);
                    acc[n][3] = fmaf(c[3], d1, acc[n][3]);
                }
            }
#pragma unroll
            for (uint32_t n = 0; n < NT; ++n)
#pragma unroll
                for (uint32_t i = 0; i < 2; ++i) {
                    s[n][i][2 * mt] = acc[n][i] * rs[n][i];
                    s[n][i][2 * mt + 1] = acc[n][2 + i] * rs[n][i];
                }
        }
        if constexpr (S::NG > 1) {
            // the team's partial scores, added in the order of the groups
            float* mine = xch + (turn * WARPS + warp) * NT * 8u * 32u + lane;
#pragma unroll
            for (uint32_t k = 0; k < NT * 8u; ++k) mine[k * 32u] = s[k / 8u][k / 4u % 2u][k % 4u];
            asm volatile("bar.sync %0, %1;" ::"r"(1u + team), "n"(32 * S::NG) : "memory");
            const float* all = xch + (turn * WARPS + team * S::NG) * NT * 8u * 32u + lane;
#pragma unroll
            for (uint32_t k = 0; k < NT * 8u; ++k) {
                float x = all[k * 32u];
#pragma unroll
                for (uint32_t j = 1; j < S::NG; ++j) x += all[(j * NT * 8u + k) * 32u];
                s[k / 8u][k / 4u % 2u][k % 4u] = x;
            }
            turn ^= 1u;
        }
        // V's scales as pairs of cells, and the largest of them
        __half2 dv[4][NB], most = __float2half2_rn(0.0f);
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
            const uint8_t* pd = sk + S::VD_AT + 8u * e * S::DS;
            uint32_t x[NB / 2], y[NB / 2];
            if constexpr (NB == 4) {
                const uint2 u = *reinterpret_cast<const uint2*>(pd + c_a * 8u), v = *reinterpret_cast<const uint2*>(pd + c_b * 8u);
                x[0] = u.x; x[1] = u.y; y[0] = v.x; y[1] = v.y;
            } else {
                x[0] = *reinterpret_cast<const uint32_t*>(pd + c_a * 4u);
                y[0] = *reinterpret_cast<const uint32_t*>(pd + c_b * 4u);
            }
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b) {
                dv[e][b] = as_h2(__byte_perm(x[b / 2], y[b / 2], b & 1u ? 0x7632 : 0x5410));
                most = __hmax2_nan(most, __habs2(dv[e][b]));
            }
        }
        uint32_t big = __reduce_max_sync(0xFFFFFFFFu, max(as_u32(most) & 0xFFFFu, as_u32(most) >> 16));
        if (big >= 0x7C00u) {
            // Seldom: such a scale counts as 0 in the products, and its block is marked for the rows that see the cell,
            // whatever weight they give it.
            uint32_t x = 0;
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e)
#pragma unroll
                for (uint32_t b = 0; b < NB; ++b) {
                    uint32_t u = as_u32(dv[e][b]);
                    u = ((u & 0x7C00u) == 0x7C00u ? 0u : u & 0xFFFFu) | ((u & 0x7C000000u) == 0x7C000000u ? 0u : u & 0xFFFF0000u);
                    dv[e][b] = as_h2(u);
                    x = max(x, max(u & 0x7FFFu, u >> 16 & 0x7FFFu));
                }
            big = __reduce_max_sync(0xFFFFFFFFu, x);
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                const uint16_t* pd = reinterpret_cast<const uint16_t*>(sk + S::VD_AT + (pg + 8u * j) * S::DS);
                const int32_t c = (int32_t)(c0 + pg + 8u * j);
                uint32_t bad = 0;
#pragma unroll
                for (uint32_t b = 0; b < NB; ++b) bad |= (pd[b] & 0x7C00u) == 0x7C00u ? 1u << b : 0u;
#pragma unroll
                for (uint32_t n = 0; n < NT; ++n)
#pragma unroll
                    for (uint32_t i = 0; i < 2; ++i)
                        if (open || (MASK ? mk[n][i][j] != -INFINITY : c >= lo[n][i] && c < hi[n][i])) lost |= bad << (4u * (2u * n + i));
            }
        }
        bool moved = false;
        float rescale = 1.0f;
        if (tiny && (big >> 10) >= kTinyExp) {                    // the same for the whole warp
            tiny = false;
            rescale = pow2(-kTinyUp);
            moved = true;
        }
        const bool far = (big >> 10) > kFarExp;                   // seldom
        auto above = [&](uint32_t j) {                            // x of the lane's cell pg + 8 j
            const uint16_t* pd = reinterpret_cast<const uint16_t*>(sk + S::VD_AT + (pg + 8u * j) * S::DS);
            uint32_t v = kFarExp;
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b) {
                const uint32_t u = pd[b] & 0x7FFFu;
                v = max(v, u < 0x7C00u ? u >> 10 : 0u);
            }
            return (int)(v - kFarExp);
        };
        if (far) {
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                const float x = (float)above(j);
#pragma unroll
                for (uint32_t n = 0; n < NT; ++n) {
                    s[n][0][j] += x;
                    s[n][1][j] += x;
                }
            }
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) {
                uint32_t va = kFarExp, vb = kFarExp;
#pragma unroll
                for (uint32_t b = 0; b < NB; ++b) {
                    va = max(va, as_u32(dv[e][b]) >> 10 & 31u);
                    vb = max(vb, as_u32(dv[e][b]) >> 26 & 31u);
                }
                const __half2 down = as_h2((15u + kFarExp - va) << 10 | (15u + kFarExp - vb) << 26);
#pragma unroll
                for (uint32_t b = 0; b < NB; ++b) dv[e][b] = __hmul2(dv[e][b], down);
            }
        }
        // running maximum and sum; what a row does not see is -inf
        float alpha[NT][2];
#pragma unroll
        for (uint32_t n = 0; n < NT; ++n)
#pragma unroll
            for (uint32_t i = 0; i < 2; ++i) {
                float (&z)[4] = s[n][i];
                float m_old = m[n][i];
                bool seen[4];
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) {
                    const int32_t c = (int32_t)(c0 + pg + 8u * j);
                    seen[j] = open || (MASK ? mk[n][i][j] != -INFINITY : c >= lo[n][i] && c < hi[n][i]);
                }
                if (MASK) {
                    // the mask's running maximum is taken out first: a row of the type's lowest value keeps its scores' digits
                    float top = fmaxf(fmaxf(mk[n][i][0], mk[n][i][1]), fmaxf(mk[n][i][2], mk[n][i][3]));
#pragma unroll
                    for (uint32_t x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, x));
                    const float was = off[n][i], now = fmaxf(was, top), base = now == -INFINITY ? 0.0f : now;
                    if (was != -INFINITY && was != now) m_old += (was - base) * kLog2e;
                    off[n][i] = now;
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j) z[j] = fmaf(mk[n][i][j] - base, kLog2e, z[j]);
                }
                if (!open) {
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j) z[j] = seen[j] ? z[j] : -INFINITY;
                }
                float top = fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3]));
#pragma unroll
                for (uint32_t x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, x));
                const float m_new = fmaxf(m_old, top), base = m_new == -INFINITY ? 0.0f : m_new, up = kWeightUp - base;
                alpha[n][i] = ex2(m_old - base);
                moved |= m_new > m[n][i] || m_old != m[n][i];
                m[n][i] = m_new;
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) z[j] = ex2(z[j] + up);
                if (!far) l[n][i] = fmaf(l[n][i], alpha[n][i], (z[0] + z[1]) + (z[2] + z[3]));
            }
        if (far) {
#pragma unroll
            for (uint32_t n = 0; n < NT; ++n) {
                l[n][0] *= alpha[n][0];
                l[n][1] *= alpha[n][1];
            }
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                const float down = pow2(-above(j));
#pragma unroll
                for (uint32_t n = 0; n < NT; ++n) {
                    l[n][0] = fmaf(s[n][0][j], down, l[n][0]);
                    l[n][1] = fmaf(s[n][1][j], down, l[n][1]);
                }
            }
        }
        if (__any_sync(0xFFFFFFFFu, moved)) {
#pragma unroll
            for (uint32_t n = 0; n < NT; ++n) {
                const float a0 = alpha[n][0] * rescale, a1 = alpha[n][1] * rescale;
#pragma unroll
                for (uint32_t b = 0; b < NB; ++b) {
#pragma unroll
                    for (uint32_t k = 0; k < 2; ++k) {
                        o[n][b][k][0] *= a0;
                        o[n][b][k][1] *= a1;
                        o[n][b][k][2] *= a0;
                        o[n][b][k][3] *= a1;
                    }
                    wsum[n][b][0] *= a0;
                    wsum[n][b][1] *= a1;
                }
            }
        }
        if (tiny) {
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e)
#pragma unroll
                for (uint32_t b = 0; b < NB; ++b) dv[e][b] = __hmul2(dv[e][b], __float2half2_rn((float)(1 << kTinyUp)));
        }
        // the weights of each block, cells now along the lane's pairs and row g in the column
        uint32_t wb[NT][SPLIT ? 2 : 1][4][NB];
#pragma unroll
        for (uint32_t n = 0; n < NT; ++n)
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) {
                const __half2 h = __floats2half2_rn(s[n][0][e], s[n][1][e]);
                __half2 ph = as_h2(transpose8(as_u32(h))), pl;
                if (SPLIT) {
                    const float2 back = __half22float2(h);
                    pl = as_h2(transpose8(pack2(s[n][0][e] - back.x, s[n][1][e] - back.y)));
                }
#pragma unroll
                for (uint32_t b = 0; b < NB; ++b) {
                    const __half2 x = __hmul2(ph, dv[e][b]);
                    wb[n][0][e][b] = as_u32(x);
                    if (SPLIT) wb[n][SPLIT ? 1 : 0][e][b] = as_u32(__hfma2(pl, dv[e][b], __hfma2(ph, dv[e][b], __hneg2(x))));
                }
            }
#pragma unroll
        for (uint32_t ks = 0; ks < 2; ++ks) {
            uint32_t v[4][NB / 2];
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                const uint8_t* p = sk + v_at + (16u * ks + 8u * (j >> 1)) * S::ROW + (j & 1u ? v_step : 0);
                if constexpr (NB == 4) {
                    const uint2 x = *reinterpret_cast<const uint2*>(p);
                    v[j][0] = x.x;
                    v[j][1] = x.y;
                } else
                    v[j][0] = *reinterpret_cast<const uint32_t*>(p);
            }
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b) {
                const uint32_t sel = b & 1u ? 0x7632 : 0x5410;
                const uint32_t x0 = __byte_perm(v[0][b / 2], v[1][b / 2], sel), x1 = __byte_perm(v[2][b / 2], v[3][b / 2], sel);
                const uint32_t y0 = x0 >> 8, y1 = x1 >> 8;
                const uint32_t e0 = even(x0), e1 = even(x1), o0 = odd(x0), o1 = odd(x1);
                const uint32_t f0 = even(y0), f1 = even(y1), p0 = odd(y0), p1 = odd(y1);
#pragma unroll
                for (uint32_t n = 0; n < NT; ++n)
#pragma unroll
                    for (uint32_t k = 0; k < (SPLIT ? 2u : 1u); ++k) {
                        const uint32_t b0 = wb[n][k][2 * ks][b], b1 = wb[n][k][2 * ks + 1][b];
                        float (&p)[4] = o[n][b][0];
                        mma16816(p, e0, o0, e1, o1, b0, b1, p[0], p[1], p[2], p[3]);
                        float (&q)[4] = o[n][b][1];
                        mma16816(q, f0, p0, f1, p1, b0, b1, q[0], q[1], q[2], q[3]);
                    }
            }
        }
#pragma unroll
        for (uint32_t n = 0; n < NT && !WHOLE; ++n)
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b) {
                constexpr uint32_t k8 = 0x00080008u;
                float c[4];
                mma16816(c, k8, k8, k8, k8, wb[n][0][0][b], wb[n][0][1][b], 0.0f, 0.0f, 0.0f, 0.0f);
                mma16816(c, k8, k8, k8, k8, wb[n][0][2][b], wb[n][0][3][b], c[0], c[1], c[2], c[3]);
                if constexpr (SPLIT) {
                    mma16816(c, k8, k8, k8, k8, wb[n][1][0][b], wb[n][1][1][b], c[0], c[1], c[2], c[3]);
                    mma16816(c, k8, k8, k8, k8, wb[n][1][2][b], wb[n][1][3][b], c[0], c[1], c[2], c[3]);
                }
                wsum[n][b][0] += c[0];
                wsum[n][b][1] += c[1];
            }
        stage = stage + 1u == kDecStages ? 0u : stage + 1u;
        __syncwarp();                                            // the tile is read: its stage may be filled
    }
    cp_wait<0>();
    __syncwarp();

    // the warp's results in its ring: [R][W] outputs without their scales; maxima and sums beside the rings
    float* wo = reinterpret_cast<float*>(ringp);
#pragma unroll
    for (uint32_t x = 4; x < 32; x <<= 1) lost |= __shfl_xor_sync(0xFFFFFFFFu, lost, x);
    const float pinv = pow2(-(int)kWeightUp), unscale = pinv * pow2((WHOLE ? 0 : 24) - (tiny ? kTinyUp : 0));
#pragma unroll
    for (uint32_t n = 0; n < NT; ++n) {
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b)
#pragma unroll
            for (uint32_t k = 0; k < 2; ++k)
#pragma unroll
                for (uint32_t i = 0; i < 2; ++i) {
                    float* p = wo + (8u * n + 2u * t + i) * S::W + 32u * b + 4u * g + 2u * k;
                    const bool none = lost >> (4u * (2u * n + i) + b) & 1u;
                    p[0] = none ? NAN : (o[n][b][k][i] - wsum[n][b][i]) * unscale;
                    p[1] = none ? NAN : (o[n][b][k][2 + i] * kOdd - wsum[n][b][i]) * unscale;
                }
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) {
            float x = l[n][i] * pinv;
#pragma unroll
            for (uint32_t k = 4; k < 32; k <<= 1) x += __shfl_xor_sync(0xFFFFFFFFu, x, k);
            if (g == 0) red[warp * 16u + 8u * n + 2u * t + i] = make_float4(MASK ? off[n][i] : 0.0f, m[n][i], x, 0.0f);
        }
    }
    __syncthreads();
    // Each warp's factor for each row (a thread per row, in order; the warps of a team share sums, and maxima but for far scales),
    // the CTA's maximum and sum; then the teams' outputs, four values a thread, into the first team's place.
    auto result = [&](uint32_t j, uint32_t r, uint32_t d) {
        return reinterpret_cast<float4*>(sm + (j * S::NG + d / S::W) * S::RING) + (r * S::W + d % S::W) / 4u;
    };
    float4* fin = red + WARPS * 16u;
    if (tid < R) {
        const uint32_t r = tid;
        float ot = -INFINITY, mt = -INFINITY, lt = 0.0f;
        if (MASK) {
#pragma unroll
            for (uint32_t j = 0; j < WARPS; ++j) ot = fmaxf(ot, red[j * 16u + r].x);
        }
        auto level = [&](const float4& p) { return !MASK || p.x == ot || p.y == -INFINITY ? p.y : p.y + (p.x - ot) * kLog2e; };
#pragma unroll
        for (uint32_t j = 0; j < WARPS; ++j) mt = fmaxf(mt, level(red[j * 16u + r]));
        const float base = mt == -INFINITY ? 0.0f : mt;
#pragma unroll
        for (uint32_t j = 0; j < WARPS; ++j) {
            const float4 p = red[j * 16u + r];
            const float f = p.z == 0.0f ? 0.0f : ex2(level(p) - base);       // a warp that saw nothing of the row: 0
            if (j % S::NG == 0) lt += f * p.z;
            red[j * 16u + r].w = f;
        }
        fin[r] = make_float4(ot, mt, lt, 0.0f);
    }
    __syncthreads();
    for (uint32_t e = tid; e < R * D / 4u; e += WARPS * 32u) {
        const uint32_t r = e / (D / 4u), d = e % (D / 4u) * 4u;
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (uint32_t j = 0; j < S::TEAMS; ++j) {
            const float f = red[(j * S::NG + d / S::W) * 16u + r].w;         // outputs are finite or marked by NaN, which a factor of 0 keeps
            const float4 x = *result(j, r, d);
            acc.x += f * x.x; acc.y += f * x.y; acc.z += f * x.z; acc.w += f * x.w;
        }
        *result(0, r, d) = acc;
    }
    __syncthreads();
    const uint32_t used = min(R, rows - rt * R);
    if (a.splits > 1u && a.part_o) {                             // joined by the merge kernel
        for (uint32_t e = tid; e < used * D / 4u; e += WARPS * 32u) {
            const uint32_t r = e / (D / 4u), d = e % (D / 4u) * 4u;
            const size_t at = ((size_t)unit * a.splits + split) * R + r;
            *reinterpret_cast<float4*>(a.part_o + at * D + d) = *result(0, r, d);
            if (d == 0) *reinterpret_cast<float4*>(a.part_ml + at * 4u) = fin[r];
        }
        return;
    }
    auto put = [&](uint32_t r, uint32_t d, float4 x, float l) {
        const uint32_t row = rt * R + r, tok = grp * a.group + row / a.G, h = hk * a.G + row % a.G;
        const float f = l == 0.0f ? 0.0f : 1.0f / l;
        float y[4] = {x.x * f, x.y * f, x.z * f, x.w * f};
        if (l == 0.0f) y[0] = y[1] = y[2] = y[3] = 0.0f;
        T* p = static_cast<T*>(a.out) + (size_t)tok * a.out_stride + (size_t)h * D + d;
        store4<T>(p, y, a.out_wide);
    };
    if (a.splits == 1u) {
        for (uint32_t e = tid; e < used * D / 4u; e += WARPS * 32u) {
            const uint32_t r = e / (D / 4u), d = e % (D / 4u) * 4u;
            put(r, d, *result(0, r, d), fin[r].z);
        }
        return;
    }
    // The cluster's CTAs, in order: each takes its share of the outputs. A thread per row and CTA finds the factors.
    float* share = xch;                                          // [R][kMaxCluster + 4]: each CTA's factor, then the sum
    cluster_sync();
    for (uint32_t e = tid; e < R * kMaxCluster; e += WARPS * 32u) {
        const uint32_t r = e / kMaxCluster, k = e % kMaxCluster;
        float4 p = make_float4(-INFINITY, -INFINITY, 0.0f, 0.0f);
        if (k < a.splits) p = remote_f32x4(fin + r, k);
        if (MASK) {
            float top = p.x;
#pragma unroll
            for (uint32_t x = 1; x < kMaxCluster; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, x));
            if (p.x != top && p.y != -INFINITY) p.y += (p.x - top) * kLog2e;
        }
        float top = p.y;
#pragma unroll
        for (uint32_t x = 1; x < kMaxCluster; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, x));
        const float f = p.z == 0.0f ? 0.0f : ex2(p.y - (top == -INFINITY ? 0.0f : top));
        float sum = p.z == 0.0f ? 0.0f : f * p.z;
#pragma unroll
        for (uint32_t x = 1; x < kMaxCluster; x <<= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, x);
        share[r * (kMaxCluster + 4u) + k] = f;
        if (k == 0) share[r * (kMaxCluster + 4u) + kMaxCluster] = sum;
    }
    __syncthreads();
    for (uint32_t e = split * WARPS * 32u + tid; e < used * D / 4u; e += a.splits * WARPS * 32u) {
        const uint32_t r = e / (D / 4u), d = e % (D / 4u) * 4u;
        const float* f = share + r * (kMaxCluster + 4u);
        float4 x[kMaxCluster], acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (uint32_t k = 0; k < kMaxCluster; ++k)
            if (k < a.splits) x[k] = remote_f32x4(result(0, r, d), k);
#pragma unroll
        for (uint32_t k = 0; k < kMaxCluster; ++k)
            if (k < a.splits) {
                acc.x += f[k] * x[k].x; acc.y += f[k] * x[k].y; acc.z += f[k] * x[k].z; acc.w += f[k] * x[k].w;
            }
        put(r, d, acc, f[kMaxCluster]);
    }
    cluster_sync();                                              // nobody's shared memory goes while it is read
}

// Adds up the splits of each row in order. One CTA per row of a unit.
template <class T, int D, uint32_t R>
__global__ void __launch_bounds__(128) fa4_merge_kernel(Fa4Args a) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t unit = blockIdx.x, r = blockIdx.y;
    const uint32_t hk = unit % a.n_head_kv, rt = unit / a.n_head_kv % a.row_tiles, grp = unit / (a.n_head_kv * a.row_tiles);
    const uint32_t row = rt * R + r;
    if (row >= a.group * a.G) return;
    const float4* ml = reinterpret_cast<const float4*>(a.part_ml) + (size_t)unit * a.splits * R + r;
    const float* po = a.part_o + ((size_t)unit * a.splits * R + r) * D;
    float ot = -INFINITY, mt = -INFINITY, lt = 0.0f;
    for (uint32_t s = threadIdx.x & 31u; s < a.splits; s += 32u) ot = fmaxf(ot, ml[(size_t)s * R].x);
    for (int x = 16; x; x >>= 1) ot = fmaxf(ot, __shfl_xor_sync(0xFFFFFFFFu, ot, x));
    auto level = [&](const float4& p) { return p.x == ot || p.y == -INFINITY ? p.y : p.y + (p.x - ot) * kLog2e; };
    for (uint32_t s = threadIdx.x & 31u; s < a.splits; s += 32u) mt = fmaxf(mt, level(ml[(size_t)s * R]));
    for (int x = 16; x; x >>= 1) mt = fmaxf(mt, __shfl_xor_sync(0xFFFFFFFFu, mt, x));
    const float base = mt == -INFINITY ? 0.0f : mt;
    constexpr uint32_t N = D / 128 ? D / 128 : 1;
    float acc[N] = {};
#pragma unroll 8
    for (uint32_t s = 0; s < a.splits; ++s) {
        const float4 p = ml[(size_t)s * R];
        const float f = p.z == 0.0f ? 0.0f : ex2(level(p) - base);
        if (p.z != 0.0f) lt += f * p.z;
#pragma unroll
        for (uint32_t k = 0; k < N; ++k)
            if (threadIdx.x + 128u * k < D) {
                const float x = po[(size_t)s * R * D + threadIdx.x + 128u * k];
                if (p.z != 0.0f) acc[k] += f * x;
            }
    }
    const uint32_t tok = grp * a.group + row / a.G, h = hk * a.G + row % a.G;
    T* out = static_cast<T*>(a.out) + (size_t)tok * a.out_stride + (size_t)h * D;
#pragma unroll
    for (uint32_t k = 0; k < N; ++k)
        if (threadIdx.x + 128u * k < D) out[threadIdx.x + 128u * k] = from_f32<T>(lt == 0.0f ? 0.0f : acc[k] / lt);
}

// The shape of a call: which rows a CTA takes and how the cells are split.
struct Fa4Plan {
    int mode;
    uint32_t group, row_tiles, units, splits, tile_rows;
    size_t o_bytes, ml_bytes;                  // of the workspace, where a merge kernel joins the splits
};

constexpr uint32_t kMaxT = 1u << 20;
Fa4Plan fa4_plan(uint32_t type, uint32_t n_head_kv, uint32_t D, uint32_t T, uint32_t n_head, uint32_t n_kv, uint32_t group, uint32_t max_len, bool mask) {
    Fa4Plan p{};
    p.group = group ? group : T;
    const uint32_t rows = p.group * (n_head / n_head_kv);
    p.splits = 1;
    const uint32_t len = max_len && max_len < n_kv ? max_len : n_kv;

    // The kernel for few rows. Splits in powers of two up to a cluster's CTAs, each warp keeping a tile at least: until the
    // GPU's places for CTAs (four an SM; three with 16 rows, whose registers are more) are taken, since a CTA costs about
    // three tiles' time beside its tiles; and where a warp keeps eight tiles even so, once more, which evens out what the
    // last CTAs leave idle (64 ragged sequences, 512 units: 80 us with 2, 89 with 1, 85 with 4). Clusters of sixteen only
    // where two CTAs an SM are all there are: more of them do not fit side by side (8 tokens, 32 / 8 heads, 4113 cells in
    // f16: 28 us with 16, 18.5 with 8). Where even these leave most SMs empty and the cells are many, more splits and a
    // merge kernel.
    p.mode = type != TSRC_TYPE_BF16 ? kRows8Split : rows <= 8u ? kRows8 : kRows16;
    const uint32_t R = p.mode == kRows16 ? 16u : 8u, all = (R == 16u ? 3u : 4u) * kSms;
    p.row_tiles = (rows + R - 1u) / R;
    p.units = (T / p.group) * n_head_kv * p.row_tiles;
    const uint32_t teams = D <= 128u ? kDecWarps : kDecWarps * 128u / D;
    const uint32_t tiles = len / kDecTile + 1u, most = tiles / teams;
    while (p.splits < (p.units <= 2u * kSms / kMaxCluster ? kMaxCluster : 8u) && p.splits * 2u <= most && p.units < all &&
           (p.units * p.splits * 2u <= all || (p.units * p.splits < all && tiles >= 16u * teams * p.splits)))
        p.splits *= 2u;
    const bool merge = p.units <= (kSms - 1u) / kMaxCluster && most >= 8u * kMaxCluster;
    const uint32_t parts = merge ? std::min(2u * kSms / p.units, most / 2u) : p.splits;      // a warp keeps two tiles
    if (D <= 128u) {
        // The kernel for many rows where it is the faster one, by what both measured (ns). Its CTAs take 1.25 (bf16) to 1.75
        // us (f32) for a tile of 64 cells, 1.4 to 1.8 more under a mask, and are split over the cells as far as there are
        // SMs; a split costs the merge about a sixth of a tile, so that the tiles left to each and the splits are balanced.
        // The other kernel's warps take 2 us for 32 cells of 8 rows (3 for 16) up to two CTAs an SM, then in proportion
        // to those. f16, 32 / 8 heads, 4113 cells: 8 tokens 19.6 us here and 18.5 there, 13 tokens 19.8 and 23.2, 64 tokens
        // 28.6 and 72; 16384 cells: 13 tokens 35 and 65.
        const uint64_t units = (uint64_t)(T / p.group) * n_head_kv * ((rows + kFa4TcRows - 1u) / kFa4TcRows), blocks = len / 64u + 1u;
        const uint64_t each = (type == TSRC_TYPE_BF16 ? 1250u : type == TSRC_TYPE_F16 ? 1450u : 1750u) + (!mask ? 0u : type == TSRC_TYPE_BF16 ? 1400u : 1800u);
        const uint64_t places = !mask && (type == TSRC_TYPE_BF16 || D == 64u) ? 2u * kSms : kSms;
        uint64_t splits = 1;
        while ((splits + 1u) * units <= kSms && (splits + 1u) * (splits + 1u) <= 6u * blocks && 2u * (splits + 1u) <= blocks) ++splits;
        const uint64_t tc = (units * splits + places - 1u) / places * ((blocks + splits - 1u) / splits) * each +
                            (splits > 1u ? 13000u + (uint64_t)T * n_head * splits * D / 750u : 8200u);
        const uint64_t ctas = (uint64_t)p.units * parts, share = (uint64_t)teams * ctas / p.units;
        const uint64_t busy = ctas * (R == 16u ? 1700u : 1050u) / kSms, alone = R == 16u ? 3000u : 2000u;
        const uint64_t dec = 8000u + (tiles + share - 1u) / share * (busy > alone ? busy : alone) / (D == 64u ? 2u : 1u) + (merge ? 3000u : 0u);
        if (tc < dec) {
            const uint64_t wide = (uint64_t)(T / p.group) * n_head_kv * ((rows + 2u * kFa4TcRows - 1u) / (2u * kFa4TcRows));
            // bf16: 256 rows a CTA where 128 give at least four CTAs to three SMs, and 256, of which an SM holds one, take no
            // more turns (32 / 8 heads, us with 256 and 128: 2048 tokens, causal 70 and 82; 4096 cells before 640 tokens 109 and
            // 125; before 1184, in two turns, 193 and 140; 400 tokens 23 and 19). For f16 they win 8 % at most and are not there.
            const bool two = type == TSRC_TYPE_BF16 && 3u * units >= 4u * kSms && (wide + kSms - 1u) / kSms <= (units + places - 1u) / places;
            p.mode = kRows128;
            p.tile_rows = two ? 2u * kFa4TcRows : kFa4TcRows;
            p.row_tiles = (rows + p.tile_rows - 1u) / p.tile_rows;
            p.units = (uint32_t)(two ? wide : units);
            p.splits = (uint32_t)splits;
            if (p.splits > 1u) {
                p.o_bytes = (size_t)p.units * p.splits * kFa4TcRows * D * 4u;
                p.ml_bytes = (size_t)p.units * p.splits * kFa4TcRows * 16u;
            }
            return p;
        }
    }
    if (merge) {
        p.splits = parts;
        p.o_bytes = (size_t)p.units * p.splits * R * D * 4u;
        p.ml_bytes = (size_t)p.units * p.splits * R * 16u;
    }
    return p;
}

// Joins the splits that a kernel left in the workspace.
template <class T, int D, uint32_t R>
cudaError_t merge_launch(const Fa4Args& a, uint32_t units, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    cfg.gridDim = dim3(units, R);
    cfg.blockDim = dim3(128);
    cfg.stream = st;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, fa4_merge_kernel<T, D, R>, a);
}
template <class T>
cudaError_t tc_launch(uint32_t type, uint32_t D, const Fa4Args& a, uint32_t units, cudaStream_t st) {
    cudaError_t e = launch_fa4_tc(type, D, a, units, st);
    if (e != cudaSuccess || a.splits == 1u) return e;
    return D == 64u ? merge_launch<T, 64, kFa4TcRows>(a, units, st) : merge_launch<T, 128, kFa4TcRows>(a, units, st);
}

template <class T, int D, int MODE, bool MASK>
cudaError_t dec_launch_m(const Fa4Args& a, uint32_t units, cudaStream_t st) {
    constexpr uint32_t smem = dec_smem<D, MODE>();
    static bool done[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !done[dev]) {             // the kernel's attributes, set once per device
        e = cudaFuncSetAttribute(fa4_dec_kernel<T, D, MODE, MASK>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(fa4_dec_kernel<T, D, MODE, MASK>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
        if (dev < 64) done[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    cfg.gridDim = dim3(units * a.splits);
    cfg.blockDim = dim3(kDecWarps * 32u);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    if (a.splits > 1u && !a.part_o) {
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = a.splits;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.numAttrs = 1;
    }
    e = cudaLaunchKernelEx(&cfg, fa4_dec_kernel<T, D, MODE, MASK>, a);
    return e != cudaSuccess || !a.part_o ? e : merge_launch<T, D, kRowsOf<MODE>>(a, units, st);
}
template <class T, int D, int MODE>
cudaError_t dec_launch(const Fa4Args& a, uint32_t units, cudaStream_t st) {
    return a.mask ? dec_launch_m<T, D, MODE, true>(a, units, st) : dec_launch_m<T, D, MODE, false>(a, units, st);
}
template <class T, int MODE>
cudaError_t dec_launch_d(const Fa4Args& a, uint32_t D, uint32_t units, cudaStream_t st) {
    switch (D) {
        case 64: return dec_launch<T, 64, MODE>(a, units, st);
        case 128: return dec_launch<T, 128, MODE>(a, units, st);
        case 256: return dec_launch<T, 256, MODE>(a, units, st);
        default: return dec_launch<T, 512, MODE>(a, units, st);
    }
}

}  // namespace

}  // namespace tsrc

using namespace tsrc;

extern "C" {

const char* tsrc_flash_attn_q4_unsupported(uint32_t type, uint32_t n_head_kv, uint32_t head_dim, uint32_t n_head) {
    if (!kv4_type_ok(type)) return "FLASH_ATTN over q4_0: q and out must be f32, f16 or bf16";
    if (!kv4_geometry_ok(n_head_kv, head_dim)) return "FLASH_ATTN over q4_0: head_dim must be 64/128/256/512, n_head_kv * head_dim / 64 in 1..511";
    if (n_head == 0 || n_head % n_head_kv) return "FLASH_ATTN over q4_0: n_head is not a positive multiple of n_head_kv";
    if (n_head / n_head_kv > 64u) return "FLASH_ATTN over q4_0: more than 64 query heads on a KV head";
    return nullptr;
}

size_t tsrc_flash_attn_q4_workspace(uint32_t type, uint32_t n_head_kv, uint32_t head_dim, uint32_t T, uint32_t n_head,
                                    uint32_t n_kv, uint32_t group, uint32_t max_len) {
    if (T == 0 || T > kMaxT || (group && T % group) || tsrc_flash_attn_q4_unsupported(type, n_head_kv, head_dim, n_head)) return 0;
    const Fa4Plan p = fa4_plan(type, n_head_kv, head_dim, T, n_head, n_kv, group, max_len, false);
    const Fa4Plan m = fa4_plan(type, n_head_kv, head_dim, T, n_head, n_kv, group, max_len, true);
    return std::max(p.o_bytes + p.ml_bytes, m.o_bytes + m.ml_bytes);        // a call may have a mask
}

int tsrc_flash_attn_q4(tsrc_ctx* ctx, const tsrc_kv4* kv, uint32_t type, const void* q, uint32_t q_stride, uint32_t T, uint32_t n_head,
                       uint32_t n_kv, const int32_t* ranges, uint32_t group, uint32_t max_len, const uint16_t* mask,
                       uint32_t mask_stride, float scale, void* out, uint32_t out_stride, void* ws, size_t ws_bytes, void* stream) {
    if (!ctx || !kv || !q || !out) return set_error(TSRC_E_ARG, "tsrc_flash_attn_q4: NULL argument");
    if (kv->ctx != ctx) return set_error(TSRC_E_ARG, "tsrc_flash_attn_q4: the cache belongs to another context");
    if (const char* why = tsrc_flash_attn_q4_unsupported(type, kv->n_head_kv, kv->D, n_head)) return set_error(TSRC_E_SHAPE, why);
    if (n_kv > kv->n_cells) return refuse(TSRC_E_ARG, "tsrc_flash_attn_q4: n_kv %u exceeds the cache's %u cells", n_kv, kv->n_cells);
    const uint32_t row = n_head * kv->D;
    if (q_stride == 0) q_stride = row;
    if (out_stride == 0) out_stride = row;
    if (q_stride < row || out_stride < row) return set_error(TSRC_E_ARG, "tsrc_flash_attn_q4: a stride is shorter than n_head * head_dim");
    if (mask && mask_stride == 0) mask_stride = n_kv;
    if (mask && mask_stride < n_kv) return set_error(TSRC_E_ARG, "tsrc_flash_attn_q4: mask_stride < n_kv");
    if (!std::isfinite(scale)) return set_error(TSRC_E_ARG, "tsrc_flash_attn_q4: scale is not finite");
    if (group == 0) group = T;
    if (T && T % group) return refuse(TSRC_E_ARG, "tsrc_flash_attn_q4: T %u is not a multiple of group %u", T, group);
    if (T > kMaxT) return set_error(TSRC_E_SHAPE, "tsrc_flash_attn_q4: T above 2^20");
    const uintptr_t m = kv4_type_size(type) - 1u;
    if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & m) || (reinterpret_cast<uintptr_t>(ranges) & 3u) ||
        (reinterpret_cast<uintptr_t>(mask) & 1u))
        return set_error(TSRC_E_ARG, "tsrc_flash_attn_q4: a pointer is not aligned to its elements");
    const size_t need = tsrc_flash_attn_q4_workspace(type, kv->n_head_kv, kv->D, T, n_head, n_kv, group, max_len);
    if (need && (!ws || ws_bytes < need || (reinterpret_cast<uintptr_t>(ws) & 255u)))
        return refuse(TSRC_E_ARG, "tsrc_flash_attn_q4: the workspace must be 256-byte aligned and hold %zu bytes", need);
    if (T == 0) return TSRC_OK;
    DeviceScope scope(ctx);
    if (scope.rc) return scope.rc;
    const Fa4Plan p = fa4_plan(type, kv->n_head_kv, kv->D, T, n_head, n_kv, group, max_len, mask != nullptr);
    Fa4Args a{};
    a.q = q;
    a.out = out;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    const uint32_t size = kv4_type_size(type);
    a.q_wide = (reinterpret_cast<uintptr_t>(q) & 15u) == 0 && (size_t)q_stride * size % 16u == 0;
    a.out_wide = (reinterpret_cast<uintptr_t>(out) & (4u * size - 1u)) == 0 && out_stride % 4u == 0;
    a.kq = kv->q[0];
    a.vq = kv->q[1];
    a.kd = kv->d[0];
    a.vd = kv->d[1];
    a.T = T;
    a.n_head = n_head;
    a.n_head_kv = kv->n_head_kv;
    a.G = n_head / kv->n_head_kv;
    a.n_kv = n_kv;
    a.n_alloc = kv->n_alloc;
    a.ranges = ranges;
    a.mask = reinterpret_cast<const __half*>(mask);
    a.mask_stride = mask_stride;
    a.mask_wide = (reinterpret_cast<uintptr_t>(mask) & 15u) == 0 && mask_stride % 8u == 0;
    a.scale = scale;
    a.group = p.group;
    a.row_tiles = p.row_tiles;
    a.tile_rows = p.tile_rows;
    a.splits = p.splits;
    if (p.o_bytes) {
        a.part_o = static_cast<float*>(ws);
        a.part_ml = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + p.o_bytes);
    }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (p.mode == kRows128)
        e = type == TSRC_TYPE_F32 ? tc_launch<float>(type, kv->D, a, p.units, st) : type == TSRC_TYPE_F16 ? tc_launch<__half>(type, kv->D, a, p.units, st)
                                                                                                      : tc_launch<__nv_bfloat16>(type, kv->D, a, p.units, st);
    else if (type == TSRC_TYPE_F32) e = dec_launch_d<float, kRows8Split>(a, kv->D, p.units, st);
    else if (type == TSRC_TYPE_F16) e = dec_launch_d<__half, kRows8Split>(a, kv->D, p.units, st);
    else e = p.mode == kRows8 ? dec_launch_d<__nv_bfloat16, kRows8>(a, kv->D, p.units, st) : dec_launch_d<__nv_bfloat16, kRows16>(a, kv->D, p.units, st);
    return e == cudaSuccess ? TSRC_OK : cuda_refuse(e, "tsrc_flash_attn_q4");
}

}  // extern "C"
