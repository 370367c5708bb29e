// tsrc_fa4.cu -- attention over the q4_0 KV cache (tsrc_flash_attn_q4). Cache layout: tsrc_kv4.cuh.
#include <cmath>
#include <cstdio>

#include "tsrc_kv4.cuh"

namespace tsrc {

namespace {

constexpr uint32_t kDecWarps = 4, kDecTile = 32;
constexpr uint32_t kDecCtas = 3 * 148;         // CTAs that fill a B200 once, three to an SM

struct Fa4Args {
    const void* q;
    void* out;
    size_t q_stride, out_stride;
    const uint8_t *kq, *vq;
    const __half *kd, *vd;
    uint32_t T, n_head, n_head_kv, G, n_kv, n_alloc;
    const int32_t* ranges;
    const __half* mask;
    size_t mask_stride;
    float scale;
    uint32_t group, row_tiles, splits;         // tokens a group, row tiles a group and KV head, splits of the cells
    float *part_o, *part_ml;                   // splits > 1: [unit][split][R][D], [unit][split][R][4]
};

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
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ __half2 as_h2(uint32_t u) { return *reinterpret_cast<const __half2*>(&u); }
__device__ __forceinline__ uint32_t as_u32(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }

// how a warp's sixteen mma rows are used
enum : int {
    kRows8Split = 0,       // eight query rows; rows 8..15 carry the second fp16 term of q and of the weights
    kRows8 = 1,            // eight query rows, one fp16 term (bf16 outputs)
    kRows16 = 2,           // sixteen query rows, one fp16 term (bf16 outputs)
};
template <int MODE> constexpr uint32_t kRowsOf = MODE == kRows16 ? 16u : 8u;

template <int D> struct DecShape {
    static constexpr uint32_t NB = D == 64 ? 2 : 4;            // blocks of a warp's group of values
    static constexpr uint32_t W = NB * 32;                      // values of a group: a warp's share of the head
    static constexpr uint32_t NG = D / W;                       // warps of a team: they share a tile's scores
    static constexpr uint32_t TEAMS = kDecWarps / NG;
    static constexpr uint32_t ROW = W / 2, DS = NB * 2;         // bytes of a cell's codes and scales in a group
    static constexpr uint32_t V_AT = kDecTile * ROW, KD_AT = 2 * kDecTile * ROW, VD_AT = KD_AT + kDecTile * DS;
    static constexpr uint32_t STAGE = VD_AT + kDecTile * DS;
    static constexpr uint32_t STAGES = NG > 1 ? 3 : 4;          // three CTAs' rings fit an SM
    static constexpr uint32_t RING = STAGE * STAGES;
};
template <int D, int MODE> __host__ __device__ constexpr uint32_t dec_smem() {
    using S = DecShape<D>;
    // ring (later the warps' results), score exchange of teams (two turns), maxima and sums of the warps
    return kDecWarps * S::RING + (S::NG > 1 ? 2u * kDecWarps * 32u * (MODE == kRows16 ? 16u : 8u) * 4u : 0u) + kDecWarps * 16u * 3u * 4u;
}

// Decode attention, one pass over the cells.
//   A CTA takes up to 8 (16) query rows -- the (token, head) pairs of a group that share a KV head -- and one split
// of the cells they span, its warps tiles of 32 cells in turn (D > 128: teams of D / 128 warps, each with 128 values
// of the head, which add up their partial scores through shared memory). Tiles come by cp.async, four deep.
//   Codes go to the tensor cores as they are: a code n in the low four bits of an fp16 is the subnormal number
// n 2^-24, in the next four n 2^-20 (q's values that meet those carry 2^-4), so an operand register of two codes
// is one AND of a word of eight (and a shift for every second pair). What is missing, sum q (n - 8) = sum q n -
// 8 sum q, is the accumulator's start value for K; for V the weights' sum comes from one more mma per block with
// 8 2^-24 in every column. The blocks' scales stay out of the products: K's multiply the four (two) partial
// sums of a score in f32; V's multiply the weights: w = p dV, one set of weights per block.
//   Precision: q and w are two fp16 terms each, 22 bits (q scaled by a power of two per row, the weights by 2^14
// and by a power of two that follows the largest |dV| seen, so that neither term leaves fp16's range); for bf16
// outputs one term, 11 bits. Running maximum, sum and outputs are f32.
template <class T, int D, int MODE, bool MASK>
__global__ void __launch_bounds__(kDecWarps * 32, 3) fa4_dec_kernel(Fa4Args a) {
    using S = DecShape<D>;
    constexpr uint32_t NB = S::NB, R = kRowsOf<MODE>, RS = MODE == kRows16 ? 2 : 1;   // RS: rows of a lane
    extern __shared__ __align__(128) uint8_t sm[];
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, g = lane >> 2, t = lane & 3u;
    const uint32_t team = warp / S::NG, sub = warp % S::NG;
    const uint32_t unit = blockIdx.x, split = blockIdx.y;
    const uint32_t hk = unit % a.n_head_kv, rt = unit / a.n_head_kv % a.row_tiles, grp = unit / (a.n_head_kv * a.row_tiles);
    const uint32_t rows = a.group * a.G;
    const uint32_t ring = smem_u32(sm) + warp * S::RING;
    uint8_t* ringp = sm + warp * S::RING;
    float* xch = reinterpret_cast<float*>(sm + kDecWarps * S::RING);
    float* red = reinterpret_cast<float*>(sm + dec_smem<D, MODE>() - kDecWarps * 16u * 3u * 4u);      // [warp][16][3]

    // the rows' cells, and the hull of them
    int32_t lo[RS], hi[RS], first = 0x7FFFFFFF, last = 0;
    const T* qrow[RS];
    const __half* mrow[RS];
#pragma unroll
    for (uint32_t r = 0; r < RS; ++r) {
        const uint32_t row = rt * R + g + 8u * r;
        lo[r] = hi[r] = 0;
        qrow[r] = nullptr;
        mrow[r] = a.mask;
        if (row < rows) {
            const uint32_t tok = grp * a.group + row / a.G, h = hk * a.G + row % a.G;
            hi[r] = (int32_t)a.n_kv;
            if (a.ranges) {
                lo[r] = max(a.ranges[2u * (size_t)tok], 0);
                hi[r] = min(a.ranges[2u * (size_t)tok + 1u], (int32_t)a.n_kv);
            }
            if (lo[r] >= hi[r]) lo[r] = hi[r] = 0;
            else {
                first = min(first, lo[r]);
                last = max(last, hi[r]);
            }
            qrow[r] = static_cast<const T*>(a.q) + (size_t)tok * a.q_stride + (size_t)h * D + sub * S::W;
            if (MASK) mrow[r] = a.mask + (size_t)tok * a.mask_stride;
        }
    }
    first = __reduce_min_sync(0xFFFFFFFFu, first);
    last = __reduce_max_sync(0xFFFFFFFFu, last);
    // the cells that every row sees (an unused row must not stop the shortcut: it has no cells to lose)
    int32_t all_lo = 0, all_hi = 0x7FFFFFFF;
#pragma unroll
    for (uint32_t r = 0; r < RS; ++r)
        if (qrow[r]) {
            all_lo = max(all_lo, lo[r]);
            all_hi = min(all_hi, hi[r]);
        }
    all_lo = __reduce_max_sync(0xFFFFFFFFu, all_lo);
    all_hi = __reduce_min_sync(0xFFFFFFFFu, all_hi);
    const uint32_t tile0 = (uint32_t)min(first, last) / kDecTile, tiles = last > first ? ((uint32_t)last + kDecTile - 1u) / kDecTile - tile0 : 0u;
    const uint32_t from = tile0 + (uint32_t)((uint64_t)tiles * split / a.splits) + team;
    const uint32_t to = tile0 + (uint32_t)((uint64_t)tiles * (split + 1u) / a.splits);

    const uint8_t* kq = a.kq + (size_t)hk * a.n_alloc * (D / 2) + sub * S::ROW;
    const uint8_t* vq = a.vq + (size_t)hk * a.n_alloc * (D / 2) + sub * S::ROW;
    const __half* kd = a.kd + (size_t)hk * a.n_alloc * (D / 32) + sub * NB;
    const __half* vd = a.vd + (size_t)hk * a.n_alloc * (D / 32) + sub * NB;
    auto fetch = [&](uint32_t tile, uint32_t stage) {
        const size_t c0 = (size_t)tile * kDecTile;
        const uint32_t at = ring + stage * S::STAGE;
        constexpr uint32_t PER = S::ROW / 16;                  // 16-byte pieces of a cell's codes
#pragma unroll
        for (uint32_t i = 0; i < PER; ++i) {
            const uint32_t p = lane + 32u * i, c = p / PER, w = p % PER;
            cp16(at + c * S::ROW + 16u * w, kq + (c0 + c) * (D / 2) + 16u * w);
            cp16(at + S::V_AT + c * S::ROW + 16u * w, vq + (c0 + c) * (D / 2) + 16u * w);
        }
        if constexpr (S::NG == 1) {                             // a tile's scales are one run
            constexpr uint32_t P = kDecTile * S::DS / 16;       // 16 pieces (8 for D = 64)
            if (lane < P) cp16(at + S::KD_AT + 16u * lane, reinterpret_cast<const uint8_t*>(kd + c0 * NB) + 16u * lane);
            else if (lane < 2u * P) cp16(at + S::VD_AT + 16u * (lane - P), reinterpret_cast<const uint8_t*>(vd + c0 * NB) + 16u * (lane - P));
        } else {
            cp8(at + S::KD_AT + 8u * lane, kd + (c0 + lane) * (D / 32));
            cp8(at + S::VD_AT + 8u * lane, vd + (c0 + lane) * (D / 32));
        }
    };
#pragma unroll
    for (uint32_t s = 0; s < S::STAGES - 1; ++s) {
        if (from + s * S::TEAMS < to) fetch(from + s * S::TEAMS, s);
        cp_commit();
    }

    // q's fragments: lane (g, t) owns values 8t .. 8t + 7 of each block of row g (and g + 8)
    uint32_t qa[NB][2][4];
    float start[NB][2], rs[RS];
    {
        float x[2][NB][8];
#pragma unroll
        for (uint32_t r = 0; r < 2; ++r)
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b)
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) x[r][b][i] = r < RS && qrow[r < RS ? r : 0] ? to_f32(qrow[r < RS ? r : 0][32u * b + 8u * t + i]) : 0.0f;
#pragma unroll
        for (uint32_t r = 0; r < RS; ++r) {
            float top = 0.0f;
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b)
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[r][b][i]));
            top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
            // the row's largest value to [2^12, 2^13); rows of tiny values by 2^100 at most
            const int e = min(12 - ((int)(__float_as_uint(top) >> 23) - 127), 100);
            const float f = __uint_as_float((uint32_t)(e + 127) << 23), inv = __uint_as_float((uint32_t)(127 - e) << 23);
            rs[r] = a.scale * 1.4426950408889634f * (inv * 16777216.0f);
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b)
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) x[r][b][i] *= f;
        }
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b) {
            float sum[2] = {};
            float y[2][8];                                       // what rows 0..7 and 8..15 of the operand hold
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                y[0][i] = __half2float(__float2half_rn(x[0][b][i]));
                if (MODE == kRows8Split) y[1][i] = __half2float(__float2half_rn(x[0][b][i] - y[0][i]));
                else if (MODE == kRows16) y[1][i] = __half2float(__float2half_rn(x[1][b][i]));
                else y[1][i] = 0.0f;
                sum[0] += y[0][i];
                sum[1] += y[1][i];
            }
#pragma unroll
            for (uint32_t r = 0; r < 2; ++r) {
                sum[r] += __shfl_xor_sync(0xFFFFFFFFu, sum[r], 1);
                sum[r] += __shfl_xor_sync(0xFFFFFFFFu, sum[r], 2);
                start[b][r] = sum[r] * (-8.0f / 16777216.0f);
#pragma unroll
                for (uint32_t j = 0; j < 2; ++j) {
                    qa[b][j][r] = pack2(y[r][2 * j], y[r][2 * j + 4]);
                    qa[b][j][2 + r] = pack2(y[r][2 * j + 1] * 0.0625f, y[r][2 * j + 5] * 0.0625f);
                }
            }
        }
    }

    float o[NB * 4][4] = {}, wsum[NB][2] = {}, m[RS], l[RS], off[RS];
    uint32_t vexp = 1;                                           // exponent field that the weights' scale follows
#pragma unroll
    for (uint32_t r = 0; r < RS; ++r) {
        m[r] = off[r] = -INFINITY;
        l[r] = 0.0f;
    }
    const uint32_t pg = g ^ ((g >> 1) & 1u);                      // the cell (of eight) whose scores column g holds
    const uint32_t c_a = (2u * t) ^ (t & 1u), c_b = c_a ^ 1u;     // the cells of this lane's columns 2t, 2t + 1

    uint32_t stage = 0, turn = 0;
    for (uint32_t tile = from; tile < to; tile += S::TEAMS) {
        {
            const uint32_t next = tile + (S::STAGES - 1) * S::TEAMS;
            if (next < to) fetch(next, (stage + S::STAGES - 1) % S::STAGES);
            cp_commit();
        }
        const uint32_t c0 = tile * kDecTile;
        float mk[RS][8];
        if (MASK) {
#pragma unroll
            for (uint32_t r = 0; r < RS; ++r)
#pragma unroll
                for (uint32_t j = 0; j < 8; ++j) {
                    const uint32_t c = c0 + 8u * (j / 2) + (j & 1u ? c_b : c_a);
                    mk[r][j] = (int32_t)c >= lo[r] && (int32_t)c < hi[r] ? __half2float(mrow[r][c]) : -INFINITY;
                }
        }
        cp_wait<S::STAGES - 1>();
        __syncwarp();
        const uint8_t* sk = ringp + stage * S::STAGE;
        float s[RS][8];
#pragma unroll
        for (uint32_t nt = 0; nt < 4; ++nt) {
            uint32_t w[4];
            const uint8_t* p = sk + (8u * nt + pg) * S::ROW + (t ^ ((pg >> 1) & 2u)) * (S::ROW / 4);
            if constexpr (NB == 4) {
                const uint4 v = *reinterpret_cast<const uint4*>(p);
                w[0] = __byte_perm(v.x, v.z, 0x5410);
                w[1] = __byte_perm(v.x, v.z, 0x7632);
                w[2] = __byte_perm(v.y, v.w, 0x5410);
                w[3] = __byte_perm(v.y, v.w, 0x7632);
            } else {
                const uint2 v = *reinterpret_cast<const uint2*>(p);
                w[0] = __byte_perm(v.x, v.y, 0x5410);
                w[1] = __byte_perm(v.x, v.y, 0x7632);
            }
            uint32_t da[NB / 2], db[NB / 2];
            const uint8_t* pd = sk + S::KD_AT + 8u * nt * S::DS;
            if constexpr (NB == 4) {
                const uint2 x = *reinterpret_cast<const uint2*>(pd + c_a * 8u), y = *reinterpret_cast<const uint2*>(pd + c_b * 8u);
                da[0] = x.x; da[1] = x.y; db[0] = y.x; db[1] = y.y;
            } else {
                da[0] = *reinterpret_cast<const uint32_t*>(pd + c_a * 4u);
                db[0] = *reinterpret_cast<const uint32_t*>(pd + c_b * 4u);
            }
            float acc[RS][2] = {};
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b) {
                const uint32_t x = w[b], y = x >> 8;
                float c[4] = {start[b][0], start[b][0], start[b][1], start[b][1]};
                mma16816(c, qa[b][0][0], qa[b][0][1], qa[b][0][2], qa[b][0][3], x & 0x000F000Fu, x & 0x00F000F0u);
                mma16816(c, qa[b][1][0], qa[b][1][1], qa[b][1][2], qa[b][1][3], y & 0x000F000Fu, y & 0x00F000F0u);
                const float2 fa = __half22float2(as_h2(da[b / 2])), fb = __half22float2(as_h2(db[b / 2]));
                const float ka = b & 1u ? fa.y : fa.x, kb = b & 1u ? fb.y : fb.x;
                if (MODE == kRows8Split) {
                    acc[0][0] = fmaf(c[0] + c[2], ka, acc[0][0]);
                    acc[0][1] = fmaf(c[1] + c[3], kb, acc[0][1]);
                } else {
                    acc[0][0] = fmaf(c[0], ka, acc[0][0]);
                    acc[0][1] = fmaf(c[1], kb, acc[0][1]);
                    if (RS == 2) {
                        acc[RS - 1][0] = fmaf(c[2], ka, acc[RS - 1][0]);
                        acc[RS - 1][1] = fmaf(c[3], kb, acc[RS - 1][1]);
                    }
                }
            }
#pragma unroll
            for (uint32_t r = 0; r < RS; ++r) {
                s[r][2 * nt] = acc[r][0] * rs[r];
                s[r][2 * nt + 1] = acc[r][1] * rs[r];
            }
        }
        if constexpr (S::NG > 1) {
            // the team's partial scores, added in the order of the groups
            float* mine = xch + ((turn * kDecWarps + warp) * RS * 8u) * 32u + lane;
#pragma unroll
            for (uint32_t r = 0; r < RS; ++r)
#pragma unroll
                for (uint32_t j = 0; j < 8; ++j) mine[(r * 8u + j) * 32u] = s[r][j];
            asm volatile("bar.sync %0, %1;" ::"r"(1u + team), "n"(32 * S::NG) : "memory");
            const float* all = xch + ((turn * kDecWarps + team * S::NG) * RS * 8u) * 32u + lane;
#pragma unroll
            for (uint32_t r = 0; r < RS; ++r)
#pragma unroll
                for (uint32_t j = 0; j < 8; ++j) {
                    float x = all[(r * 8u + j) * 32u];
#pragma unroll
                    for (uint32_t k = 1; k < S::NG; ++k) x += all[(k * RS * 8u + r * 8u + j) * 32u];
                    s[r][j] = x;
                }
            turn ^= 1u;
        }
        // what a row does not see: -inf here, and no scale of V below
        const bool open = !MASK && (int32_t)c0 >= all_lo && (int32_t)(c0 + kDecTile) <= all_hi;
        uint32_t seen[RS];
#pragma unroll
        for (uint32_t r = 0; r < RS; ++r) {
            seen[r] = 0xFFu;
            if (!open) {
#pragma unroll
                for (uint32_t j = 0; j < 8; ++j) {
                    const int32_t c = (int32_t)(c0 + 8u * (j / 2) + (j & 1u ? c_b : c_a));
                    const bool in = c >= lo[r] && c < hi[r] && !(MASK && mk[r][j] == -INFINITY);
                    if (!in) seen[r] &= ~(1u << j);
                }
            }
        }
        float alpha[RS];
        bool moved = false;
#pragma unroll
        for (uint32_t r = 0; r < RS; ++r) {
            float m_old = m[r];
            if (MASK) {
                // the mask's running maximum is taken out first: a row of the type's lowest value keeps its scores' digits
                float top = -INFINITY;
#pragma unroll
                for (uint32_t j = 0; j < 8; ++j) top = fmaxf(top, seen[r] >> j & 1u ? mk[r][j] : -INFINITY);
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
                const float off_new = fmaxf(off[r], top), base = off_new == -INFINITY ? 0.0f : off_new;
                if (off[r] != -INFINITY && off[r] != off_new) m_old += (off[r] - base) * 1.4426950408889634f;
                off[r] = off_new;
#pragma unroll
                for (uint32_t j = 0; j < 8; ++j) s[r][j] = fmaf(mk[r][j] - base, 1.4426950408889634f, s[r][j]);
            }
            float top = -INFINITY;
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j) {
                if (!open) s[r][j] = seen[r] >> j & 1u ? s[r][j] : -INFINITY;
                top = fmaxf(top, s[r][j]);
            }
            top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
            const float m_new = fmaxf(m_old, top);
            const float base = m_new == -INFINITY ? 0.0f : m_new;
            alpha[r] = ex2(m_old - base);
            moved |= m_new > m[r] || m_old != m[r];
            m[r] = m_new;
            l[r] *= alpha[r];
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j) {
                s[r][j] = ex2(s[r][j] - (base - 14.0f));         // 2^14 p: l and o share the factor
                l[r] += s[r][j];
            }
        }
        // V's scales as pairs (cells 2t, 2t + 1 of each eight), the largest of them, and the weights
        __half2 dv[4][NB];
        __half2 most = __float2half2_rn(0.0f);
#pragma unroll
        for (uint32_t nt = 0; nt < 4; ++nt) {
            const uint8_t* pd = sk + S::VD_AT + 8u * nt * S::DS;
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
                uint32_t v = __byte_perm(x[b / 2], y[b / 2], b & 1u ? 0x7632 : 0x5410);
                if (!open) {
                    uint32_t any = seen[0];
                    if (RS == 2) any |= seen[RS - 1];
                    v &= (any >> (2 * nt) & 1u ? 0x0000FFFFu : 0u) | (any >> (2 * nt) & 2u ? 0xFFFF0000u : 0u);
                }
                dv[nt][b] = as_h2(v);
                most = __hmax2(most, __habs2(dv[nt][b]));
            }
        }
        {
            const uint32_t u = as_u32(most), x = max(u & 0xFFFFu, u >> 16);
            const uint32_t e = __reduce_max_sync(0xFFFFFFFFu, x >= 0x7C00u ? 0u : x) >> 10;
            if (e > vexp) {                                      // the same for the whole warp
                const float f = __uint_as_float((127u + vexp - e) << 23);
                vexp = e;
#pragma unroll
                for (uint32_t r = 0; r < RS; ++r) alpha[r] *= f;
                moved = true;                                    // l does not have this factor
            }
        }
        if (__any_sync(0xFFFFFFFFu, moved)) {
            const float a0 = alpha[0], a1 = MODE == kRows16 ? alpha[RS - 1] : alpha[0];
#pragma unroll
            for (uint32_t i = 0; i < NB * 4; ++i) {
                o[i][0] *= a0;
                o[i][1] *= a0;
                o[i][2] *= a1;
                o[i][3] *= a1;
            }
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b) {
                wsum[b][0] *= a0;
                wsum[b][1] *= a1;
            }
        }
        const __half2 vs = __half2half2(__ushort_as_half(vexp < 30u ? (unsigned short)((30u - vexp) << 10) : (unsigned short)0x0200u));   // 2^(15 - vexp)
        uint32_t wa[4][NB][2];                                   // the weights' operand: rows 0..7, rows 8..15
#pragma unroll
        for (uint32_t nt = 0; nt < 4; ++nt) {
            const __half2 ph = __floats2half2_rn(s[0][2 * nt], s[0][2 * nt + 1]);
            __half2 pl;
            if (MODE == kRows8Split) {
                const float2 back = __half22float2(ph);
                pl = __floats2half2_rn(s[0][2 * nt] - back.x, s[0][2 * nt + 1] - back.y);
            } else if (MODE == kRows16) {
                pl = __floats2half2_rn(s[RS - 1][2 * nt], s[RS - 1][2 * nt + 1]);
            }
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b) {
                const __half2 d2 = __hmul2(dv[nt][b], vs);
                const __half2 h = __hmul2(ph, d2);
                wa[nt][b][0] = as_u32(h);
                if (MODE == kRows8Split) wa[nt][b][1] = as_u32(__hfma2(pl, d2, __hfma2(ph, d2, __hneg2(h))));
                else if (MODE == kRows16) wa[nt][b][1] = as_u32(__hmul2(pl, d2));
                else wa[nt][b][1] = 0u;
                if (MODE == kRows16 && !open) {
                    // the two rows of a lane may see different cells
                    const uint32_t k0 = seen[0] >> (2 * nt), k1 = seen[RS - 1] >> (2 * nt);
                    wa[nt][b][0] &= (k0 & 1u ? 0x0000FFFFu : 0u) | (k0 & 2u ? 0xFFFF0000u : 0u);
                    wa[nt][b][1] &= (k1 & 1u ? 0x0000FFFFu : 0u) | (k1 & 2u ? 0xFFFF0000u : 0u);
                }
            }
        }
#pragma unroll
        for (uint32_t ks = 0; ks < 2; ++ks) {
            const uint8_t* pv = sk + S::V_AT + 16u * ks * S::ROW + (g ^ ((t >> 1) * 4u)) * (S::ROW / 8);
            uint32_t v[4][2];
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                const uint8_t* p = pv + (8u * (j >> 1) + (j & 1u ? c_b : c_a)) * S::ROW;
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
                const uint32_t a0 = wa[2 * ks][b][0], a1 = wa[2 * ks][b][1], a2 = wa[2 * ks + 1][b][0], a3 = wa[2 * ks + 1][b][1];
                mma16816(o[4 * b], a0, a1, a2, a3, x0 & 0x000F000Fu, x1 & 0x000F000Fu);
                mma16816(o[4 * b + 1], a0, a1, a2, a3, x0 & 0x00F000F0u, x1 & 0x00F000F0u);
                mma16816(o[4 * b + 2], a0, a1, a2, a3, (x0 >> 8) & 0x000F000Fu, (x1 >> 8) & 0x000F000Fu);
                mma16816(o[4 * b + 3], a0, a1, a2, a3, (x0 >> 8) & 0x00F000F0u, (x1 >> 8) & 0x00F000F0u);
            }
        }
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b) {
            float c[4] = {};
            mma16816(c, wa[0][b][0], wa[0][b][1], wa[1][b][0], wa[1][b][1], 0x00080008u, 0x00080008u);
            mma16816(c, wa[2][b][0], wa[2][b][1], wa[3][b][0], wa[3][b][1], 0x00080008u, 0x00080008u);
            wsum[b][0] += c[0];
            wsum[b][1] += c[2];
        }
        stage = (stage + 1u) % S::STAGES;
        __syncwarp();                                            // the tile is read: its stage may be filled
    }
    cp_wait<0>();
    __syncwarp();

    // the warp's results in its ring: [R][W] outputs; 2^14 and 2^(15 - vexp) and 2^-24 (2^-20) are undone here
    float* wo = reinterpret_cast<float*>(ringp);
    const float unscale = __uint_as_float((127u + 24u + vexp - 15u) << 23);
#pragma unroll
    for (uint32_t b = 0; b < NB; ++b)
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            const float f = i & 1u ? unscale * 0.0625f : unscale, k = i & 1u ? 16.0f : 1.0f;
            const float* c = o[4 * b + i];
            const uint32_t d0 = 32u * b + 8u * t + i;             // columns 2t, 2t + 1: chunks 2t, 2t + 1
            if (MODE == kRows8Split) {
                const float ws = (wsum[b][0] + wsum[b][1]) * k;
                wo[g * S::W + d0] = ((c[0] + c[2]) - ws) * f;
                wo[g * S::W + d0 + 4] = ((c[1] + c[3]) - ws) * f;
            } else {
                wo[g * S::W + d0] = (c[0] - wsum[b][0] * k) * f;
                wo[g * S::W + d0 + 4] = (c[1] - wsum[b][0] * k) * f;
                if (MODE == kRows16) {
                    wo[(g + 8u) * S::W + d0] = (c[2] - wsum[b][1] * k) * f;
                    wo[(g + 8u) * S::W + d0 + 4] = (c[3] - wsum[b][1] * k) * f;
                }
            }
        }
#pragma unroll
    for (uint32_t r = 0; r < RS; ++r) {
        l[r] += __shfl_xor_sync(0xFFFFFFFFu, l[r], 1);
        l[r] += __shfl_xor_sync(0xFFFFFFFFu, l[r], 2);
        if (t == 0) {
            float* p = red + (warp * 16u + g + 8u * r) * 3u;
            p[0] = MASK ? off[r] : 0.0f;
            p[1] = m[r];
            p[2] = l[r];
        }
    }
    __syncthreads();
    // the CTA's teams, added in order; then the output, or the split's share of it
    for (uint32_t e = tid; e < R * D; e += kDecWarps * 32u) {
        const uint32_t r = e / D, d = e % D, row = rt * R + r;
        if (row >= rows) continue;
        float ot = -INFINITY, mt = -INFINITY, lt = 0.0f, acc = 0.0f;
#pragma unroll
        for (uint32_t j = 0; j < S::TEAMS; ++j) ot = fmaxf(ot, red[(j * S::NG * 16u + r) * 3u]);
        float sh[S::TEAMS];
#pragma unroll
        for (uint32_t j = 0; j < S::TEAMS; ++j) {
            const float* p = red + (j * S::NG * 16u + r) * 3u;
            sh[j] = p[1] == -INFINITY ? -INFINITY : MASK ? p[1] + (p[0] - ot) * 1.4426950408889634f : p[1];
            mt = fmaxf(mt, sh[j]);
        }
        const float base = mt == -INFINITY ? 0.0f : mt;
#pragma unroll
        for (uint32_t j = 0; j < S::TEAMS; ++j) {
            const float* p = red + (j * S::NG * 16u + r) * 3u;
            const float f = ex2(sh[j] - base);
            if (p[2] == 0.0f) continue;                          // a team that saw nothing of the row
            lt += f * p[2];
            acc += f * reinterpret_cast<const float*>(sm + (j * S::NG + d / S::W) * S::RING)[r * S::W + d % S::W];
        }
        if (a.splits == 1u) {
            const uint32_t tok = grp * a.group + row / a.G, h = hk * a.G + row % a.G;
            static_cast<T*>(a.out)[(size_t)tok * a.out_stride + (size_t)h * D + d] = from_f32<T>(lt == 0.0f ? 0.0f : acc / lt);
        } else {
            const size_t at = ((size_t)unit * a.splits + split) * R + r;
            a.part_o[at * D + d] = acc;
            if (d == 0) *reinterpret_cast<float4*>(a.part_ml + at * 4u) = make_float4(ot, mt, lt, 0.0f);
        }
    }
}

// Adds up the splits of each row in order. One CTA per row of a unit.
template <class T, int D, uint32_t R>
__global__ void __launch_bounds__(128) fa4_merge_kernel(Fa4Args a) {
    const uint32_t unit = blockIdx.x, r = blockIdx.y;
    const uint32_t hk = unit % a.n_head_kv, rt = unit / a.n_head_kv % a.row_tiles, grp = unit / (a.n_head_kv * a.row_tiles);
    const uint32_t row = rt * R + r;
    if (row >= a.group * a.G) return;
    const float4* ml = reinterpret_cast<const float4*>(a.part_ml) + (size_t)unit * a.splits * R + r;
    const float* po = a.part_o + ((size_t)unit * a.splits * R + r) * D;
    float ot = -INFINITY, mt = -INFINITY, lt = 0.0f;
    for (uint32_t s = 0; s < a.splits; ++s) ot = fmaxf(ot, ml[(size_t)s * R].x);
    for (uint32_t s = 0; s < a.splits; ++s) {
        const float4 p = ml[(size_t)s * R];
        if (p.y != -INFINITY) mt = fmaxf(mt, p.x == ot ? p.y : p.y + (p.x - ot) * 1.4426950408889634f);
    }
    const float base = mt == -INFINITY ? 0.0f : mt;
    constexpr uint32_t N = D / 128 ? D / 128 : 1;
    float acc[N] = {};
    for (uint32_t s = 0; s < a.splits; ++s) {
        const float4 p = ml[(size_t)s * R];
        if (p.z == 0.0f) continue;
        const float f = ex2((p.x == ot ? p.y : p.y + (p.x - ot) * 1.4426950408889634f) - base);
        lt += f * p.z;
#pragma unroll
        for (uint32_t k = 0; k < N; ++k)
            if (threadIdx.x + 128u * k < D) acc[k] += f * po[(size_t)s * R * D + threadIdx.x + 128u * k];
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
    uint32_t group, row_tiles, units, splits;
    size_t o_bytes, ml_bytes;
};

Fa4Plan fa4_plan(uint32_t type, uint32_t n_head_kv, uint32_t D, uint32_t T, uint32_t n_head, uint32_t n_kv, uint32_t group, uint32_t max_len) {
    Fa4Plan p{};
    p.group = group ? group : T;
    const uint32_t rows = p.group * (n_head / n_head_kv);
    p.mode = type != TSRC_TYPE_BF16 ? kRows8Split : rows <= 8u ? kRows8 : kRows16;
    const uint32_t R = p.mode == kRows16 ? 16u : 8u;
    p.row_tiles = (rows + R - 1u) / R;
    p.units = (T / p.group) * n_head_kv * p.row_tiles;
    const uint32_t len = max_len && max_len < n_kv ? max_len : n_kv;
    const uint32_t teams = D <= 128u ? kDecWarps : kDecWarps * 128u / D;
    // split until the CTAs fill the GPU once, each warp keeping at least two tiles
    const uint32_t most = (len / kDecTile + 1u + 2u * teams - 1u) / (2u * teams);
    p.splits = p.units ? kDecCtas / p.units : 1u;
    if (p.splits > most) p.splits = most;
    if (p.splits < 1u) p.splits = 1u;
    if (p.splits > 1u) {
        p.o_bytes = (size_t)p.units * p.splits * R * D * 4u;
        p.ml_bytes = (size_t)p.units * p.splits * R * 16u;
    }
    return p;
}

template <class T, int D, int MODE, bool MASK>
cudaError_t dec_launch_m(const Fa4Args& a, uint32_t units, cudaStream_t st) {
    constexpr uint32_t smem = dec_smem<D, MODE>();
    cudaError_t e = cudaFuncSetAttribute(fa4_dec_kernel<T, D, MODE, MASK>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    fa4_dec_kernel<T, D, MODE, MASK><<<dim3(units, a.splits), kDecWarps * 32, smem, st>>>(a);
    e = cudaGetLastError();
    if (e != cudaSuccess || a.splits == 1u) return e;
    fa4_merge_kernel<T, D, kRowsOf<MODE>><<<dim3(units, kRowsOf<MODE>), 128, 0, st>>>(a);
    return cudaGetLastError();
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

template <class... A>
int refuse(int code, const char* fmt, A... a) {
    char msg[256];
    snprintf(msg, sizeof msg, fmt, a...);
    return set_error(code, msg);
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
    if (T == 0 || tsrc_flash_attn_q4_unsupported(type, n_head_kv, head_dim, n_head)) return 0;
    const Fa4Plan p = fa4_plan(type, n_head_kv, head_dim, T, n_head, n_kv, group, max_len);
    return p.o_bytes + p.ml_bytes;
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
    if (T > (1u << 20)) return set_error(TSRC_E_SHAPE, "tsrc_flash_attn_q4: T above 2^20");
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
    const Fa4Plan p = fa4_plan(type, kv->n_head_kv, kv->D, T, n_head, n_kv, group, max_len);
    Fa4Args a{};
    a.q = q;
    a.out = out;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
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
    a.scale = scale;
    a.group = p.group;
    a.row_tiles = p.row_tiles;
    a.splits = p.splits;
    a.part_o = static_cast<float*>(ws);
    a.part_ml = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + p.o_bytes);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (type == TSRC_TYPE_F32) e = dec_launch_d<float, kRows8Split>(a, kv->D, p.units, st);
    else if (type == TSRC_TYPE_F16) e = dec_launch_d<__half, kRows8Split>(a, kv->D, p.units, st);
    else e = p.mode == kRows8 ? dec_launch_d<__nv_bfloat16, kRows8>(a, kv->D, p.units, st) : dec_launch_d<__nv_bfloat16, kRows16>(a, kv->D, p.units, st);
    if (e != cudaSuccess) return refuse(TSRC_E_CUDA, "tsrc_flash_attn_q4: %s (%s)", cudaGetErrorString(e), cudaGetErrorName(e));
    return TSRC_OK;
}

}  // extern "C"
