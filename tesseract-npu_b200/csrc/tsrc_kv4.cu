// tsrc_kv4.cu -- the q4_0 KV cache: storing rows (quantizing them), reading them back, the ggml image, and beam
// search's reordering, with the cache's C ABI entry points. Layout: tsrc_kv4.cuh.
#include <new>

#include "tsrc_kv4.cuh"

namespace tsrc {

namespace {

__device__ unsigned int g_kv4_error;

// Plane geometry of a launch.
struct Kv4Planes {
    uint8_t* q[2];
    __half* d[2];
    uint32_t n_head_kv, D, n_cells, n_alloc;
};

Kv4Planes planes_of(const tsrc_kv4* kv) {
    Kv4Planes p{};
    for (int w = 0; w < 2; ++w) {
        p.q[w] = kv->q[w];
        p.d[w] = kv->d[w];
    }
    p.n_head_kv = kv->n_head_kv;
    p.D = kv->D;
    p.n_cells = kv->n_cells;
    p.n_alloc = kv->n_alloc;
    return p;
}

// The unit of storing and reading is a lane t of four that share NB blocks (NB = 4 for a 128-value group, 2 where
// D = 64): values 8t .. 8t + 7 of each, the two neighbouring chunks 2t and 2t + 1 of the codes. The four lanes read
// or write whole 64 / 128-byte lines of the rows and 16 (8) bytes of codes each.
struct Kv4Unit {
    uint32_t head, group, t;    // group: of NB * 32 values inside the head
    uint32_t value;             // the unit's first value in the row of E, + 32 b for block b
};

template <uint32_t NB>
__device__ __forceinline__ Kv4Unit unit_of(uint32_t u, uint32_t D) {
    Kv4Unit r;
    const uint32_t per_head = D / (NB * 32u);
    r.t = u & 3u;
    const uint32_t grp = u >> 2;
    r.head = grp / per_head;
    r.group = grp - r.head * per_head;
    r.value = grp * NB * 32u + 8u * r.t;
    return r;
}

__device__ __forceinline__ int64_t cell_of(const int64_t* cells, uint32_t cell0, uint32_t i) {
    return cells ? cells[i] : (int64_t)cell0 + i;
}

// Where chunks 2t and 2t + 1 of a group lie, in bytes from the group's row (kv4_place keeps such pairs together).
template <uint32_t NB>
__device__ __forceinline__ uint32_t pair_at(uint32_t t, size_t cell) { return kv4_place(2u * t, cell) * (NB * 2u); }

// The codes of eight values of a block by the format's own steps, whatever they are (zeros, NaN, infinities, scales
// below f32's normal numbers, largest values of either sign): every lane of the warp comes here together.
__device__ __forceinline__ void kv4_block_any(const float (&x)[8], uint32_t& lo, uint32_t& hi, float& d) {
    const uint32_t lane = threadIdx.x & 31u;
    uint32_t mag[8], top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        mag[j] = __float_as_uint(x[j]) & 0x7FFFFFFFu;
        if (mag[j] > 0x7F800000u) mag[j] = 0u;                   // a NaN does not count
        top = max(top, mag[j]);
    }
    top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
    top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
    uint32_t sign = 0;
    bool has = false;
#pragma unroll
    for (int j = 7; j >= 0; --j)
        if (mag[j] == top && x[j] == x[j]) {
            has = true;
            sign = __float_as_uint(x[j]) & 0x80000000u;
        }
    const uint32_t first = __ffs((__ballot_sync(0xFFFFFFFFu, has) >> (lane & 28u)) & 0xFu);
    sign = __shfl_sync(0xFFFFFFFFu, sign, (lane & 28u) | ((first - 1u) & 3u));
    d = (top ? __uint_as_float(top | sign) : 0.0f) * -0.125f;
    const float id = d != 0.0f ? __frcp_rn(d) : 0.0f;
    lo = hi = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float z = __fadd_rn(__fmul_rn(x[j], id), 8.5f);
        const uint32_t c = z == z ? (uint32_t)fminf(fmaxf(z, 0.0f), 15.0f) : 8u;
        if (j < 4) lo |= c << (4 * j);
        else hi |= c << (4 * (j - 4));
    }
}

// max and min that keep a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Four codes z = x id + 8.5 (0.5 <= z < 17) cut to 0..15: z + 2^23 rounded down has the code in its last bits, and
// four such words, weighted 1, 16, 256, 4096, add up to the 16 bits and a constant.
__device__ __forceinline__ uint32_t pack4(const float* x, float id) {
    uint32_t acc = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float z = fminf(__fadd_rn(__fmul_rn(x[j], id), 8.5f), 15.5f);
        acc += __float_as_uint(__fadd_rd(z, 8388608.0f)) << (4 * j);
    }
    return acc - 0x4B000000u * 0x1111u;
}

// Rows -> blocks. The block's first value of largest magnitude is its maximum or its minimum, so two maxima over
// the eight values and two shuffles each find it; where they tie in magnitude (the first decides), or the block
// has no ordinary scale, the warp takes the general steps.
// 8192 rows of 1024 bf16 values, K and V (33.6 MB in, 9.4 out): 24.8 us with eight lanes a block, magnitudes and
// signs by value and 64-bit divisions; 13.7 us so.
template <class T, uint32_t NB, bool VEC>
__global__ void __launch_bounds__(256) kv4_store_kernel(const T* __restrict__ k, const T* __restrict__ v, uint32_t n, size_t row_stride,
                                                        const int64_t* cells, uint32_t cell0, Kv4Planes p) {
    const uint32_t per_row = p.n_head_kv * p.D / (NB * 8u);
    const uint32_t t = blockIdx.x * blockDim.x + threadIdx.x;
    const uint32_t i0 = t / per_row;
    const bool live = i0 < n;                                   // whole groups of four lanes live or not
    const uint32_t i = live ? i0 : n - 1u;
    const uint32_t which = blockIdx.y + (k ? 0u : 1u);
    const Kv4Unit u = unit_of<NB>(t - i0 * per_row, p.D);
    const int64_t cell = cell_of(cells, cell0, i);
    const bool inside = cell >= 0 && cell < (int64_t)p.n_cells;
    const T* row = (which ? v : k) + (size_t)i * row_stride + u.value;
    float x[NB][8];
#pragma unroll
    for (uint32_t b = 0; b < NB; ++b) load8<T, VEC>(row + 32u * b, x[b]);
    uint32_t lo[NB], hi[NB];
    float d[NB];
#pragma unroll
    for (uint32_t b = 0; b < NB; ++b) {
        float up = x[b][0], down = x[b][0];
#pragma unroll
        for (int j = 1; j < 8; ++j) {
            up = max_nan(up, x[b][j]);
            down = min_nan(down, x[b][j]);
        }
#pragma unroll
        for (int s = 1; s < 4; s <<= 1) {
            up = max_nan(up, __shfl_xor_sync(0xFFFFFFFFu, up, s));
            down = min_nan(down, __shfl_xor_sync(0xFFFFFFFFu, down, s));
        }
        const float big = fabsf(up) > fabsf(down) ? up : down;
        const bool plain = up + down != 0.0f && fabsf(big) >= 1e-30f && fabsf(big) < INFINITY;       // false for NaN
        d[b] = big * -0.125f;                                   // m / -8: a power of two
        if (__all_sync(0xFFFFFFFFu, plain)) {
            const float id = __frcp_rn(d[b]);
            lo[b] = pack4(x[b], id);
            hi[b] = pack4(x[b] + 4, id);
        } else
            kv4_block_any(x[b], lo[b], hi[b], d[b]);
    }
    if (!live) return;
    if (!inside) {
        if (u.value == 0) atomicOr(&g_kv4_error, kKv4ErrSet);
        return;
    }
    const size_t hc = (size_t)u.head * p.n_alloc + (size_t)cell;
    uint8_t* q = p.q[which] + hc * (p.D / 2u) + u.group * (NB * 16u) + pair_at<NB>(u.t, (size_t)cell);
    if constexpr (NB == 4)
        *reinterpret_cast<uint4*>(q) = make_uint4(lo[0] | (lo[1] << 16), lo[2] | (lo[3] << 16), hi[0] | (hi[1] << 16), hi[2] | (hi[3] << 16));
    else *reinterpret_cast<uint2*>(q) = make_uint2(lo[0] | (lo[1] << 16), hi[0] | (hi[1] << 16));
    if (u.t < NB) {
        float db = d[0];
#pragma unroll
        for (uint32_t b = 1; b < NB; ++b)
            if (u.t == b) db = d[b];
        p.d[which][hc * (p.D / 32u) + u.group * NB + u.t] = __float2half_rn(db);
    }
}

// Blocks -> rows. n - 8 comes from fp16 arithmetic without rounding (n + 1024 is an fp16 whose last bits are n).
// d (n - 8) has at most 15 significant bits: the f32 product is exact, and so is an fp16 product before its one
// rounding.
// 131072 cells of 1024 values to fp16, K and V (151 MB in, 537 out): 181 us with eight lanes a group, 128 us so (5.4 TB/s).
template <class T, uint32_t NB, bool VEC>
__global__ void __launch_bounds__(256) kv4_read_kernel(T* __restrict__ k, T* __restrict__ v, uint32_t n, size_t row_stride,
                                                       const int64_t* cells, uint32_t cell0, Kv4Planes p) {
    const uint32_t per_row = p.n_head_kv * p.D / (NB * 8u);
    const uint32_t t = blockIdx.x * blockDim.x + threadIdx.x;
    const uint32_t i = t / per_row;
    if (i >= n) return;
    const uint32_t which = blockIdx.y + (k ? 0u : 1u);
    const Kv4Unit u = unit_of<NB>(t - i * per_row, p.D);
    const int64_t cell = cell_of(cells, cell0, i);
    if (cell < 0 || cell >= (int64_t)p.n_cells) {
        if (u.value == 0) atomicOr(&g_kv4_error, kKv4ErrGet);
        return;
    }
    const size_t hc = (size_t)u.head * p.n_alloc + (size_t)cell;
    const uint8_t* q = p.q[which] + hc * (p.D / 2u) + u.group * (NB * 16u) + pair_at<NB>(u.t, (size_t)cell);
    const __half* ds = p.d[which] + hc * (p.D / 32u) + u.group * NB;
    uint32_t w[NB], s[NB / 2];                                  // w: two blocks' values 8t .. + 3, then 8t + 4 .. + 7
    if constexpr (NB == 4) {
        const uint4 a = __ldcs(reinterpret_cast<const uint4*>(q));
        const uint2 c = *reinterpret_cast<const uint2*>(ds);
        w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
        s[0] = c.x; s[1] = c.y;
    } else {
        const uint2 a = __ldcs(reinterpret_cast<const uint2*>(q));
        w[0] = a.x; w[1] = a.y;
        s[0] = *reinterpret_cast<const uint32_t*>(ds);
    }
    T* row = (which ? v : k) + (size_t)i * row_stride + u.value;
#pragma unroll
    for (uint32_t b = 0; b < NB; ++b) {
        // the block's halves side by side: codes i and i + 4 of the eight in the two halves of a word
        const uint32_t c = __byte_perm(w[b / 2], w[NB / 2 + b / 2], b & 1u ? 0x7632 : 0x5410);
        const __half d = __ushort_as_half((unsigned short)(s[b / 2] >> (16u * (b & 1u))));
        __half2 x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t bits = ((c >> (4 * j)) & 0x000F000Fu) | 0x64006400u;
            x[j] = __hsub2(*reinterpret_cast<const __half2*>(&bits), __float2half2_rn(1032.0f));
        }
        store8<T, VEC>(row + 32u * b, x, d);
    }
}

// ggml q4_0 rows <-> planes, one thread per block. A block is 18 bytes, so its address is even.
__global__ void kv4_from_ggml_kernel(const uint8_t* ggml, uint32_t n, uint32_t cell0, uint32_t which, Kv4Planes p) {
    const uint32_t nb = p.n_head_kv * p.D / 32u, NB = p.D == 64u ? 2u : 4u;
    const size_t t = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (t >= (size_t)n * nb) return;
    const uint32_t i = (uint32_t)(t / nb), blk = (uint32_t)(t - (size_t)i * nb);
    const uint32_t head = 32u * blk / p.D, b = blk - head * (p.D / 32u);
    const uint8_t* src = ggml + t * 18u;
    const size_t hc = (size_t)head * p.n_alloc + cell0 + i;
    p.d[which][hc * (p.D / 32u) + b] = __ushort_as_half((unsigned short)(src[0] | (src[1] << 8)));
    uint8_t* row = p.q[which] + hc * (p.D / 2u) + (b / NB) * (NB * 16u) + (b % NB) * 2u;
    for (uint32_t g = 0; g < 8; ++g) {
        uint32_t c = 0;
        for (uint32_t j = 0; j < 4; ++j) {
            const uint32_t e = 4u * g + j;
            c |= (e < 16u ? src[2 + e] & 15u : src[2 + e - 16u] >> 4) << (4u * j);
        }
        *reinterpret_cast<uint16_t*>(row + kv4_place(g, (size_t)cell0 + i) * NB * 2u) = (uint16_t)c;
    }
}

__global__ void kv4_to_ggml_kernel(uint8_t* ggml, uint32_t n, uint32_t cell0, uint32_t which, Kv4Planes p) {
    const uint32_t nb = p.n_head_kv * p.D / 32u, NB = p.D == 64u ? 2u : 4u;
    const size_t t = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (t >= (size_t)n * nb) return;
    const uint32_t i = (uint32_t)(t / nb), blk = (uint32_t)(t - (size_t)i * nb);
    const uint32_t head = 32u * blk / p.D, b = blk - head * (p.D / 32u);
    uint8_t* dst = ggml + t * 18u;
    const size_t hc = (size_t)head * p.n_alloc + cell0 + i;
    const uint32_t d = __half_as_ushort(p.d[which][hc * (p.D / 32u) + b]);
    dst[0] = (uint8_t)d;
    dst[1] = (uint8_t)(d >> 8);
    const uint8_t* row = p.q[which] + hc * (p.D / 2u) + (b / NB) * (NB * 16u) + (b % NB) * 2u;
    for (uint32_t g = 0; g < 4; ++g) {
        const uint32_t lo = *reinterpret_cast<const uint16_t*>(row + kv4_place(g, (size_t)cell0 + i) * NB * 2u);
        const uint32_t hi = *reinterpret_cast<const uint16_t*>(row + kv4_place(g + 4u, (size_t)cell0 + i) * NB * 2u);
        for (uint32_t j = 0; j < 4; ++j)
            dst[2 + 4u * g + j] = (uint8_t)(((lo >> (4u * j)) & 15u) | (((hi >> (4u * j)) & 15u) << 4));
    }
}

// Reordering in place: the same thread owns the same values of every sequence of a group, reads those that move
// and then writes them, so no copy overtakes another. U: the unit of bytes (16 for codes; the scales of a cell
// need not be 16-byte aligned where a sequence starts). swap: the bit of a unit's index that the chunks' places
// flip (kv4_place) where the cell has its bit 2 set: half a group's units for codes, 0 for scales.
template <class U, uint32_t NBEAM>
__device__ __forceinline__ void reorder_unit(U* plane, size_t j, uint32_t units_cell, uint32_t swap, const int32_t* par, uint32_t n_beam,
                                             size_t first, uint32_t seq_stride) {
    const uint32_t i = (uint32_t)(j / units_cell), unit = (uint32_t)(j - (size_t)i * units_cell);
    auto at = [&](uint32_t s) {
        const size_t cell = first + i + (size_t)s * seq_stride;
        return plane + cell * units_cell + (unit ^ ((cell & 4u) ? swap : 0u));
    };
    U w[NBEAM];
#pragma unroll
    for (uint32_t s = 0; s < NBEAM; ++s) {
        if (s >= n_beam) break;
        const int32_t from = par[s];
        if (from >= 0 && from < (int32_t)n_beam && from != (int32_t)s) w[s] = *at((uint32_t)from);
        else if ((from < -1 || from >= (int32_t)n_beam) && j == 0) atomicOr(&g_kv4_error, kKv4ErrParent);
    }
#pragma unroll
    for (uint32_t s = 0; s < NBEAM; ++s) {
        if (s >= n_beam) break;
        const int32_t from = par[s];
        if (from >= 0 && from < (int32_t)n_beam && from != (int32_t)s) *at(s) = w[s];
    }
}

// The first code_blocks CTAs of x take codes, the others scales. What is kept is neither read nor written.
template <uint32_t NBEAM, class DU>
__global__ void __launch_bounds__(256) kv4_reorder_kernel(Kv4Planes p, uint32_t code_blocks, const int32_t* parent, uint32_t n_beam,
                                                          uint32_t cell0, uint32_t seq_stride, uint32_t n) {
    const uint32_t group = blockIdx.y, head = blockIdx.z >> 1, which = blockIdx.z & 1u;
    const int32_t* par = parent + (size_t)group * n_beam;
    const size_t first = (size_t)cell0 + (size_t)group * n_beam * seq_stride;
    if (blockIdx.x < code_blocks) {
        const uint32_t per = p.D / 32u;
        const size_t j = (size_t)blockIdx.x * 256u + threadIdx.x;
        if (j >= (size_t)n * per) return;
        reorder_unit<uint4, NBEAM>(reinterpret_cast<uint4*>(p.q[which]) + (size_t)head * p.n_alloc * per, j, per, p.D == 64u ? 1u : 2u,
                                   par, n_beam, first, seq_stride);
    } else {
        const uint32_t per = p.D / 16u / (uint32_t)sizeof(DU);
        const size_t j = (size_t)(blockIdx.x - code_blocks) * 256u + threadIdx.x;
        if (j >= (size_t)n * per) return;
        reorder_unit<DU, NBEAM>(reinterpret_cast<DU*>(p.d[which]) + (size_t)head * p.n_alloc * per, j, per, 0u, par, n_beam, first, seq_stride);
    }
}

template <class DU>
cudaError_t launch_reorder(const Kv4Planes& p, const int32_t* parent, uint32_t n_group, uint32_t n_beam, uint32_t cell0, uint32_t seq_stride,
                           uint32_t n, cudaStream_t st) {
    const size_t codes = ((size_t)n * (p.D / 32u) + 255u) / 256u, scales = ((size_t)n * (p.D / 16u / sizeof(DU)) + 255u) / 256u;
    const dim3 grid((unsigned)(codes + scales), n_group, 2u * p.n_head_kv);
    if (n_beam <= 8u) kv4_reorder_kernel<8, DU><<<grid, 256, 0, st>>>(p, (uint32_t)codes, parent, n_beam, cell0, seq_stride, n);
    else kv4_reorder_kernel<32, DU><<<grid, 256, 0, st>>>(p, (uint32_t)codes, parent, n_beam, cell0, seq_stride, n);
    return cudaGetLastError();
}

template <class T, uint32_t NB, bool VEC>
void launch_store(const T* k, const T* v, uint32_t n, size_t stride, const int64_t* cells, uint32_t cell0, const Kv4Planes& p, cudaStream_t st) {
    const size_t threads = (size_t)n * (p.n_head_kv * p.D / (NB * 8u));
    kv4_store_kernel<T, NB, VEC><<<dim3((unsigned)((threads + 255u) / 256u), k && v ? 2u : 1u), 256, 0, st>>>(k, v, n, stride, cells, cell0, p);
}
template <class T, uint32_t NB, bool VEC>
void launch_read(T* k, T* v, uint32_t n, size_t stride, const int64_t* cells, uint32_t cell0, const Kv4Planes& p, cudaStream_t st) {
    const size_t threads = (size_t)n * (p.n_head_kv * p.D / (NB * 8u));
    kv4_read_kernel<T, NB, VEC><<<dim3((unsigned)((threads + 255u) / 256u), k && v ? 2u : 1u), 256, 0, st>>>(k, v, n, stride, cells, cell0, p);
}

// The variant by D, and by alignment: eight values at once where rows and stride allow 16-byte accesses.
template <class T>
cudaError_t rows_io(bool store, void* k, void* v, uint32_t n, size_t stride, const int64_t* cells, uint32_t cell0, const Kv4Planes& p, cudaStream_t st) {
    const bool vec = ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15u) == 0 && stride * sizeof(T) % 16u == 0;
    T *kt = static_cast<T*>(k), *vt = static_cast<T*>(v);
    if (p.D == 64u) {
        if (store) vec ? launch_store<T, 2, true>(kt, vt, n, stride, cells, cell0, p, st) : launch_store<T, 2, false>(kt, vt, n, stride, cells, cell0, p, st);
        else vec ? launch_read<T, 2, true>(kt, vt, n, stride, cells, cell0, p, st) : launch_read<T, 2, false>(kt, vt, n, stride, cells, cell0, p, st);
    } else {
        if (store) vec ? launch_store<T, 4, true>(kt, vt, n, stride, cells, cell0, p, st) : launch_store<T, 4, false>(kt, vt, n, stride, cells, cell0, p, st);
        else vec ? launch_read<T, 4, true>(kt, vt, n, stride, cells, cell0, p, st) : launch_read<T, 4, false>(kt, vt, n, stride, cells, cell0, p, st);
    }
    return cudaGetLastError();
}

// set_rows and get_rows: the same checks and geometry.
int kv4_rows(const char* who, bool store, tsrc_ctx* ctx, const tsrc_kv4* kv, uint32_t type, void* k, void* v, uint32_t n,
             uint32_t row_stride, const int64_t* cells, uint32_t cell0, void* stream) {
    if (!ctx || !kv || (!k && !v)) return refuse(TSRC_E_ARG, "%s: NULL argument", who);
    if (kv->ctx != ctx) return refuse(TSRC_E_ARG, "%s: the cache belongs to another context", who);
    if (!kv4_type_ok(type)) return refuse(TSRC_E_ARG, "%s: type %u is none of f32, f16, bf16", who, type);
    const uint32_t E = kv->n_head_kv * kv->D;
    if (row_stride == 0) row_stride = E;
    if (row_stride < E) return refuse(TSRC_E_ARG, "%s: row_stride %u < E %u", who, row_stride, E);
    if (!cells && (uint64_t)cell0 + n > kv->n_cells)
        return refuse(TSRC_E_ARG, "%s: cells [%u, %u+%u) outside the cache", who, cell0, cell0, n);
    const uintptr_t m = kv4_type_size(type) - 1u;
    if (((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & m) || (reinterpret_cast<uintptr_t>(cells) & 7u))
        return refuse(TSRC_E_ARG, "%s: a pointer is not aligned to its elements", who);
    if (n == 0) return TSRC_OK;
    if ((uint64_t)n * (E / 16u) > 0xFFFF0000ull) return refuse(TSRC_E_SHAPE, "%s: n %u: more than 2^32 / (E / 16) rows in a call", who, n);
    DeviceScope scope(ctx);
    if (scope.rc) return scope.rc;
    const Kv4Planes p = planes_of(kv);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (type == TSRC_TYPE_F32) e = rows_io<float>(store, k, v, n, row_stride, cells, cell0, p, st);
    else if (type == TSRC_TYPE_F16) e = rows_io<__half>(store, k, v, n, row_stride, cells, cell0, p, st);
    else e = rows_io<__nv_bfloat16>(store, k, v, n, row_stride, cells, cell0, p, st);
    return e == cudaSuccess ? TSRC_OK : cuda_refuse(e, who);
}

int kv4_bytes(const char* who, const tsrc_kv4* kv, uint32_t which, void* rows, uint32_t cell0, uint32_t n, bool store) {
    if (!kv || !rows) return refuse(TSRC_E_ARG, "%s: NULL argument", who);
    if (which > TSRC_KV_V) return refuse(TSRC_E_ARG, "%s: which must be TSRC_KV_K or TSRC_KV_V", who);
    if ((uint64_t)cell0 + n > kv->n_cells) return refuse(TSRC_E_ARG, "%s: cells [%u, %u+%u) outside the cache", who, cell0, cell0, n);
    if (n == 0) return TSRC_OK;
    DeviceScope scope(kv->ctx);
    if (scope.rc) return scope.rc;
    const Kv4Planes p = planes_of(kv);
    // staged in parts, so that a large cache needs no copy of its own size beside it
    const size_t row = (size_t)(kv->n_head_kv * kv->D / 32u) * 18u;
    const uint32_t part = (uint32_t)(n < 1u + (64u << 20) / row ? n : 1u + (64u << 20) / row);
    uint8_t* stage = nullptr;
    cudaError_t e = cudaMalloc(&stage, part * row);
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        return refuse(TSRC_E_NOMEM, "%s: cudaMalloc of %zu staging bytes: %s", who, part * row, cudaGetErrorString(e));
    }
    e = cudaDeviceSynchronize();
    for (uint32_t at = 0; at < n && e == cudaSuccess; at += part) {
        const uint32_t m = n - at < part ? n - at : part;
        uint8_t* host = static_cast<uint8_t*>(rows) + at * row;
        const size_t threads = (size_t)m * (p.n_head_kv * p.D / 32u);
        const unsigned grid = (unsigned)((threads + 255u) / 256u);
        if (store) {
            e = cudaMemcpy(stage, host, m * row, cudaMemcpyDefault);
            if (e == cudaSuccess) kv4_from_ggml_kernel<<<grid, 256>>>(stage, m, cell0 + at, which, p);
        } else
            kv4_to_ggml_kernel<<<grid, 256>>>(stage, m, cell0 + at, which, p);
        if (e == cudaSuccess) e = cudaGetLastError();
        if (e == cudaSuccess && !store) e = cudaMemcpy(host, stage, m * row, cudaMemcpyDefault);
        if (e == cudaSuccess) e = cudaDeviceSynchronize();
    }
    cudaFree(stage);
    return e == cudaSuccess ? TSRC_OK : cuda_refuse(e, who);
}

}  // namespace

void kv4_drop(tsrc_kv4* kv) {
    if (!kv) return;
    cudaFree(kv->mem);
    ctx_remove_kv4(kv->ctx, kv);
    delete kv;
}

cudaError_t kv4_error(uint32_t* code, bool clear) {
    cudaError_t e = cudaMemcpyFromSymbol(code, g_kv4_error, sizeof(uint32_t));
    if (e == cudaSuccess && clear && *code) {
        const uint32_t zero = 0;
        e = cudaMemcpyToSymbol(g_kv4_error, &zero, sizeof(uint32_t));
    }
    return e;
}

}  // namespace tsrc

using namespace tsrc;

extern "C" {

int tsrc_kv4_create(tsrc_ctx* ctx, uint32_t n_head_kv, uint32_t head_dim, uint32_t n_cells, tsrc_kv4** out) {
    if (!ctx || !out) return set_error(TSRC_E_ARG, "tsrc_kv4_create: NULL argument");
    *out = nullptr;
    if (!kv4_geometry_ok(n_head_kv, head_dim)) return set_error(TSRC_E_SHAPE, "tsrc_kv4_create: head_dim must be 64/128/256/512, E / 64 <= 511");
    if (n_cells == 0 || n_cells > (1u << 30)) return set_error(TSRC_E_SHAPE, "tsrc_kv4_create: n_cells must be 1..2^30");
    DeviceScope scope(ctx);
    if (scope.rc) return scope.rc;
    const uint32_t n_alloc = (n_cells + kKv4Pad - 1u) / kKv4Pad * kKv4Pad;
    const size_t qb = (size_t)n_head_kv * n_alloc * (head_dim / 2u), db = (size_t)n_head_kv * n_alloc * (head_dim / 32u) * 2u;
    tsrc_kv4* kv = new (std::nothrow) tsrc_kv4{};
    if (!kv) return set_error(TSRC_E_NOMEM, "tsrc_kv4_create: out of host memory");
    cudaError_t e = cudaMalloc(&kv->mem, 2u * (qb + db));
    if (e != cudaSuccess) {
        delete kv;
        (void)cudaGetLastError();
        return refuse(TSRC_E_NOMEM, "tsrc_kv4_create: cudaMalloc of %zu bytes: %s", 2u * (qb + db), cudaGetErrorString(e));
    }
    e = cudaMemset(kv->mem, 0, 2u * (qb + db));
    if (e == cudaSuccess) e = cudaDeviceSynchronize();       // the zeros are there for every stream
    try {
        if (e == cudaSuccess) ctx_add_kv4(ctx, kv);
    } catch (...) {
        e = cudaErrorMemoryAllocation;
    }
    if (e != cudaSuccess) {
        cudaFree(kv->mem);
        delete kv;
        return cuda_refuse(e, "tsrc_kv4_create");
    }
    kv->ctx = ctx;
    kv->n_head_kv = n_head_kv;
    kv->D = head_dim;
    kv->n_cells = n_cells;
    kv->n_alloc = n_alloc;
    for (int w = 0; w < 2; ++w) {
        kv->q[w] = kv->mem + (size_t)w * qb;
        kv->d[w] = reinterpret_cast<__half*>(kv->mem + 2u * qb + (size_t)w * db);
    }
    *out = kv;
    return TSRC_OK;
}

int tsrc_kv4_free(tsrc_kv4* kv) {
    if (!kv) return set_error(TSRC_E_ARG, "tsrc_kv4_free: NULL cache");
    DeviceScope scope(kv->ctx);
    cudaDeviceSynchronize();
    kv4_drop(kv);
    return TSRC_OK;
}

int tsrc_kv4_set_rows(tsrc_ctx* ctx, tsrc_kv4* kv, uint32_t type, const void* k, const void* v, uint32_t n, uint32_t row_stride,
                      const int64_t* cells, uint32_t cell0, void* stream) {
    return kv4_rows("tsrc_kv4_set_rows", true, ctx, kv, type, const_cast<void*>(k), const_cast<void*>(v), n, row_stride, cells, cell0, stream);
}

int tsrc_kv4_get_rows(tsrc_ctx* ctx, const tsrc_kv4* kv, uint32_t type, void* k, void* v, uint32_t n, uint32_t row_stride,
                      const int64_t* cells, uint32_t cell0, void* stream) {
    return kv4_rows("tsrc_kv4_get_rows", false, ctx, kv, type, k, v, n, row_stride, cells, cell0, stream);
}

int tsrc_kv4_set_bytes(tsrc_kv4* kv, uint32_t which, const void* ggml_rows, uint32_t cell0, uint32_t n) {
    return kv4_bytes("tsrc_kv4_set_bytes", kv, which, const_cast<void*>(ggml_rows), cell0, n, true);
}

int tsrc_kv4_get_bytes(const tsrc_kv4* kv, uint32_t which, void* ggml_rows, uint32_t cell0, uint32_t n) {
    return kv4_bytes("tsrc_kv4_get_bytes", kv, which, ggml_rows, cell0, n, false);
}

int tsrc_kv4_reorder(tsrc_ctx* ctx, tsrc_kv4* kv, const int32_t* parent, uint32_t n_group, uint32_t n_beam, uint32_t cell0,
                     uint32_t seq_stride, uint32_t n, void* stream) {
    if (!ctx || !kv || !parent) return set_error(TSRC_E_ARG, "tsrc_kv4_reorder: NULL argument");
    if (kv->ctx != ctx) return set_error(TSRC_E_ARG, "tsrc_kv4_reorder: the cache belongs to another context");
    if (reinterpret_cast<uintptr_t>(parent) & 3u) return set_error(TSRC_E_ARG, "tsrc_kv4_reorder: parent is not aligned to its elements");
    if (n_beam < 1u || n_beam > 32u) return refuse(TSRC_E_SHAPE, "tsrc_kv4_reorder: n_beam %u is not in 1..32", n_beam);
    if (n_group > 65535u) return refuse(TSRC_E_SHAPE, "tsrc_kv4_reorder: n_group %u above 65535", n_group);
    if (n_group == 0 || n == 0) return TSRC_OK;
    if (seq_stride < n) return refuse(TSRC_E_ARG, "tsrc_kv4_reorder: seq_stride %u < n %u", seq_stride, n);
    if ((uint64_t)cell0 + ((uint64_t)n_group * n_beam - 1u) * seq_stride + n > kv->n_cells)
        return set_error(TSRC_E_ARG, "tsrc_kv4_reorder: a sequence runs past the cache");
    DeviceScope scope(ctx);
    if (scope.rc) return scope.rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const Kv4Planes p = planes_of(kv);
    cudaError_t e = kv->D == 64u ? launch_reorder<uint32_t>(p, parent, n_group, n_beam, cell0, seq_stride, n, st)
                                 : launch_reorder<uint2>(p, parent, n_group, n_beam, cell0, seq_stride, n, st);
    return e == cudaSuccess ? TSRC_OK : cuda_refuse(e, "tsrc_kv4_reorder");
}

}  // extern "C"
