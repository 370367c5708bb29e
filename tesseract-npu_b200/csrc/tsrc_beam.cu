// tsrc_beam.cu -- one step of beam search: the best continuations over the beams and the vocabulary
// (tsrc_beam_select).
//
//   s[b][v] = score[b] + x[b][v] - log(sum_u exp(x[b][u]))
//
// Inside a beam s grows with x, so a beam's best are those of the raw logits, which compare exactly; only the few
// kept of each beam meet the other beams' in f64. Two kernels, the logits read once:
//   part    one CTA per 8192 logits of a row: maximum and sum of exponentials, and the largest of every 32 neighbours;
//   select  a cluster per group, a CTA per row (or several): the n_out groups of neighbours with the largest maxima
//           hold the row's n_out best -- each has one that beats whatever the others hold -- and their few logits are
//           read again; then the cluster's first CTA merges the rows' ordered lists.
// A candidate is one 64-bit key, the logit's bits made monotone above the complement of its index, so that equal
// logits go to the lowest index and no two keys are equal. Key 0 stands for none.
#include <cmath>
#include <type_traits>

#include "tsrc_kv4.cuh"

namespace tsrc {

namespace {

constexpr uint32_t kBeamThreads = 256, kBeamEach = 32, kBeamPart = kBeamThreads * kBeamEach;
constexpr uint32_t kBeamOut = 64, kBeamBeams = 64, kBeamVocab = 1u << 20;
constexpr uint32_t kBeamCap = kBeamOut * kBeamEach;      // a list's room: what n_out threads can hold
constexpr uint32_t kBeamLists = kBeamVocab / kBeamPart / 32u;    // parts that a lane adds up
constexpr uint32_t kBeamRows = 8;                        // rows that a cluster takes at once

__host__ __device__ inline uint32_t beam_parts(uint32_t n_vocab) { return (n_vocab + kBeamPart - 1u) / kBeamPart; }

// Neighbours that a maximum stands for in the first selection, as a power of two: 32, and 64 or 128 in the largest
// vocabularies, whose maxima would be more than a CTA holds.
__host__ __device__ constexpr uint32_t beam_fold(uint32_t n_parts) {
    uint32_t fold = 0;
    while (n_parts * kBeamThreads >> fold > kBeamPart) ++fold;
    return fold;
}
// the second selection holds the neighbours of n_out of them
static_assert(kBeamOut << (5u + beam_fold(kBeamVocab / kBeamPart)) <= kBeamPart, "room for the largest vocabulary");

struct BeamPart {
    float max, sum;      // sum of exp(x - max) over the part (-inf and 0 where the part is all -inf)
};

// unsigned order of floats; -inf and NaN below everything that can be chosen
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t u = __float_as_uint(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o); }
__device__ __forceinline__ unsigned long long order_of(double x) {
    const unsigned long long u = (unsigned long long)__double_as_longlong(x);
    return u >> 63 ? ~u : u | (1ull << 63);
}
__device__ __forceinline__ double value_of(unsigned long long o) {
    return __longlong_as_double((long long)(o >> 63 ? o ^ (1ull << 63) : ~o));
}

__device__ __forceinline__ float beam_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ unsigned long long key_of(float x, uint32_t index) {
    if (!(x > -INFINITY)) return 0ull;
    if (x == 0.0f) x = 0.0f;                              // -0 and +0 are equal
    return ((unsigned long long)order_of(x) << 32) | (uint32_t)~index;
}

__device__ __forceinline__ __half low_of(__half2 h) { return __low2half(h); }
__device__ __forceinline__ __half high_of(__half2 h) { return __high2half(h); }
__device__ __forceinline__ __nv_bfloat16 low_of(__nv_bfloat162 h) { return __low2bfloat16(h); }
__device__ __forceinline__ __nv_bfloat16 high_of(__nv_bfloat162 h) { return __high2bfloat16(h); }

// 16 bytes of logits, as values
template <class T> struct BeamVec {
    static constexpr uint32_t N = 16 / sizeof(T);
    uint4 raw;
    __device__ __forceinline__ float at(uint32_t i) const {
        const uint32_t w = i * sizeof(T) / 4u == 0u ? raw.x : i * sizeof(T) / 4u == 1u ? raw.y : i * sizeof(T) / 4u == 2u ? raw.z : raw.w;
        if constexpr (sizeof(T) == 4) return __uint_as_float(w);
        else if constexpr (std::is_same_v<T, __nv_bfloat16>) return __uint_as_float(i & 1u ? w & 0xFFFF0000u : w << 16);
        else return __half2float(__ushort_as_half((unsigned short)(i & 1u ? w >> 16 : w)));
    }
    // the largest of them, NaN passed over
    __device__ __forceinline__ float top() const {
        if constexpr (sizeof(T) == 4) return fmaxf(fmaxf(at(0), at(1)), fmaxf(at(2), at(3)));
        else {
            using H2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
            const H2 a = *reinterpret_cast<const H2*>(&raw.x), b = *reinterpret_cast<const H2*>(&raw.y);
            const H2 c = *reinterpret_cast<const H2*>(&raw.z), d = *reinterpret_cast<const H2*>(&raw.w);
            const H2 m = __hmax2(__hmax2(a, b), __hmax2(c, d));
            return fmaxf(to_f32(low_of(m)), to_f32(high_of(m)));
        }
    }
};

// The 16 bytes that begin `bytes` (2 .. 14, the same for the whole CTA) into 32.
__device__ __forceinline__ uint4 shifted(const uint4& lo, const uint4& hi, uint32_t bytes) {
    uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    if (bytes & 8u) {
#pragma unroll
        for (int k = 0; k < 6; ++k) w[k] = w[k + 2];
    }
    if (bytes & 4u) {
#pragma unroll
        for (int k = 0; k < 5; ++k) w[k] = w[k + 1];
    }
    const uint32_t bits = 8u * (bytes & 3u);
    return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits), __funnelshift_r(w[2], w[3], bits),
                      __funnelshift_r(w[3], w[4], bits));
}

// A part is 8192 logits counted from the row's own start, a warp's share 1024 neighbours, so 32 neighbours are 4 (f32: 8)
// lanes of one load. Where the row starts off a 16-byte boundary (`lead` values behind one) a thread's 16 bytes are cut from
// two aligned loads: which values are added up together, and in which order, does not depend on the row's address, so that
// alike rows get the same normaliser to the last bit and their candidates tie.
// Each thread adds up its 32 exponentials against its own largest, without waiting for anyone.
// 256 rows of 128256 bf16 logits (65.7 MB): 82 us with scalar loads and the best chosen in every part, 37 us with wide
// loads, 14.7 us so (4.5 TB/s). Rows off a boundary: 256 of 50257 fp16 logits, both kernels, 38 us (36 with parts
// cut by address).
template <class T>
__global__ void __launch_bounds__(kBeamThreads) beam_part_kernel(const T* __restrict__ logits, size_t stride, uint32_t n_vocab, BeamPart* parts,
                                                                 float* maxima) {
    using V = BeamVec<T>;
    constexpr uint32_t NV = kBeamEach / V::N, LANES = 32 / V::N;
    __shared__ float redm[8], reds[8];
    asm volatile("griddepcontrol.launch_dependents;");
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    const size_t row = blockIdx.y, at = row * gridDim.x + blockIdx.x;
    const T* x = logits + row * stride;
    const uint32_t lead = (uint32_t)(reinterpret_cast<uintptr_t>(x) & 15u) / (uint32_t)sizeof(T);
    const uint32_t first = blockIdx.x * kBeamPart + (warp * NV * 32u + lane) * V::N;
    V v[NV];
    auto ends = [&](uint32_t i) {                                // a row's ends
        T t[V::N];
#pragma unroll
        for (uint32_t k = 0; k < V::N; ++k) t[k] = i + k < n_vocab ? x[i + k] : from_f32<T>(-INFINITY);
        uint4 r;
        __builtin_memcpy(&r, t, 16);
        return r;
    };
    if (lead == 0) {
#pragma unroll
        for (uint32_t j = 0; j < NV; ++j) {
            const uint32_t i = first + j * 32u * V::N;
            v[j].raw = i + V::N <= n_vocab ? __ldcs(reinterpret_cast<const uint4*>(x + i)) : ends(i);
        }
    } else {
#pragma unroll
        for (uint32_t j0 = 0; j0 < NV; j0 += 4) {                // four loads under way together, in the row whatever the place
            uint4 lo[4], hi[4];
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                const uint32_t i = first + (j0 + j) * 32u * V::N;
                lo[j] = hi[j] = make_uint4(0, 0, 0, 0);
                if (i >= lead && i - lead + 2u * V::N <= n_vocab) {
                    const uint4* p = reinterpret_cast<const uint4*>(x + i - lead);
                    lo[j] = p[0];
                    hi[j] = p[1];
                }
            }
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                const uint32_t i = first + (j0 + j) * 32u * V::N;
                v[j0 + j].raw = i >= lead && i - lead + 2u * V::N <= n_vocab ? shifted(lo[j], hi[j], lead * (uint32_t)sizeof(T)) : ends(i);
            }
        }
    }
    float m = -INFINITY;
#pragma unroll
    for (uint32_t j = 0; j < NV; ++j) {
        float top = v[j].top();
        m = fmaxf(m, top);                                       // NaN is passed over
#pragma unroll
        for (uint32_t s = 1; s < LANES; s <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, s));
        if (lane % LANES == 0) maxima[at * kBeamThreads + warp * 32u + j * (32u / LANES) + lane / LANES] = top > -INFINITY ? top : -INFINITY;
    }
    // exp(y - m) as 2^(y L - c) 2^(c - m L), c the rounded m L, L = log2 e in f32: one fused step a logit; the second
    // factor is near 1 while m is not far from 0
    constexpr float L = 1.4426950408889634f;
    const float shift = m > -INFINITY ? m : 0.0f;
    float sum = 0.0f;
    if (fabsf(shift) < 4096.0f) {
        const float c = shift * -L;
#pragma unroll
        for (uint32_t j = 0; j < NV; ++j)
#pragma unroll
            for (uint32_t k = 0; k < V::N; ++k) sum += beam_ex2(fmaf(v[j].at(k), L, c));
        sum *= beam_ex2(-fmaf(shift, L, c));
    } else {
#pragma unroll
        for (uint32_t j = 0; j < NV; ++j)
#pragma unroll
            for (uint32_t k = 0; k < V::N; ++k) sum += beam_ex2((v[j].at(k) - shift) * L);
    }
    float top = m;
#pragma unroll
    for (int s = 16; s; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, s));
    if (sum != 0.0f) sum *= beam_ex2((shift - (top > -INFINITY ? top : 0.0f)) * L);
#pragma unroll
    for (int s = 16; s; s >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, s);
    if (lane == 0) {
        redm[warp] = top;
        reds[warp] = sum;
    }
    __syncthreads();
    if (tid == 0) {
        float most = redm[0], total = 0.0f;
        for (int w = 1; w < 8; ++w) most = fmaxf(most, redm[w]);
        for (int w = 0; w < 8; ++w)
            if (reds[w] != 0.0f) total += reds[w] * beam_ex2((redm[w] - (most > -INFINITY ? most : 0.0f)) * L);
        parts[at] = BeamPart{most, total};
    }
}

__device__ __forceinline__ unsigned long long warp_max(unsigned long long k) {
    const uint32_t hi = __reduce_max_sync(0xFFFFFFFFu, (uint32_t)(k >> 32));
    const uint32_t lo = __reduce_max_sync(0xFFFFFFFFu, (uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
    return ((unsigned long long)hi << 32) | lo;
}

struct SelectShared {
    unsigned long long list[kBeamCap], best[kBeamOut];   // candidates; the chosen, in order
    uint32_t least, count;
};

// A bound below the n_out-th largest of the values that the CTA's threads hold, m being this thread's largest: the least
// of n_out maxima over disjoint sets of threads. About n_out (1 + 1/2 + ... + 1/n_out) values reach it where the large
// ones lie scattered.
__device__ __forceinline__ float select_bound(SelectShared& s, float m, uint32_t n_out) {
    const uint32_t tid = threadIdx.x;
    uint32_t width = 1;
    while (width * 2u * n_out <= kBeamThreads && width < 32u) width *= 2u;
    uint32_t set = m > -INFINITY ? order_of(m) : 0u;
    for (uint32_t x = 1; x < width; x <<= 1) set = max(set, __shfl_xor_sync(0xFFFFFFFFu, set, x));
    const uint32_t low = __reduce_min_sync(0xFFFFFFFFu, tid / width < n_out ? set : 0xFFFFFFFFu);
    if (tid == 0) s.least = 0xFFFFFFFFu;
    __syncthreads();
    if ((tid & 31u) == 0 && low != 0xFFFFFFFFu) atomicMin(&s.least, low);
    __syncthreads();
    return s.least ? value_of(s.least) : -3.4028234e38f;
}

// The n_out largest of up to 8192 values, all of which reach `bound`, into s.best in order (0 where there are fewer);
// value j of this thread is candidate `index(j)`. What reaches the bound is listed, and the order comes from counting
// what is larger. Where the list overflows (sorted values, ties) the exact n_out-th largest of the threads' own best
// keys, found bit by bit, takes the bound's place: n_out threads hold all that reaches it.
template <class I>
__device__ __forceinline__ void select_best(SelectShared& s, const float (&v)[kBeamEach], uint32_t used, float bound, uint32_t n_out, const I& index) {
    const uint32_t tid = threadIdx.x;
    uint32_t mine = 0;
#pragma unroll
    for (uint32_t j = 0; j < kBeamEach; ++j) mine += j < used && v[j] >= bound ? 1u : 0u;        // false for -inf and NaN
    if (tid == 0) s.count = 0;
    __syncthreads();
    if (mine) {
        uint32_t n = atomicAdd(&s.count, mine);
#pragma unroll
        for (uint32_t j = 0; j < kBeamEach; ++j)
            if (j < used && v[j] >= bound) {
                if (n < kBeamCap) s.list[n] = key_of(v[j], index(j));
                ++n;
            }
    }
    __syncthreads();
    if (s.count > kBeamCap) {
        unsigned long long best = 0, limit = 0;
#pragma unroll
        for (uint32_t j = 0; j < kBeamEach; ++j) {
            const unsigned long long key = j < used ? key_of(v[j], index(j)) : 0ull;
            best = key > best ? key : best;
        }
#pragma unroll 1
        for (int bit = 63; bit >= 0; --bit) {
            const unsigned long long trial = limit | (1ull << bit);
            if (__syncthreads_count(best >= trial) >= (int)n_out) limit = trial;
        }
        if (tid == 0) s.count = 0;
        __syncthreads();
#pragma unroll
        for (uint32_t j = 0; j < kBeamEach; ++j) {
            const unsigned long long key = j < used ? key_of(v[j], index(j)) : 0ull;
            if (key != 0 && key >= limit) s.list[atomicAdd(&s.count, 1u)] = key;
        }
        __syncthreads();
    }
    const uint32_t n = s.count;
    for (uint32_t i = tid; i < n; i += kBeamThreads) {
        const unsigned long long k = s.list[i];
        uint32_t rank = 0;
        for (uint32_t j = 0; j < n; ++j) rank += s.list[j] > k ? 1u : 0u;
        if (rank < n_out) s.best[rank] = k;
    }
    for (uint32_t i = n + tid; i < n_out; i += kBeamThreads) s.best[i] = 0ull;
    __syncthreads();
}

template <class T>
__global__ void __launch_bounds__(kBeamThreads, 3) beam_select_kernel(const T* __restrict__ logits, size_t stride, uint32_t n_vocab, const BeamPart* parts,
                                                                   const float* maxima, uint32_t n_parts, const float* scores, uint32_t n_beam,
                                                                   uint32_t n_out, float* out_scores, int32_t* out_beam, int32_t* out_token) {
    extern __shared__ unsigned long long lists[];        // in the cluster's first CTA: [n_beam][n_out] f64 order of s, then tokens
    __shared__ SelectShared s;
    __shared__ double norm;
    __shared__ float top;
    uint32_t rank, size;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(size));
    const uint32_t tid = threadIdx.x, lane = tid & 31u;
    const size_t group = blockIdx.x / size;
    // every CTA of the cluster has begun before one writes into the first one's shared memory
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    for (uint32_t b = rank; b < n_beam; b += size) {
        const size_t row = group * n_beam + b;
        const T* x = logits + row * stride;
        const float* mx = maxima + row * n_parts * kBeamThreads;
        const uint32_t fold = beam_fold(n_parts);
        const uint32_t n_groups = (n_parts * kBeamThreads + (1u << fold) - 1u) >> fold;
        float v[kBeamEach];
#pragma unroll
        for (uint32_t j = 0; j < kBeamEach; ++j) {       // all loads together
            const uint32_t i = j * kBeamThreads + tid;
            v[j] = i < n_groups ? mx[i << fold] : -INFINITY;
        }
        for (uint32_t k = 1; k < 1u << fold; ++k)
#pragma unroll
            for (uint32_t j = 0; j < kBeamEach; ++j) {
                const uint32_t i = ((j * kBeamThreads + tid) << fold) + k;
                if (i < n_parts * kBeamThreads) v[j] = fmaxf(v[j], mx[i]);
            }
        if (tid < 32u) {                                 // the row's normaliser
            const BeamPart* pr = parts + row * n_parts;
            float mp[kBeamLists], p[kBeamLists], t = -INFINITY;
#pragma unroll
            for (uint32_t j = 0; j < kBeamLists; ++j) {
                const BeamPart q = lane + 32u * j < n_parts ? pr[lane + 32u * j] : BeamPart{-INFINITY, 0.0f};
                mp[j] = q.max;
                p[j] = q.sum;
                t = fmaxf(t, q.max);
            }
            for (int k = 16; k; k >>= 1) t = fmaxf(t, __shfl_xor_sync(0xFFFFFFFFu, t, k));
            double sum = 0.0;
#pragma unroll
            for (uint32_t j = 0; j < kBeamLists; ++j)
                if (p[j] != 0.0f) sum += (double)p[j] * (double)beam_ex2((mp[j] - t) * 1.4426950408889634f);
            for (int k = 16; k; k >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, k);
            if (lane == 0) {
                norm = log(sum);                         // above top, so that logits far from 0 keep their digits
                top = t;
            }
        }
        float m = v[0];
#pragma unroll
        for (uint32_t j = 1; j < kBeamEach; ++j) m = fmaxf(m, v[j]);
        select_best(s, v, (n_groups + kBeamThreads - 1u) / kBeamThreads, select_bound(s, m, n_out), n_out, [&](uint32_t j) { return j * kBeamThreads + tid; });
        // their logits: the last group's largest bounds the row's best
        const float least = s.best[n_out - 1u] ? value_of((uint32_t)(s.best[n_out - 1u] >> 32)) : -3.4028234e38f;
        const uint32_t shift = 5u + fold, n = n_out << shift;
        auto token = [&](uint32_t j) {                   // of this thread's logit j (s.best changes only when all have asked)
            const uint32_t e = j * kBeamThreads + tid;
            return (int32_t)(~(uint32_t)s.best[min(e >> shift, n_out - 1u)] << shift) + (int32_t)(e & ((1u << shift) - 1u));
        };
#pragma unroll
        for (uint32_t j = 0; j < kBeamEach; ++j) {
            v[j] = -INFINITY;
            if (j * kBeamThreads >= n) continue;
            const uint32_t e = j * kBeamThreads + tid;
            const int32_t i = token(j);
            if (e < n && s.best[min(e >> shift, n_out - 1u)] != 0 && i < (int32_t)n_vocab) v[j] = to_f32(x[i]);
        }
        select_best(s, v, (n + kBeamThreads - 1u) / kBeamThreads, least, n_out, [&](uint32_t j) { return (uint32_t)token(j); });
        for (uint32_t k = tid; k < n_out; k += kBeamThreads) {
            const unsigned long long key = s.best[k];
            const double score = scores ? (double)scores[row] : 0.0;
            const double z = score + (((double)value_of((uint32_t)(key >> 32)) - (double)top) - norm);
            const unsigned long long order = key != 0 && z > -INFINITY ? order_of(z == 0.0 ? 0.0 : z) : 0ull;      // NaN: none
            const uint32_t best = ~(uint32_t)key;
            uint32_t to = (uint32_t)__cvta_generic_to_shared(lists + b * n_out + k), far;
            asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(far) : "r"(to));
            asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(far), "l"(order) : "memory");
            to = (uint32_t)__cvta_generic_to_shared(reinterpret_cast<uint32_t*>(lists + n_beam * n_out) + b * n_out + k);
            asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(far) : "r"(to));
            asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(far), "r"(best) : "memory");
        }
        __syncthreads();
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (rank || tid >= 32u) return;
    // the rows' lists: the best of their heads, n_out times; equal scores: the lowest beam
    const uint32_t* tok = reinterpret_cast<const uint32_t*>(lists + n_beam * n_out);
    uint32_t at[2] = {0, 0};
    unsigned long long h[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) h[j] = lane + 32u * j < n_beam ? lists[(lane + 32u * j) * n_out] : 0ull;
    for (uint32_t k = 0; k < n_out; ++k) {
        const unsigned long long best = warp_max(h[1] > h[0] ? h[1] : h[0]);
        const uint32_t b = __reduce_min_sync(0xFFFFFFFFu, h[0] == best ? lane : h[1] == best ? lane + 32u : 0xFFFFFFFFu);
        const size_t o = group * n_out + k;
        if (best == 0) {
            if (lane == 0) {
                out_scores[o] = -INFINITY;
                out_beam[o] = -1;
                out_token[o] = -1;
            }
        } else if ((b & 31u) == lane) {
            const uint32_t j = b >> 5;
            out_scores[o] = (float)value_of(best);
            out_beam[o] = (int32_t)b;
            out_token[o] = (int32_t)tok[b * n_out + at[j]];
            ++at[j];
            h[j] = at[j] < n_out ? lists[b * n_out + at[j]] : 0ull;
        }
    }
}

size_t beam_parts_bytes(uint32_t rows, uint32_t n_vocab) { return ((size_t)rows * beam_parts(n_vocab) * sizeof(BeamPart) + 255u) & ~(size_t)255u; }

template <class T>
cudaError_t launch_beam(const void* logits, size_t stride, const float* scores, uint32_t n_group, uint32_t n_beam, uint32_t n_vocab, uint32_t n_out,
                        float* out_scores, int32_t* out_beam, int32_t* out_token, BeamPart* parts, float* maxima, cudaStream_t st) {
    const uint32_t n_parts = beam_parts(n_vocab), size = n_beam < kBeamRows ? n_beam : kBeamRows;
    const T* x = static_cast<const T*>(logits);
    beam_part_kernel<T><<<dim3(n_parts, n_group * n_beam), kBeamThreads, 0, st>>>(x, stride, n_vocab, parts, maxima);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    static bool done[64];
    int dev = 0;
    e = cudaGetDevice(&dev);
    if (e == cudaSuccess && (dev >= 64 || !done[dev])) {
        e = cudaFuncSetAttribute(beam_select_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(kBeamBeams * kBeamOut * 12u));
        if (e == cudaSuccess && dev < 64) done[dev] = true;
    }
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(n_group * size);
    cfg.blockDim = dim3(kBeamThreads);
    cfg.dynamicSmemBytes = (size_t)n_beam * n_out * 12u;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = size;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, beam_select_kernel<T>, x, stride, n_vocab, static_cast<const BeamPart*>(parts), static_cast<const float*>(maxima), n_parts,
                              scores, n_beam, n_out, out_scores, out_beam, out_token);
}

}  // namespace

}  // namespace tsrc

using namespace tsrc;

extern "C" {

const char* tsrc_beam_select_unsupported(uint32_t type, uint32_t n_beam, uint32_t n_vocab, uint32_t n_out) {
    if (!kv4_type_ok(type)) return "beam_select: logits must be f32, f16 or bf16";
    if (n_beam < 1u || n_beam > kBeamBeams) return "beam_select: n_beam is not in 1..64";
    if (n_vocab < 1u || n_vocab > kBeamVocab) return "beam_select: n_vocab is not in 1..2^20";
    if (n_out < 1u || n_out > kBeamOut) return "beam_select: n_out is not in 1..64";
    return nullptr;
}

size_t tsrc_beam_select_workspace(uint32_t n_group, uint32_t n_beam, uint32_t n_vocab, uint32_t n_out) {
    if (tsrc_beam_select_unsupported(TSRC_TYPE_F32, n_beam, n_vocab, n_out)) return 0;
    const size_t rows = (size_t)n_group * n_beam;
    return beam_parts_bytes((uint32_t)rows, n_vocab) + rows * beam_parts(n_vocab) * kBeamThreads * 4u;
}

int tsrc_beam_select(tsrc_ctx* ctx, uint32_t type, const void* logits, uint32_t stride, const float* scores, uint32_t n_group,
                     uint32_t n_beam, uint32_t n_vocab, uint32_t n_out, float* out_scores, int32_t* out_beam, int32_t* out_token,
                     void* ws, size_t ws_bytes, void* stream) {
    if (!ctx || !logits || !out_scores || !out_beam || !out_token) return set_error(TSRC_E_ARG, "tsrc_beam_select: NULL argument");
    if (const char* why = tsrc_beam_select_unsupported(type, n_beam, n_vocab, n_out)) return set_error(TSRC_E_SHAPE, why);
    if (stride == 0) stride = n_vocab;
    if (stride < n_vocab) return set_error(TSRC_E_ARG, "tsrc_beam_select: stride < n_vocab");
    if ((uint64_t)n_group * n_beam > 65535u) return set_error(TSRC_E_SHAPE, "tsrc_beam_select: more than 65535 rows");
    if ((reinterpret_cast<uintptr_t>(logits) & (kv4_type_size(type) - 1u)) ||
        ((reinterpret_cast<uintptr_t>(scores) | reinterpret_cast<uintptr_t>(out_scores) | reinterpret_cast<uintptr_t>(out_beam) |
          reinterpret_cast<uintptr_t>(out_token)) & 3u))
        return set_error(TSRC_E_ARG, "tsrc_beam_select: a pointer is not aligned to its elements");
    if (n_group == 0) return TSRC_OK;
    const size_t need = tsrc_beam_select_workspace(n_group, n_beam, n_vocab, n_out);
    if (!ws || ws_bytes < need || (reinterpret_cast<uintptr_t>(ws) & 255u))
        return refuse(TSRC_E_ARG, "tsrc_beam_select: the workspace must be 256-byte aligned and hold %zu bytes", need);
    DeviceScope scope(ctx);
    if (scope.rc) return scope.rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    BeamPart* parts = static_cast<BeamPart*>(ws);
    float* maxima = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + beam_parts_bytes(n_group * n_beam, n_vocab));
    cudaError_t e;
    if (type == TSRC_TYPE_F32) e = launch_beam<float>(logits, stride, scores, n_group, n_beam, n_vocab, n_out, out_scores, out_beam, out_token, parts, maxima, st);
    else if (type == TSRC_TYPE_F16) e = launch_beam<__half>(logits, stride, scores, n_group, n_beam, n_vocab, n_out, out_scores, out_beam, out_token, parts, maxima, st);
    else e = launch_beam<__nv_bfloat16>(logits, stride, scores, n_group, n_beam, n_vocab, n_out, out_scores, out_beam, out_token, parts, maxima, st);
    return e == cudaSuccess ? TSRC_OK : cuda_refuse(e, "tsrc_beam_select");
}

}  // extern "C"
