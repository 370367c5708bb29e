// tsrc_beam.cu -- one step of beam search: the best continuations over the beams and the vocabulary
// (tsrc_beam_select).
//
//   s[b][v] = score[b] + x[b][v] - log(sum_u exp(x[b][u]))
//
// Inside a beam s grows with x, so a beam's best are those of the raw logits, which compare exactly; only the few
// kept of each beam meet the other beams' in f64. Two kernels, the logits read once:
//   part   one CTA per 8192 logits of a row: maximum, sum of exponentials, and the part's n_out best in order;
//   merge  one CTA per group: a warp per beam merges its parts' ordered lists and adds up the normaliser, then one
//          warp merges the beams' lists.
// A candidate is one 64-bit key, the logit's bits made monotone above the complement of its index, so that equal
// logits go to the lowest index and no two keys are equal. Key 0 stands for none.
#include <cmath>
#include <cstdio>
#include <type_traits>

#include "tsrc_kv4.cuh"

namespace tsrc {

namespace {

constexpr uint32_t kBeamThreads = 256, kBeamEach = 32, kBeamPart = kBeamThreads * kBeamEach;
constexpr uint32_t kBeamOut = 64, kBeamBeams = 64, kBeamVocab = 1u << 20;
constexpr uint32_t kBeamCap = kBeamOut * kBeamEach;      // the list's room: what n_out threads can hold
constexpr size_t kBeamSmem = 220u * 1024u;

// parts of a row, with room for the up to seven values before it that its first 16 bytes may hold
__host__ __device__ inline uint32_t beam_parts(uint32_t n_vocab) { return (n_vocab + 7u + kBeamPart - 1u) / kBeamPart; }
constexpr uint32_t kBeamLists = (kBeamVocab + 7u + kBeamPart - 1u) / kBeamPart / 32u + 1u;    // parts that a lane merges

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

// A part is 8192 logits from a 16-byte boundary on (`lead` of the first part's lie before the row); a thread holds
// 32 of them in registers, as they came, for two passes: the largest, then the sum of exponentials and the few that
// can be among the part's best. Those few are what reaches a bound below the n_out-th best, the least of n_out
// maxima over disjoint sets of threads: about n_out (1 + 1/2 + ... + 1/n_out) of them where the large ones lie
// scattered. Where they do not (a sorted row) the list overflows, and the exact n_out-th largest of the threads'
// own best keys, found bit by bit, takes the bound's place: n_out threads hold all that reaches it.
// 256 rows of 128256 bf16 logits (65.7 MB): 82 us with scalar loads and a count before the list, 37 us as here.
template <class T>
__global__ void __launch_bounds__(kBeamThreads, sizeof(T) == 4 ? 4 : 6) beam_part_kernel(const T* __restrict__ logits, size_t stride, uint32_t n_vocab,
                                                                 uint32_t n_out, BeamPart* parts, unsigned long long* keys) {
    using V = BeamVec<T>;
    constexpr uint32_t NV = kBeamEach / V::N;
    __shared__ unsigned long long list[kBeamCap];
    __shared__ float redm[8], reds[8];
    __shared__ uint32_t least, count;
    asm volatile("griddepcontrol.launch_dependents;");
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    const size_t row = blockIdx.y, at = row * gridDim.x + blockIdx.x;
    const T* x = logits + row * stride;
    const uint32_t lead = (uint32_t)(reinterpret_cast<uintptr_t>(x) & 15u) / (uint32_t)sizeof(T);
    const int64_t first = (int64_t)blockIdx.x * kBeamPart - lead + tid * V::N;       // this thread's first logit
    V v[NV];
#pragma unroll
    for (uint32_t j = 0; j < NV; ++j) {
        const int64_t i = first + j * kBeamThreads * V::N;
        if (i >= 0 && i + V::N <= n_vocab) v[j].raw = __ldcs(reinterpret_cast<const uint4*>(x + i));
        else {                                                   // a row's ends
            T t[V::N];
#pragma unroll
            for (uint32_t k = 0; k < V::N; ++k) t[k] = i + k >= 0 && i + k < n_vocab ? x[i + k] : from_f32<T>(-INFINITY);
            __builtin_memcpy(&v[j].raw, t, 16);
        }
    }
    float m = -INFINITY, tops[NV];
#pragma unroll
    for (uint32_t j = 0; j < NV; ++j) {
        tops[j] = v[j].top();
        m = fmaxf(m, tops[j]);                                   // NaN only where all are
    }
    // the least of n_out maxima over sets of `width` threads (all keys of floats above -inf are above 0)
    const uint32_t mine = m > -INFINITY ? order_of(m) : 0u;
    uint32_t width = 1;
    while (width * 2u * n_out <= kBeamThreads && width < 32u) width *= 2u;
    uint32_t set = mine;
    for (uint32_t s = 1; s < width; s <<= 1) set = max(set, __shfl_xor_sync(0xFFFFFFFFu, set, s));
    const uint32_t low = __reduce_min_sync(0xFFFFFFFFu, tid / width < n_out ? set : 0xFFFFFFFFu);
    const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, mine);
    if (tid == 0) {
        least = 0xFFFFFFFFu;
        count = 0;
    }
    if (lane == 0) redm[warp] = top ? value_of(top) : -INFINITY;
    __syncthreads();
    if (lane == 0 && low != 0xFFFFFFFFu) atomicMin(&least, low);
    float most = redm[0];
#pragma unroll
    for (int w = 1; w < 8; ++w) most = fmaxf(most, redm[w]);
    __syncthreads();
    const float bound = least ? value_of(least) : -3.4028234e38f;
    // exp(y - most) as 2^(y L - c) 2^(c - most L), c the rounded most L, L = log2 e in f32: one fused step a logit; the
    // second factor is near 1 while most is not far from 0
    constexpr float L = 1.4426950408889634f;
    const float shift = most > -INFINITY ? most : 0.0f;
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
#pragma unroll
    for (uint32_t j = 0; j < NV; ++j) {
        if (!(tops[j] >= bound)) continue;
        const uint32_t at0 = (uint32_t)(first + j * kBeamThreads * V::N);
#pragma unroll
        for (uint32_t k = 0; k < V::N; ++k) {
            const float y = v[j].at(k);
            if (y >= bound) {                                    // false for -inf and NaN
                const uint32_t n = atomicAdd(&count, 1u);
                if (n < kBeamCap) list[n] = key_of(y, at0 + k);
            }
        }
    }
    for (int s = 16; s; s >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, s);
    if (lane == 0) reds[warp] = sum;
    __syncthreads();
    if (count > kBeamCap) {
        unsigned long long best = 0, limit = 0;
#pragma unroll
        for (uint32_t j = 0; j < NV; ++j)
#pragma unroll
            for (uint32_t k = 0; k < V::N; ++k) {
                const unsigned long long key = key_of(v[j].at(k), (uint32_t)(first + j * kBeamThreads * V::N + k));
                best = key > best ? key : best;
            }
        for (int bit = 63; bit >= 0; --bit) {
            const unsigned long long trial = limit | (1ull << bit);
            if (__syncthreads_count(best >= trial) >= (int)n_out) limit = trial;
        }
        if (tid == 0) count = 0;
        __syncthreads();
#pragma unroll
        for (uint32_t j = 0; j < NV; ++j)
#pragma unroll
            for (uint32_t k = 0; k < V::N; ++k) {
                const unsigned long long key = key_of(v[j].at(k), (uint32_t)(first + j * kBeamThreads * V::N + k));
                if (key != 0 && key >= limit) list[atomicAdd(&count, 1u)] = key;
            }
        __syncthreads();
    }
    // the list's order by counting what is larger: few are in it as a rule
    const uint32_t n = count;
    unsigned long long* out = keys + at * n_out;
    for (uint32_t i = tid; i < n; i += kBeamThreads) {
        const unsigned long long k = list[i];
        uint32_t rank = 0;
        for (uint32_t j = 0; j < n; ++j) rank += list[j] > k ? 1u : 0u;
        if (rank < n_out) out[rank] = k;
    }
    for (uint32_t i = n + tid; i < n_out; i += kBeamThreads) out[i] = 0ull;
    if (tid == 0) {
        float total = 0.0f;
        for (int w = 0; w < 8; ++w) total += reds[w];
        parts[at] = BeamPart{most, total};
    }
}

__device__ __forceinline__ unsigned long long warp_max(unsigned long long k) {
    const uint32_t hi = __reduce_max_sync(0xFFFFFFFFu, (uint32_t)(k >> 32));
    const uint32_t lo = __reduce_max_sync(0xFFFFFFFFu, (uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
    return ((unsigned long long)hi << 32) | lo;
}

// One CTA per group; warp w takes beams w, w + warps, ...: it brings the beam's lists into shared memory, takes the
// best of the lists' heads n_out times, and has the normaliser summed in f64 meanwhile.
template <uint32_t LISTS>
__global__ void __launch_bounds__(512) beam_merge_kernel(const BeamPart* parts, const unsigned long long* keys, uint32_t n_parts,
                                                         const float* scores, uint32_t n_beam, uint32_t n_out, float* out_scores,
                                                         int32_t* out_beam, int32_t* out_token) {
    extern __shared__ unsigned long long sm[];
    unsigned long long* val = sm;                                        // [n_beam][n_out] f64 order of s
    uint32_t* tok = reinterpret_cast<uint32_t*>(sm + n_beam * n_out);    // [n_beam][n_out]
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    unsigned long long* mine = sm + (n_beam * n_out * 12u + 15u) / 16u * 2u + (size_t)warp * n_parts * n_out;
    const size_t group = blockIdx.x;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    for (uint32_t b = warp; b < n_beam; b += warps) {
        const size_t row = group * n_beam + b;
        const unsigned long long* kr = keys + row * n_parts * n_out;
        for (uint32_t i = lane; i < n_parts * n_out; i += 32u) mine[i] = kr[i];
        const BeamPart* pr = parts + row * n_parts;
        float top = -INFINITY;
        for (uint32_t i = lane; i < n_parts; i += 32u) top = fmaxf(top, pr[i].max);
        for (int s = 16; s; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, s));
        double sum = 0.0;
        for (uint32_t i = lane; i < n_parts; i += 32u)
            if (pr[i].sum != 0.0f) sum += (double)pr[i].sum * exp((double)pr[i].max - (double)top);
        for (int s = 16; s; s >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, s);
        const double norm = log(sum);                        // above top, so that logits far from 0 keep their digits
        const double score = scores ? (double)scores[row] : 0.0;
        __syncwarp();
        uint32_t at[LISTS];
        unsigned long long head[LISTS];
#pragma unroll
        for (uint32_t j = 0; j < LISTS; ++j) {
            at[j] = (lane + 32u * j) * n_out;
            head[j] = lane + 32u * j < n_parts ? mine[at[j]] : 0ull;
        }
        for (uint32_t k = 0; k < n_out; ++k) {
            unsigned long long best = 0;
#pragma unroll
            for (uint32_t j = 0; j < LISTS; ++j) best = head[j] > best ? head[j] : best;
            best = warp_max(best);
#pragma unroll
            for (uint32_t j = 0; j < LISTS; ++j)
                if (best != 0 && head[j] == best) head[j] = ++at[j] < (lane + 32u * j + 1u) * n_out ? mine[at[j]] : 0ull;
            if (lane == 0) {
                val[b * n_out + k] = best;
                tok[b * n_out + k] = ~(uint32_t)best;
            }
        }
        __syncwarp();
        for (uint32_t k = lane; k < n_out; k += 32u) {
            const unsigned long long best = val[b * n_out + k];
            const double s = score + (((double)value_of((uint32_t)(best >> 32)) - (double)top) - norm);
            val[b * n_out + k] = best != 0 && s > -INFINITY ? order_of(s == 0.0 ? 0.0 : s) : 0ull;      // NaN: none
        }
    }
    __syncthreads();
    if (warp) return;
    uint32_t at[2] = {0, 0};
    unsigned long long h[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) h[j] = lane + 32u * j < n_beam ? val[(lane + 32u * j) * n_out] : 0ull;
    for (uint32_t k = 0; k < n_out; ++k) {
        const unsigned long long best = warp_max(h[1] > h[0] ? h[1] : h[0]);
        // equal scores: the lowest beam
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
            h[j] = at[j] < n_out ? val[b * n_out + at[j]] : 0ull;
        }
    }
}

size_t beam_parts_bytes(uint32_t rows, uint32_t n_vocab) { return ((size_t)rows * beam_parts(n_vocab) * sizeof(BeamPart) + 255u) & ~(size_t)255u; }

template <class T>
void launch_part(const void* x, size_t stride, uint32_t rows, uint32_t n_vocab, uint32_t n_out, BeamPart* parts, unsigned long long* keys, cudaStream_t st) {
    beam_part_kernel<T><<<dim3(beam_parts(n_vocab), rows), kBeamThreads, 0, st>>>(static_cast<const T*>(x), stride, n_vocab, n_out, parts, keys);
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
    return beam_parts_bytes((uint32_t)rows, n_vocab) + rows * beam_parts(n_vocab) * n_out * 8u;
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
    const uint32_t rows = n_group * n_beam, n_parts = beam_parts(n_vocab);
    BeamPart* parts = static_cast<BeamPart*>(ws);
    unsigned long long* keys = reinterpret_cast<unsigned long long*>(static_cast<uint8_t*>(ws) + beam_parts_bytes(rows, n_vocab));
    if (type == TSRC_TYPE_F32) launch_part<float>(logits, stride, rows, n_vocab, n_out, parts, keys, st);
    else if (type == TSRC_TYPE_F16) launch_part<__half>(logits, stride, rows, n_vocab, n_out, parts, keys, st);
    else launch_part<__nv_bfloat16>(logits, stride, rows, n_vocab, n_out, parts, keys, st);
    cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) {
        // as many warps as beams, up to sixteen and to the shared memory that their lists take
        const size_t fixed = (size_t)(n_beam * n_out * 12u + 15u) / 16u * 16u, each = (size_t)n_parts * n_out * 8u;
        uint32_t warps = n_beam < 16u ? n_beam : 16u;
        while (warps > 1u && fixed + warps * each > kBeamSmem) --warps;
        const auto kernel = n_parts <= 32u ? beam_merge_kernel<1> : beam_merge_kernel<kBeamLists>;
        static bool done[64];
        int dev = 0;
        e = cudaGetDevice(&dev);
        if (e == cudaSuccess && (dev >= 64 || !done[dev])) {
            e = cudaFuncSetAttribute(beam_merge_kernel<1>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kBeamSmem);
            if (e == cudaSuccess) e = cudaFuncSetAttribute(beam_merge_kernel<kBeamLists>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kBeamSmem);
            if (e == cudaSuccess && dev < 64) done[dev] = true;
        }
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(n_group);
        cfg.blockDim = dim3(warps * 32u);
        cfg.dynamicSmemBytes = fixed + warps * each;
        cfg.stream = st;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        if (e == cudaSuccess)
            e = cudaLaunchKernelEx(&cfg, kernel, static_cast<const BeamPart*>(parts), static_cast<const unsigned long long*>(keys), n_parts,
                                   scores, n_beam, n_out, out_scores, out_beam, out_token);
    }
    if (e != cudaSuccess) return refuse(TSRC_E_CUDA, "tsrc_beam_select: %s (%s)", cudaGetErrorString(e), cudaGetErrorName(e));
    return TSRC_OK;
}

}  // extern "C"
