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

#include "tsrc_kv4.cuh"

namespace tsrc {

namespace {

constexpr uint32_t kBeamThreads = 256, kBeamEach = 32, kBeamPart = kBeamThreads * kBeamEach;
constexpr uint32_t kBeamOut = 64, kBeamBeams = 64, kBeamVocab = 1u << 20;
constexpr uint32_t kBeamCap = kBeamOut * kBeamEach;

__host__ __device__ inline uint32_t beam_parts(uint32_t n_vocab) { return (n_vocab + kBeamPart - 1u) / kBeamPart; }

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

__device__ __forceinline__ unsigned long long key_of(float x, uint32_t index) {
    if (!(x > -INFINITY)) return 0ull;
    if (x == 0.0f) x = 0.0f;                              // -0 and +0 are equal
    return ((unsigned long long)order_of(x) << 32) | (uint32_t)~index;
}

template <class T>
__global__ void __launch_bounds__(kBeamThreads) beam_part_kernel(const T* __restrict__ logits, size_t stride, uint32_t n_vocab,
                                                                 uint32_t n_out, BeamPart* parts, unsigned long long* keys) {
    __shared__ unsigned long long list[kBeamCap];
    __shared__ float redm[8], reds[8];
    __shared__ uint32_t least, count;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    const size_t row = blockIdx.y, at = row * gridDim.x + blockIdx.x;
    const T* x = logits + row * stride;
    const uint32_t first = blockIdx.x * kBeamPart;
    float v[kBeamEach];
#pragma unroll
    for (uint32_t j = 0; j < kBeamEach; ++j) {
        const uint32_t i = first + j * kBeamThreads + tid;
        v[j] = i < n_vocab ? to_f32(x[i]) : -INFINITY;
    }
    float m = v[0];
#pragma unroll
    for (uint32_t j = 1; j < kBeamEach; ++j) m = fmaxf(m, v[j]);
    const uint32_t mine = m > -INFINITY ? order_of(m) : 0u;
    float top = m;
    for (int s = 16; s; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, s));
    if (lane == 0) redm[warp] = top;
    if (tid == 0) {
        least = 0xFFFFFFFFu;
        count = 0;
    }
    __syncthreads();
    top = redm[0];
#pragma unroll
    for (int w = 1; w < 8; ++w) top = fmaxf(top, redm[w]);
    const float safe = top > -INFINITY ? top : 0.0f;      // a part of -inf and NaN: 0
    float sum = 0.0f;
#pragma unroll
    for (uint32_t j = 0; j < kBeamEach; ++j) sum += __expf(v[j] - safe);
    for (int s = 16; s; s >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, s);
    if (lane == 0) reds[warp] = sum;
    // A bound below the n_out-th best: the least of n_out maxima over disjoint sets of threads.
    uint32_t width = 1;
    while (width * 2u * n_out <= kBeamThreads && width < 32u) width *= 2u;
    uint32_t bound = mine;
    for (uint32_t s = 1; s < width; s <<= 1) bound = max(bound, __shfl_xor_sync(0xFFFFFFFFu, bound, s));
    if (tid / width < n_out && tid % width == 0) atomicMin(&least, bound);
    __syncthreads();
    bound = least;
    // exactly n_out threads could hold everything above it: then the list would hold at most n_out * kBeamEach, but
    // a set's maximum says nothing of how many lie above the least, so the count is checked first
    uint32_t above = 0;
#pragma unroll
    for (uint32_t j = 0; j < kBeamEach; ++j) above += v[j] > -INFINITY && order_of(v[j]) >= bound ? 1u : 0u;
    if (above) atomicAdd(&count, above);
    __syncthreads();
    const bool fits = count <= kBeamCap;
    unsigned long long limit = (unsigned long long)bound << 32;
    __syncthreads();
    if (!fits) {
        // the n_out-th largest of the threads' best keys, bit by bit: n_out threads hold all that is above it
        unsigned long long best = 0;
#pragma unroll
        for (uint32_t j = 0; j < kBeamEach; ++j) {
            const unsigned long long k = key_of(v[j], first + j * kBeamThreads + tid);
            best = k > best ? k : best;
        }
        limit = 0;
        for (int bit = 63; bit >= 0; --bit) {
            const unsigned long long trial = limit | (1ull << bit);
            if (__syncthreads_count(best >= trial) >= (int)n_out) limit = trial;
        }
    }
    if (tid == 0) count = 0;
    __syncthreads();
#pragma unroll
    for (uint32_t j = 0; j < kBeamEach; ++j) {
        const unsigned long long k = key_of(v[j], first + j * kBeamThreads + tid);
        if (k != 0 && k >= limit) list[atomicAdd(&count, 1u)] = k;
    }
    __syncthreads();
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
        parts[at] = BeamPart{top, total};
    }
}

__device__ __forceinline__ unsigned long long warp_max(unsigned long long k) {
    const uint32_t hi = __reduce_max_sync(0xFFFFFFFFu, (uint32_t)(k >> 32));
    const uint32_t lo = __reduce_max_sync(0xFFFFFFFFu, (uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
    return ((unsigned long long)hi << 32) | lo;
}

// One CTA per group; warp w takes beams w, w + warps, ... Lists are read where they lie (they were just written).
__global__ void __launch_bounds__(512) beam_merge_kernel(const BeamPart* parts, const unsigned long long* keys, uint32_t n_parts,
                                                         const float* scores, uint32_t n_beam, uint32_t n_out, float* out_scores,
                                                         int32_t* out_beam, int32_t* out_token) {
    extern __shared__ unsigned long long sm[];
    unsigned long long* val = sm;                                        // [n_beam][n_out] f64 order of s
    uint32_t* tok = reinterpret_cast<uint32_t*>(sm + n_beam * n_out);    // [n_beam][n_out]
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const size_t group = blockIdx.x;
    for (uint32_t b = warp; b < n_beam; b += warps) {
        const size_t row = group * n_beam + b;
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
        const unsigned long long* kr = keys + row * n_parts * n_out;
        uint32_t at[kBeamVocab / kBeamPart / 32u] = {};
        unsigned long long head[kBeamVocab / kBeamPart / 32u];
#pragma unroll
        for (uint32_t j = 0; j < kBeamVocab / kBeamPart / 32u; ++j) head[j] = lane + 32u * j < n_parts ? kr[(size_t)(lane + 32u * j) * n_out] : 0ull;
        for (uint32_t k = 0; k < n_out; ++k) {
            unsigned long long best = 0;
#pragma unroll
            for (uint32_t j = 0; j < kBeamVocab / kBeamPart / 32u; ++j) best = head[j] > best ? head[j] : best;
            best = warp_max(best);
#pragma unroll
            for (uint32_t j = 0; j < kBeamVocab / kBeamPart / 32u; ++j)
                if (best != 0 && head[j] == best) head[j] = ++at[j] < n_out ? kr[(size_t)(lane + 32u * j) * n_out + at[j]] : 0ull;
            if (lane == 0) {
                const double s = score + (((double)value_of((uint32_t)(best >> 32)) - (double)top) - norm);
                const bool any = best != 0 && s > -INFINITY;             // false for NaN
                val[b * n_out + k] = any ? order_of(s == 0.0 ? 0.0 : s) : 0ull;
                tok[b * n_out + k] = ~(uint32_t)best;
            }
        }
    }
    __syncthreads();
    if (warp) return;
    uint32_t at[2] = {0, 0};
    for (uint32_t k = 0; k < n_out; ++k) {
        unsigned long long h[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t b = lane + 32u * j;
            h[j] = b < n_beam && at[j] < n_out ? val[b * n_out + at[j]] : 0ull;
        }
        const unsigned long long best = warp_max(h[1] > h[0] ? h[1] : h[0]);
        // equal scores: the lowest beam
        const uint32_t who = h[0] == best ? lane : h[1] == best ? lane + 32u : 0xFFFFFFFFu;
        const uint32_t b = __reduce_min_sync(0xFFFFFFFFu, who);
        const size_t o = group * n_out + k;
        if (best == 0) {
            if (lane == 0) {
                out_scores[o] = -INFINITY;
                out_beam[o] = -1;
                out_token[o] = -1;
            }
            continue;
        }
        if ((b & 31u) == lane) {
            const uint32_t j = b >> 5;
            out_scores[o] = (float)value_of(best);
            out_beam[o] = (int32_t)b;
            out_token[o] = (int32_t)tok[b * n_out + at[j]];
            ++at[j];
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
        const uint32_t warps = n_beam < 16u ? n_beam : 16u;
        beam_merge_kernel<<<n_group, warps * 32u, (size_t)n_beam * n_out * 12u, st>>>(parts, keys, n_parts, scores, n_beam, n_out, out_scores, out_beam, out_token);
        e = cudaGetLastError();
    }
    if (e != cudaSuccess) return refuse(TSRC_E_CUDA, "tsrc_beam_select: %s (%s)", cudaGetErrorString(e), cudaGetErrorName(e));
    return TSRC_OK;
}

}  // extern "C"
