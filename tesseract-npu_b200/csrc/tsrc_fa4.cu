// tsrc_fa4.cu -- attention over the q4_0 KV cache (tsrc_flash_attn_q4). Cache layout: tsrc_kv4.cuh.
#include <cmath>
#include <cstdio>

#include "tsrc_kv4.cuh"

namespace tsrc {

namespace {

struct Fa4Args {
    const void* q;
    void* out;
    size_t q_stride, out_stride;
    const uint8_t *kq, *vq;
    const __half *kd, *vd;
    uint32_t T, n_head, n_head_kv, D, n_kv, n_alloc;
    const int32_t* ranges;
    const __half* mask;
    size_t mask_stride;
    float scale;
};

// value e of a code row (head dimension D)
__device__ __forceinline__ float fa4_value(const uint8_t* q, const __half* d, uint32_t D, uint32_t e) {
    const uint32_t NB = D == 64u ? 2u : 4u, b = e / 32u, w = e % 32u;
    const uint32_t half = *reinterpret_cast<const uint16_t*>(q + (b / NB) * (NB * 16u) + (w / 4u) * (NB * 2u) + (b % NB) * 2u);
    return __half2float(d[b]) * (float)((int)((half >> (4u * (w % 4u))) & 15u) - 8);
}

// One CTA of 128 threads per (token, head), 128 cells at a time: a thread scores one cell, then the threads share
// the head's values among them; running maximum and sum as the cells pass.
template <class T>
__global__ void __launch_bounds__(128) fa4_simple_kernel(Fa4Args a) {
    extern __shared__ float sm[];
    float* qs = sm;                    // [D]
    float* ps = sm + a.D;              // [128]
    __shared__ float red[4];
    const uint32_t t = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, D = a.D;
    const uint32_t hk = h / (a.n_head / a.n_head_kv);
    const T* q = static_cast<const T*>(a.q) + (size_t)t * a.q_stride + (size_t)h * D;
    for (uint32_t e = tid; e < D; e += 128u) qs[e] = to_f32(q[e]);
    int32_t lo = 0, hi = (int32_t)a.n_kv;
    if (a.ranges) {
        lo = max(a.ranges[2 * t], 0);
        hi = min(a.ranges[2 * t + 1], (int32_t)a.n_kv);
    }
    float m = -INFINITY, l = 0.0f, off = -INFINITY, o[4] = {};
    __syncthreads();
    for (int32_t c0 = lo; c0 < hi; c0 += 128) {
        const int32_t c = c0 + (int32_t)tid;
        bool seen = c < hi;
        float mk = 0.0f;
        if (seen && a.mask) {
            mk = __half2float(a.mask[(size_t)t * a.mask_stride + c]);
            seen = mk != -INFINITY;
        }
        // the mask's running maximum is taken out first: a row of the type's lowest value keeps its scores' digits
        float best = seen && a.mask ? mk : -INFINITY;
        for (int s = 16; s; s >>= 1) best = fmaxf(best, __shfl_xor_sync(0xFFFFFFFFu, best, s));
        if ((tid & 31u) == 0) red[tid >> 5] = best;
        __syncthreads();
        best = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        __syncthreads();
        const float off_new = a.mask ? fmaxf(off, best) : 0.0f;
        const float base = off_new == -INFINITY ? 0.0f : off_new;
        float s = -INFINITY;
        if (seen) {
            const size_t hc = (size_t)hk * a.n_alloc + (size_t)c;
            float acc = 0.0f;
            for (uint32_t e = 0; e < D; ++e) acc = fmaf(qs[e], fa4_value(a.kq + hc * (D / 2u), a.kd + hc * (D / 32u), D, e), acc);
            s = acc * a.scale + (mk - base);
        }
        float top = s;
        for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, x));
        if ((tid & 31u) == 0) red[tid >> 5] = top;
        __syncthreads();
        top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        const float m_old = off == -INFINITY && a.mask ? -INFINITY : m - (a.mask ? base - off : 0.0f);
        const float m_new = fmaxf(m_old, top), m_safe = m_new == -INFINITY ? 0.0f : m_new;
        const float alpha = expf(m_old - m_safe);
        const float p = seen ? expf(s - m_safe) : 0.0f;
        ps[tid] = p;
        __syncthreads();
        l *= alpha;
        for (int j = 0; j < 128; ++j) l += ps[j];
        for (uint32_t k = 0; k * 128u + tid < D; ++k) {
            const uint32_t e = k * 128u + tid;
            o[k] *= alpha;
            for (int j = 0; j < 128 && c0 + j < hi; ++j) {
                if (ps[j] == 0.0f) continue;
                const size_t hc = (size_t)hk * a.n_alloc + (size_t)(c0 + j);
                o[k] = fmaf(ps[j], fa4_value(a.vq + hc * (D / 2u), a.vd + hc * (D / 32u), D, e), o[k]);
            }
        }
        __syncthreads();
        m = m_new;
        off = off_new;
    }
    T* out = static_cast<T*>(a.out) + (size_t)t * a.out_stride + (size_t)h * D;
    for (uint32_t k = 0; k * 128u + tid < D; ++k) out[k * 128u + tid] = from_f32<T>(l == 0.0f ? 0.0f : o[k] / l);
}

template <class T>
cudaError_t fa4_launch(const Fa4Args& a, cudaStream_t st) {
    fa4_simple_kernel<T><<<dim3(a.T, a.n_head), 128, (a.D + 128u) * 4u, st>>>(a);
    return cudaGetLastError();
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
    (void)type; (void)n_head_kv; (void)head_dim; (void)T; (void)n_head; (void)n_kv; (void)group; (void)max_len;
    return 0;
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
    a.D = kv->D;
    a.n_kv = n_kv;
    a.n_alloc = kv->n_alloc;
    a.ranges = ranges;
    a.mask = reinterpret_cast<const __half*>(mask);
    a.mask_stride = mask_stride;
    a.scale = scale;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e = type == TSRC_TYPE_F32 ? fa4_launch<float>(a, st) : type == TSRC_TYPE_F16 ? fa4_launch<__half>(a, st) : fa4_launch<__nv_bfloat16>(a, st);
    if (e != cudaSuccess) return refuse(TSRC_E_CUDA, "tsrc_flash_attn_q4: %s (%s)", cudaGetErrorString(e), cudaGetErrorName(e));
    return TSRC_OK;
}

}  // extern "C"
