// tsrc_kv4.cuh -- the q4_0 KV cache's device layout, shared by its kernels (tsrc_kv4.cu) and the attention
// over it (tsrc_fa4.cu).
//
// A plane (K or V) is split per KV head. A cell of one head is a row of D / 2 bytes of codes and D / 32 fp16
// scales, in separate arrays:
//   codes   q[head][cell][D / 2]
//   scales  d[head][cell][D / 32]
// A code row is cut into groups of up to 128 values (four blocks of 32; two for D = 64), and a group into eight
// chunks, one for each g = 0..7: chunk g holds, block after block, the 16 bits {n(4g), n(4g+1), n(4g+2), n(4g+3)}
// (low to high) of the block's values 4g .. 4g + 3. So the eight lanes that share an mma column index each own
// one chunk (8 bytes; 4 for D = 64) with four values of every block, and two neighbouring chunks (16 bytes) are
// the eight values of every block that a lane feeds to the four k indices it owns: K and V are both read in the
// fragment layout with wide loads and no shuffles, and K and V planes look alike.
// In every second run of four cells chunk g lies in place g ^ 4: the lanes that read one chunk of four or eight
// cells of a tile in shared memory then meet no bank twice.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include <type_traits>

#include "../../include/tsrc.h"
#include "tsrc_internal.h"

struct tsrc_kv4 {
    tsrc_ctx* ctx;
    uint32_t n_head_kv, D, n_cells, n_alloc;   // n_alloc: n_cells rounded up to 64 (zero padding)
    uint8_t* q[2];                              // [K, V] codes [n_head_kv][n_alloc][D / 2]
    __half* d[2];                               //        scales [n_head_kv][n_alloc][D / 32]
    uint8_t* mem;
};

namespace tsrc {

constexpr uint32_t kKv4Pad = 64;

// where chunk g of a cell's row lies
__host__ __device__ __forceinline__ uint32_t kv4_place(uint32_t g, size_t cell) { return g ^ ((uint32_t)cell & 4u); }

// Restores the calling thread's current device when it leaves an entry point.
class DeviceScope {
public:
    explicit DeviceScope(const tsrc_ctx* ctx) {
        int dev = -1;
        if (cudaGetDevice(&was_) != cudaSuccess) was_ = -1;
        rc = ctx_device(ctx, &dev);
        if (was_ == dev) was_ = -1;
    }
    ~DeviceScope() {
        if (was_ >= 0) cudaSetDevice(was_);
    }
    DeviceScope(const DeviceScope&) = delete;
    DeviceScope& operator=(const DeviceScope&) = delete;
    int rc;

private:
    int was_ = -1;
};

template <class... A>
inline int refuse(int code, const char* fmt, A... a) {
    char msg[256];
    snprintf(msg, sizeof msg, fmt, a...);
    return set_error(code, msg);
}
// A CUDA call's error as the entry point's. The runtime keeps it as the thread's last error, which the next launch would take
// for its own, so it is taken from there.
inline int cuda_refuse(cudaError_t e, const char* who) {
    (void)cudaGetLastError();
    return refuse(TSRC_E_CUDA, "%s: %s (%s)", who, cudaGetErrorString(e), cudaGetErrorName(e));
}

inline bool kv4_type_ok(uint32_t type) { return type == TSRC_TYPE_F32 || type == TSRC_TYPE_F16 || type == TSRC_TYPE_BF16; }
inline uint32_t kv4_type_size(uint32_t type) { return type == TSRC_TYPE_F32 ? 4u : 2u; }
inline bool kv4_geometry_ok(uint32_t n_head_kv, uint32_t D) {
    return (D == 64 || D == 128 || D == 256 || D == 512) && n_head_kv >= 1 && n_head_kv <= 511u * 64u / D;
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Eight neighbouring values, loaded with 16-byte accesses where the address allows (VEC) or one by one.
template <class T, bool VEC>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
    if constexpr (VEC && sizeof(T) == 4) {
        const float4 a = __ldcs(reinterpret_cast<const float4*>(p)), b = __ldcs(reinterpret_cast<const float4*>(p) + 1);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else if constexpr (VEC) {
        const uint4 a = __ldcs(reinterpret_cast<const uint4*>(p));
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same_v<T, __half>) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                v[2 * i] = f.x;
                v[2 * i + 1] = f.y;
            } else {
                v[2 * i] = __uint_as_float(w[i] << 16);
                v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_f32(p[i]);
    }
}
// d x of eight small whole numbers x, paired as (0, 4), (1, 5), (2, 6), (3, 7), rounded once to T and stored.
template <class T, bool VEC>
__device__ __forceinline__ void store8(T* p, const __half2 (&x)[4], __half d) {
    if constexpr (std::is_same_v<T, __half>) {
        uint32_t y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2 h = __hmul2(x[i], __half2half2(d));
            y[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        if constexpr (VEC)
            __stcs(reinterpret_cast<uint4*>(p), make_uint4(__byte_perm(y[0], y[1], 0x5410), __byte_perm(y[2], y[3], 0x5410),
                                                           __byte_perm(y[0], y[1], 0x7632), __byte_perm(y[2], y[3], 0x7632)));
        else {
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = __ushort_as_half((unsigned short)(y[i & 3] >> (i & 4 ? 16 : 0)));
        }
    } else {
        const float f = __half2float(d);
        float y[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 h = __half22float2(x[i]);
            y[i] = f * h.x;
            y[i + 4] = f * h.y;
        }
        if constexpr (VEC && sizeof(T) == 4) {
            __stcs(reinterpret_cast<float4*>(p), make_float4(y[0], y[1], y[2], y[3]));
            __stcs(reinterpret_cast<float4*>(p) + 1, make_float4(y[4], y[5], y[6], y[7]));
        } else if constexpr (VEC) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(y[2 * i], y[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&h);
            }
            __stcs(reinterpret_cast<uint4*>(p), make_uint4(w[0], w[1], w[2], w[3]));
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = from_f32<T>(y[i]);
        }
    }
}

}  // namespace tsrc
