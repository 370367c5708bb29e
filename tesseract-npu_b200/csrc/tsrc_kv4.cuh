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

// Four neighbouring values, loaded or stored at once where the address allows (VEC) or one by one.
template <class T, bool VEC>
__device__ __forceinline__ void load4(const T* p, float (&v)[4]) {
    if constexpr (VEC) {
        if constexpr (sizeof(T) == 4) {
            const float4 w = *reinterpret_cast<const float4*>(p);
            v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
        } else {
            const uint2 w = *reinterpret_cast<const uint2*>(p);
            T t[4];
            __builtin_memcpy(t, &w, 8);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = to_f32(t[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = to_f32(p[i]);
    }
}
template <class T, bool VEC>
__device__ __forceinline__ void store4(T* p, const float (&v)[4]) {
    if constexpr (VEC) {
        T t[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i] = from_f32<T>(v[i]);
        if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
        else {
            uint2 w;
            __builtin_memcpy(&w, t, 8);
            *reinterpret_cast<uint2*>(p) = w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = from_f32<T>(v[i]);
    }
}

}  // namespace tsrc
