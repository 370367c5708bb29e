// tsrc_fa4.cuh -- what the two kernels of the attention over the q4_0 cache share (tsrc_fa4.cu, tsrc_fa4_tc.cu).
#pragma once

#include "tsrc_kv4.cuh"

namespace tsrc {

struct Fa4Args {
    const void* q;
    void* out;
    size_t q_stride, out_stride;
    bool q_wide, out_wide, mask_wide;          // rows allow 16-byte (out: four-value) accesses
    const uint8_t *kq, *vq;
    const __half *kd, *vd;
    uint32_t T, n_head, n_head_kv, G, n_kv, n_alloc;
    const int32_t* ranges;
    const __half* mask;
    size_t mask_stride;
    float scale;
    uint32_t tile_rows;                        // rows of a row tile, in the kernel for many rows
    uint32_t group, row_tiles, splits;         // tokens a group, row tiles a group and KV head, splits of the cells
    float *part_o, *part_ml;                   // splits joined by the merge kernel: [unit][split][R][D], [unit][split][R][4]
};

template <class T>
__device__ __forceinline__ void store4(T* p, const float (&x)[4], bool wide) {
    if (wide) {
        if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
        else {
            T t[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) t[i] = from_f32<T>(x[i]);
            uint2 w;
            w.x = (uint32_t)reinterpret_cast<const unsigned short&>(t[0]) | (uint32_t)reinterpret_cast<const unsigned short&>(t[1]) << 16;
            w.y = (uint32_t)reinterpret_cast<const unsigned short&>(t[2]) | (uint32_t)reinterpret_cast<const unsigned short&>(t[3]) << 16;
            *reinterpret_cast<uint2*>(p) = w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = from_f32<T>(x[i]);
    }
}

// Many query rows on one stretch of cells: D 64 or 128, row tiles of 128, or of 256 for bf16 (one split)
// (tsrc_fa4_tc.cu).
constexpr uint32_t kFa4TcRows = 128;
cudaError_t launch_fa4_tc(uint32_t type, uint32_t D, const Fa4Args& a, uint32_t units, cudaStream_t st);
// The error word of its waits (kKv4ErrWait), cleared when read with clear = true.
cudaError_t fa4_error(uint32_t* code, bool clear);

}  // namespace tsrc
