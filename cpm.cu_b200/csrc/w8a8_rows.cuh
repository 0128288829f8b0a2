// What the kernels that round rows to 8-bit integers share: a row's values, and maxima and sums over a CTA.
#pragma once
#include "row_ops.cuh"
#include "w8a8.cuh"

namespace w8 {
namespace {

enum Source { SRC_PLAIN, SRC_NORM, SRC_ADD_NORM, SRC_F32 };

// VEC elements of a row from column c on.  fetch() loads them, combine() makes of them what is rounded; apart, so that a thread's loads are
// all in flight before the first residual sum is stored.
template <Source SRC, int VEC>
struct Values {
    float v[VEC], d[SRC == SRC_ADD_NORM ? VEC : 1], w[SRC == SRC_NORM || SRC == SRC_ADD_NORM ? VEC : 1];
    __device__ __forceinline__ void fetch(const RowSource& s, size_t row, int K, int c) {
        if constexpr (SRC == SRC_F32) load_vec<VEC>(s.x32 + row * s.ldx + c, v);
        else load_vec<VEC>(s.x + row * s.ldx + c, v);
        if constexpr (SRC == SRC_ADD_NORM) load_vec<VEC>(s.delta + row * K + c, d);
        if constexpr (SRC == SRC_NORM || SRC == SRC_ADD_NORM) load_vec<VEC>(s.norm + c, w);
    }
    // ss += the squares that a norm needs; `write`: stores the residual sum
    __device__ __forceinline__ void combine(const RowSource& s, size_t row, int K, int c, float& ss, bool write) {
        if constexpr (SRC == SRC_ADD_NORM) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = __bfloat162float(__float2bfloat16(fmaf(d[e], s.delta_scale, v[e])));
            if (write) store_vec<VEC>(s.total + row * K + c, v);
        }
        if constexpr (SRC == SRC_NORM || SRC == SRC_ADD_NORM) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                ss = fmaf(v[e], v[e], ss);
                v[e] *= w[e];
            }
        }
    }
};

__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* sh) {
    v = __reduce_max_sync(0xffffffffu, v);
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    v = (threadIdx.x & 31) < (blockDim.x >> 5) ? sh[threadIdx.x & 31] : 0u;
    return __reduce_max_sync(0xffffffffu, v);
}
// the same value in every thread, summed in the same order whatever the thread
__device__ __forceinline__ float block_total(float v, float* sh) {
    v = warp_sum(v);
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    return warp_sum((threadIdx.x & 31) < (blockDim.x >> 5) ? sh[threadIdx.x & 31] : 0.f);
}

template <int VEC>
__device__ __forceinline__ void store_ints(int8_t* q, const RowRound& round, const float (&v)[VEC]) {
    if constexpr (VEC == 8) {
        uint2 w = make_uint2(0u, 0u);
        if (round.finite) w = make_uint2(pack4(round(v[0]), round(v[1]), round(v[2]), round(v[3])), pack4(round(v[4]), round(v[5]), round(v[6]), round(v[7])));
        *reinterpret_cast<uint2*>(q) = w;
    } else {
        *q = static_cast<int8_t>(round.finite ? round(v[0]) : 0);
    }
}

// whether 16-byte accesses fit the source
inline bool rows_in_vectors(const RowSource& s, int K) {
    auto bits = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
    return K % 8 == 0 && s.ldx % 8 == 0 && ((bits(s.x) | bits(s.x32) | bits(s.norm) | bits(s.delta) | bits(s.total)) & 15) == 0;
}
__device__ __forceinline__ int ceil_div_dev(int a, int b) { return (a + b - 1) / b; }

}  // namespace
}  // namespace w8
