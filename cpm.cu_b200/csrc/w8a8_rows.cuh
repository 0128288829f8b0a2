// What the kernels that round rows to 8-bit integers share: a row's values, the rounding, and maxima and sums over a CTA.
#pragma once
#include <type_traits>

#include "row_ops.cuh"
#include "w8a8.cuh"

namespace w8 {
namespace {

enum Source { SRC_PLAIN, SRC_NORM, SRC_ADD_NORM, SRC_F32 };
template <Source S>
constexpr bool HAS_NORM = S == SRC_NORM || S == SRC_ADD_NORM;

// whether 16-byte accesses fit the source
inline bool rows_in_vectors(const RowSource& s, int K) {
    auto bits = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
    return K % 8 == 0 && s.ldx % 8 == 0 && ((bits(s.x) | bits(s.x32) | bits(s.norm) | bits(s.delta) | bits(s.total)) & 15) == 0;
}

// ---------------------------------------------------------------- the largest magnitude
// NaN, where there is one, stays
__device__ __forceinline__ float max_magnitude(float top, float v) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(top), "f"(fabsf(v)));
    return r;
}
// as a bit pattern: infinities and NaN are above all finite magnitudes
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

// ---------------------------------------------------------------- rounding
// q = round(127 v / top) to nearest, even at ties, exactly.  v * k, k = 127 / top rounded, is off by less than 127 * 2^-23 from 127 v / top, so that
// its nearest integer is the one, unless it lies within NEAR of the middle between two; a vector with such a value is rounded again by exact().
// There v and top are scaled by a power of two so that nothing over- or underflows, an estimate is at most one off, and the rest
// 127 v - q top, which fp32 holds exactly for v of up to 17 significant bits (bf16 values and products of two of them), decides.  (Rows of
// fp32 values round the middle as their fp32 rests have it.)
struct RowRound {
    float k, c127, top, inv;
    bool finite, plain;   // plain: k is exact enough; not for rows of tiny values
    static constexpr float MAGIC = 12582912.f;       // 1.5 * 2^23: v + MAGIC has round(v) in its low byte
    static constexpr float NEAR = 0.49996f;
    __device__ __forceinline__ explicit RowRound(uint32_t bits) {
        finite = bits < 0x7f800000u;
        plain = finite && bits >= 0x10000000u;                   // 2^-95
        const float v = __uint_as_float(bits);
        k = plain ? 127.f / v : 0.f;
        int e = static_cast<int>(bits >> 23) - 127;              // v is in [2^e, 2^(e+1)), or below where it is subnormal
        e = e < -119 ? -119 : e;
        const float c = __uint_as_float(static_cast<uint32_t>(127 - (e > 126 ? 126 : e)) << 23);
        const bool some = finite && bits != 0u;
        c127 = some ? 127.f * c : 0.f;
        top = v * c;
        inv = some ? 1.f / top : 0.f;
    }
    __device__ __forceinline__ int exact(float v) const {
        const float p = v * c127;
        float r = rintf(p * inv);
        const float rest = fmaf(-r, top, p);
        const float twice = 2.f * fabsf(rest);
        if (twice > top || (twice == top && (static_cast<int>(r) & 1))) r += copysignf(1.f, rest);
        return static_cast<int>(r);
    }
    // four values to four bytes; near: largest distance from an integer so far
    __device__ __forceinline__ uint32_t four(const float* v, float& near) const {
        uint32_t y[4];
        const f32x2 kk = pair(k, k), magic = pair(MAGIC, MAGIC), minus = pair(-1.f, -1.f);
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            const f32x2 x = pair(v[i], v[i + 1]);
            const f32x2 sum = fma2(x, kk, magic);
            const float2 off = unpair(fma2(x, kk, fma2(sum, minus, magic)));   // v k - round(v k)
            near = fmaxf(near, fmaxf(fabsf(off.x), fabsf(off.y)));
            const float2 f = unpair(sum);
            y[i] = __float_as_uint(f.x);
            y[i + 1] = __float_as_uint(f.y);
        }
        return __byte_perm(__byte_perm(y[0], y[1], 0x0040), __byte_perm(y[2], y[3], 0x0040), 0x5410);
    }
    // the row's scale: NaN for a row with an infinity or a NaN, so that its outputs are NaN
    __device__ __forceinline__ static float scale(uint32_t bits, float factor) {
        return bits < 0x7f800000u ? __uint_as_float(bits) / 127.f * factor : __uint_as_float(0x7fffffffu);
    }
};

__device__ __forceinline__ uint32_t pack4(int a, int b, int c, int d) {
    return (a & 0xff) | (b & 0xff) << 8 | (c & 0xff) << 16 | static_cast<uint32_t>(d) << 24;
}

// Eight values of a vector that has one near a border, or of a row of tiny values.  Out of line: it is rarely run, and a launch begins by fetching its
// instructions.
__device__ __noinline__ uint2 exact8(float v0, float v1, float v2, float v3, float v4, float v5, float v6, float v7, float c127, float top, float inv) {
    RowRound r(0u);
    r.c127 = c127; r.top = top; r.inv = inv;
    return make_uint2(pack4(r.exact(v0), r.exact(v1), r.exact(v2), r.exact(v3)), pack4(r.exact(v4), r.exact(v5), r.exact(v6), r.exact(v7)));
}

template <int VEC>
__device__ __forceinline__ void store_ints(int8_t* q, const RowRound& round, const float (&v)[VEC]) {
    if constexpr (VEC == 8) {
        uint2 w = make_uint2(0u, 0u);
        float near = 0.f;
        if (round.plain) w = make_uint2(round.four(v, near), round.four(v + 4, near));
        if (round.finite && (near > RowRound::NEAR || !round.plain)) {
            w = exact8(v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7], round.c127, round.top, round.inv);
        }
        *reinterpret_cast<uint2*>(q) = w;
    } else {
        *q = static_cast<int8_t>(round.finite ? round.exact(v[0]) : 0);
    }
}

// ---------------------------------------------------------------- VEC consecutive elements of a row
// fetch() loads them, combine() makes the residual sum, the largest magnitude and the squares of it, values() gives what is rounded.  A row waits for its
// maximum in registers: as it came (bf16, fp32), or as the products with the norm's weights (fp32, in the registers of x and the weights).
template <Source SRC, int VEC>
struct Values {
    using T = typename std::conditional<SRC == SRC_F32, float, bf16>::type;
    struct alignas(VEC == 8 ? 16 : sizeof(T)) Block { T e[VEC]; };
    Block t, d, w;
    float p[VEC];
    __device__ __forceinline__ static const T* base(const RowSource& s) {
        if constexpr (SRC == SRC_F32) return s.x32;
        else return s.x;
    }
    // asks for the lines ahead of the wait for the predecessor: into L2 only, where later writes find them
    __device__ __forceinline__ static void ask(const RowSource& s, size_t row, int K, int c) {
        prefetch_l2(base(s) + row * s.ldx + c);
        if constexpr (SRC == SRC_ADD_NORM) prefetch_l2(s.delta + row * K + c);
        if constexpr (HAS_NORM<SRC>) prefetch_l2(s.norm + c);
    }
    __device__ __forceinline__ void fetch(const RowSource& s, size_t row, int K, int c) {
        t = *reinterpret_cast<const Block*>(base(s) + row * s.ldx + c);
        if constexpr (SRC == SRC_ADD_NORM) d = *reinterpret_cast<const Block*>(s.delta + row * K + c);
        if constexpr (HAS_NORM<SRC>) w = *reinterpret_cast<const Block*>(s.norm + c);
    }
    // `write`: stores the residual sum
    __device__ __forceinline__ void combine(const RowSource& s, size_t row, int K, int c, bool write, uint32_t& top, float& ss) {
        if constexpr (SRC == SRC_ADD_NORM) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) t.e[e] = __float2bfloat16(fmaf(__bfloat162float(d.e[e]), s.delta_scale, __bfloat162float(t.e[e])));
            if (write) *reinterpret_cast<Block*>(s.total + row * K + c) = t;
        }
        if constexpr (SRC == SRC_PLAIN && VEC == 8) {   // two magnitudes at a time, as 16-bit patterns
            const uint32_t* pairs = reinterpret_cast<const uint32_t*>(t.e);
            uint32_t m = 0u;
#pragma unroll
            for (int i = 0; i < 4; ++i) m = __vmaxu2(m, pairs[i] & 0x7fff7fffu);
            top = max(top, max(m << 16, m & 0xffff0000u));
        } else {
            float m = 0.f;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                float v = to_float(t.e[e]);
                if constexpr (HAS_NORM<SRC>) {
                    ss = fmaf(v, v, ss);
                    v *= to_float(w.e[e]);
                    p[e] = v;
                }
                m = max_magnitude(m, v);
            }
            top = max(top, __float_as_uint(m));
        }
    }
    __device__ __forceinline__ void values(float (&v)[VEC]) const {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            if constexpr (HAS_NORM<SRC>) v[e] = p[e];
            else v[e] = to_float(t.e[e]);
        }
    }
};

}  // namespace
}  // namespace w8
