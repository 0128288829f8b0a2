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

// whether 16-byte accesses fit the source (activations are made for them)
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
// q = round(127 v / top) to nearest, even at ties, exactly, for bf16 values and products of two of them.
// Let v and top be integers m and M times powers of two, m, M < 2^16, and r = 127 v / top.  Where r is not half-way between two integers it is at least
// r / (254 m) > r 2^-23.98 away from there (the difference is a fraction with that denominator), and v k, k = 127 / top correctly rounded, is off by
// r 2^-24 at most: one fused multiply-add to a number whose unit is 1 rounds r itself.  Half-way lie (1) |v| = top / 2, r = 63.5, which
// has to become 64; where k was rounded down it would become 63, so that k is taken one step up (bf16 values: m < 2^8, there is room) or v is made a
// little larger (products); and (2) values of rows whose M is a multiple of 127.  Those rows, and rows of tiny values, go through exact(): v and top
// scaled by a power of two so that nothing over- or underflows, an estimate that is at most one off, and the rest 127 v - q top, which fp32 holds
// exactly, decides.  (fp32 rows round 127 v / top as the fused product has it.)
struct RowRound {
    float k, half, c127, top, inv;
    bool finite, plain;   // plain: k rounds the row
    static constexpr float MAGIC = 12582912.f;       // 1.5 * 2^23: v + MAGIC has round(v) in its low byte
    __device__ __forceinline__ RowRound() {}
    // bits: of the row's largest magnitude; products: of two bf16 values; ties: half-way values are to become even (not of fp32 rows)
    __device__ __forceinline__ RowRound(uint32_t bits, bool products, bool ties) {
        finite = bits < 0x7f800000u;
        const float v = __uint_as_float(bits);
        plain = finite && bits >= 0x10000000u && !(ties && ((bits & 0x7fffffu) | 0x800000u) % 127u == 0u);   // 2^-95
        k = plain ? 127.f / v : 0.f;
        half = __uint_as_float(0x7f800000u);                     // no value's magnitude
        if (plain && ties && fmaf(k, v, -127.f) < 0.f) {
            if (products) half = 0.5f * v;
            else k = __uint_as_float(__float_as_uint(k) + 1u);
        }
        int e = static_cast<int>(bits >> 23) - 127;              // v is in [2^e, 2^(e+1)), or below where it is subnormal
        e = e < -119 ? -119 : e;
        const float c = __uint_as_float(static_cast<uint32_t>(127 - (e > 126 ? 126 : e)) << 23);
        const bool some = finite && bits != 0u;
        c127 = some ? 127.f * c : 0.f;
        top = v * c;
        inv = some ? 1.f / top : 0.f;
    }
    // a number whose low byte is the integer
    __device__ __forceinline__ uint32_t exact(float v) const {
        const float p = v * c127;
        const float y = fmaf(p, inv, MAGIC), r = y - MAGIC;
        const float rest = fmaf(-r, top, p), twice = 2.f * fabsf(rest);
        const bool other = twice > top || (twice == top && (__float_as_uint(y) & 1u));
        return __float_as_uint(other ? y + copysignf(1.f, rest) : y);
    }
    // four values to four bytes
    __device__ __forceinline__ static uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
        return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
    }
    template <bool PRODUCTS>
    __device__ __forceinline__ uint32_t four(const float* v) const {
        uint32_t y[4];
        const f32x2 kk = pair(k, k), magic = pair(MAGIC, MAGIC);
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            float a = v[i], b = v[i + 1];
            if constexpr (PRODUCTS) {
                if (fabsf(a) == half) a *= 1.000001f;
                if (fabsf(b) == half) b *= 1.000001f;
            }
            const float2 f = unpair(fma2(pair(a, b), kk, magic));
            y[i] = __float_as_uint(f.x);
            y[i + 1] = __float_as_uint(f.y);
        }
        return low_bytes(y[0], y[1], y[2], y[3]);
    }
    // the row's scale: NaN for a row with an infinity or a NaN, so that its outputs are NaN, and for one whose squares do not fit fp32 (a factor of 0 would
    // give zeros); 0 for a row of zeros, whatever its norm
    __device__ __forceinline__ static float scale(uint32_t bits, float factor) {
        if (bits == 0u) return 0.f;
        return bits < 0x7f800000u && factor != 0.f ? __uint_as_float(bits) / 127.f * factor : __uint_as_float(0x7fffffffu);
    }
};

// Out of line: few rows need it, and a launch begins by fetching its instructions.
__device__ __noinline__ uint2 exact8(float v0, float v1, float v2, float v3, float v4, float v5, float v6, float v7, float c127, float top, float inv) {
    RowRound r;
    r.c127 = c127; r.top = top; r.inv = inv;
    return make_uint2(RowRound::low_bytes(r.exact(v0), r.exact(v1), r.exact(v2), r.exact(v3)),
                      RowRound::low_bytes(r.exact(v4), r.exact(v5), r.exact(v6), r.exact(v7)));
}

// eight values to eight integers
template <bool PRODUCTS>
__device__ __forceinline__ uint2 ints_of(const RowRound& round, const float (&v)[8]) {
    if (round.plain) return make_uint2(round.four<PRODUCTS>(v), round.four<PRODUCTS>(v + 4));
    if (round.finite) return exact8(v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7], round.c127, round.top, round.inv);
    return make_uint2(0u, 0u);
}

// ---------------------------------------------------------------- eight consecutive elements of a row
// fetch() loads them, combine() makes the residual sum, the largest magnitude and the squares of it, values() gives what is rounded.  A row waits for its
// maximum in registers: as it came (bf16, fp32), or as the products with the norm's weights (fp32, in the registers of x and the weights).
// WIDE: 16-byte accesses; otherwise element by element (rows at odd places, or of other widths than multiples of eight), zeros beyond the row's end.
// (2000 rows of 5121 and a product of 64 columns: 17.8 us; one element per thread and step 33.5.)
template <Source SRC, bool WIDE>
struct Values {
    using T = typename std::conditional<SRC == SRC_F32, float, bf16>::type;
    struct alignas(16) Block {
        T e[8];
        __device__ __forceinline__ float at(int i) const {
            if constexpr (SRC == SRC_F32) {
                return e[i];
            } else {
                const uint32_t two = reinterpret_cast<const uint32_t*>(e)[i >> 1];
                return i & 1 ? high(two) : low(two);
            }
        }
        __device__ __forceinline__ void load(const T* p, int left) {   // left: elements to the row's end
            if constexpr (WIDE) {
                *this = *reinterpret_cast<const Block*>(p);
            } else {
                uint16_t w[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) w[i] = i < left ? reinterpret_cast<const uint16_t*>(p)[i] : uint16_t(0);
#pragma unroll
                for (int i = 0; i < 4; ++i) reinterpret_cast<uint32_t*>(e)[i] = w[2 * i] | static_cast<uint32_t>(w[2 * i + 1]) << 16;
            }
        }
        __device__ __forceinline__ void store(T* p, int left) const {
            if constexpr (WIDE) {
                *reinterpret_cast<Block*>(p) = *this;
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t two = reinterpret_cast<const uint32_t*>(e)[i >> 1];
                    if (i < left) reinterpret_cast<uint16_t*>(p)[i] = static_cast<uint16_t>(i & 1 ? two >> 16 : two);
                }
            }
        }
    };
    static_assert(WIDE || SRC != SRC_F32, "activations come in whole vectors");
    Block t, d, w;
    float p[8];
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
        t.load(base(s) + row * s.ldx + c, K - c);
        if constexpr (SRC == SRC_ADD_NORM) d.load(s.delta + row * K + c, K - c);
        if constexpr (HAS_NORM<SRC>) w.load(s.norm + c, K - c);
    }
    // `write`: stores the residual sum
    __device__ __forceinline__ void combine(const RowSource& s, size_t row, int K, int c, bool write, uint32_t& top, float& ss) {
        if constexpr (SRC == SRC_ADD_NORM) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                reinterpret_cast<uint32_t*>(t.e)[i] = two_bf16(fmaf(d.at(2 * i), s.delta_scale, t.at(2 * i)), fmaf(d.at(2 * i + 1), s.delta_scale, t.at(2 * i + 1)));
            }
            if (write) t.store(s.total + row * K + c, K - c);
        }
        if constexpr (SRC == SRC_PLAIN) {   // two magnitudes at a time, as 16-bit patterns
            const uint32_t* pairs = reinterpret_cast<const uint32_t*>(t.e);
            uint32_t m = 0u;
#pragma unroll
            for (int i = 0; i < 4; ++i) m = __vmaxu2(m, pairs[i] & 0x7fff7fffu);
            top = max(top, max(m << 16, m & 0xffff0000u));
        } else {
            float m = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float v = t.at(e);
                if constexpr (HAS_NORM<SRC>) {
                    ss = fmaf(v, v, ss);
                    v *= w.at(e);
                    p[e] = v;
                }
                m = max_magnitude(m, v);
            }
            top = max(top, __float_as_uint(m));
        }
    }
    __device__ __forceinline__ void values(float (&v)[8]) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if constexpr (HAS_NORM<SRC>) v[e] = p[e];
            else v[e] = t.at(e);
        }
    }
};

}  // namespace
}  // namespace w8
