// Rotary positions, sm_100a:  pair i of every query and key head of a row becomes
//   (a cos - b sin, b cos + a sin),  angle = pos * inv_freq[i],  sines and cosines times a factor,
// with pair i = elements (2 i, 2 i + 1) (interleaved) or (i, i + half), on the first 2 * half elements of a head; the rest of it is copied.
// Rotated keys, and values as they are, go to the row's cache slot.
//
// The angle is a 64-bit product, reduced to a fraction of a turn before it becomes fp32: at position 10^6 an fp32 product is off by 0.03
// radians.  One CTA per row: its loads are in flight while some threads make the row's `half` sines and cosines.
//
// Bound: every element in and out once.
#include "row_ops.cuh"
#include "rotary.cuh"

namespace {

// VEC elements as they lie in memory; WIDE: in one access
template <int VEC, bool WIDE>
struct Elems {
    bf16 e[VEC];
    __device__ __forceinline__ void load(const bf16* p) {
        if constexpr (!WIDE) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) e[i] = p[i];
        } else if constexpr (VEC == 8) *reinterpret_cast<uint4*>(e) = *reinterpret_cast<const uint4*>(p);
        else if constexpr (VEC == 4) *reinterpret_cast<uint2*>(e) = *reinterpret_cast<const uint2*>(p);
        else *reinterpret_cast<uint32_t*>(e) = *reinterpret_cast<const uint32_t*>(p);
    }
    __device__ __forceinline__ void store(bf16* p) const {
        if constexpr (!WIDE) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) p[i] = e[i];
        } else if constexpr (VEC == 8) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(e);
        else if constexpr (VEC == 4) *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(e);
        else *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<const uint32_t*>(e);
    }
};

__device__ __forceinline__ void turn(bf16& a, bf16& b, float cs, float sn) {
    const float x = __bfloat162float(a), y = __bfloat162float(b);
    a = __float2bfloat16(fmaf(x, cs, -(y * sn)));
    b = __float2bfloat16(fmaf(y, cs, x * sn));
}

// A piece of a row: with PAIRED halves VEC elements and their partners `half` further on, or VEC elements that lie together.
template <int VEC, bool INTERLEAVED, bool WIDE>
struct Piece {
    Elems<VEC, WIDE> lo, hi;
    __device__ __forceinline__ void load(const bf16* p, int half) {
        lo.load(p);
        if constexpr (!INTERLEAVED) hi.load(p + half);
    }
    // c: first element in the head
    __device__ __forceinline__ void rotate(int c, int half, const float2* table) {
        if constexpr (INTERLEAVED) {
#pragma unroll
            for (int j = 0; j < VEC; j += 2) {
                const int i = (c + j) >> 1;
                if (i < half) turn(lo.e[j], lo.e[(j + 1) % VEC], table[i].x, table[i].y);
            }
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j) turn(lo.e[j], hi.e[j], table[c + j].x, table[c + j].y);
        }
    }
    __device__ __forceinline__ void store(bf16* p, int half) const {
        lo.store(p);
        if constexpr (!INTERLEAVED) hi.store(p + half);
    }
};

constexpr int MAX_HALF = 512;

// R rows per CTA.  Each thread's first pieces of all its rows are in flight before the tables are made.
template <int VEC, bool INTERLEAVED, bool WIDE, int R>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryArgs a, int rows) {
    extern __shared__ float2 table[];   // [R][half]
    constexpr int AHEAD = 2;
    const int kv_dim = a.kv_heads * a.dim, all = a.heads + a.kv_heads;
    // pieces of a head that are rotated (interleaved: all of it, the unrotated pairs as they are), and that are copied
    const int turned = INTERLEAVED ? a.dim / VEC : a.half / VEC, copied = INTERLEAVED ? 0 : (a.dim - 2 * a.half) / VEC;
    const int items = all * turned;
    const int v0 = threadIdx.x * VEC;
    const long long r0 = static_cast<long long>(blockIdx.x) * R;
    // where this thread's first pieces lie in a row
    int head[AHEAD], first[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
        const int i = threadIdx.x + j * blockDim.x;
        head[j] = turned > 0 ? i / turned : 0;
        first[j] = turned > 0 ? (i - head[j] * turned) * VEC : 0;
    }
    grid_dep_wait();
    grid_dep_trigger();
    auto row_at = [&](int r) { return a.qkv + (r0 + r) * a.ld; };
    Piece<VEC, INTERLEAVED, WIDE> piece[R][AHEAD];
    Elems<VEC, WIDE> value[R];
    int32_t slot[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        slot[r] = a.kv_heads > 0 && r0 + r < rows ? a.slots[r0 + r] : -1;
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            if (threadIdx.x + j * blockDim.x < items && r0 + r < rows) piece[r][j].load(row_at(r) + head[j] * a.dim + first[j], a.half);
        }
        if (v0 < kv_dim && r0 + r < rows) value[r].load(row_at(r) + all * a.dim + v0);
    }
    for (int t = threadIdx.x; t < R * a.half; t += blockDim.x) {
        const int r = R > 1 ? t / a.half : 0, i = t - r * a.half;
        if (r0 + r < rows) {
            const double turns = static_cast<double>(a.pos[r0 + r]) * static_cast<double>(a.inv_freq[i]) * 0.15915494309189533577;
            float sn, cs;
            sincospif(2.f * static_cast<float>(turns - rint(turns)), &sn, &cs);
            table[t] = make_float2(cs * a.factor, sn * a.factor);
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (slot[r] >= a.cache_rows) {   // memory stays intact; the host hears of it
            slot[r] = -1;
            if (threadIdx.x == 0) atomicOr(a.error, ERR_KV_OVERFLOW);
        }
        if (slot[r] >= 0 && v0 < kv_dim) value[r].store(a.v_cache + static_cast<long long>(slot[r]) * kv_dim + v0);
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (r0 + r >= rows) break;
        const bf16* row = row_at(r);
        bf16* q = a.q + (r0 + r) * a.ldq;
        const bool keep = slot[r] >= 0;
        bf16* k = a.k_cache + static_cast<long long>(slot[r]) * kv_dim;
        auto target = [&](int h, int c) { return h < a.heads ? q + h * a.dim + c : k + (h - a.heads) * a.dim + c; };
        auto finish = [&](Piece<VEC, INTERLEAVED, WIDE>& e, int h, int c) {
            e.rotate(c, a.half, table + r * a.half);
            if (h < a.heads || keep) e.store(target(h, c), a.half);
        };
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            if (threadIdx.x + j * blockDim.x < items) finish(piece[r][j], head[j], first[j]);
        }
        for (int i = threadIdx.x + AHEAD * blockDim.x; i < items; i += blockDim.x) {
            const int h = i / turned, c = (i - h * turned) * VEC;
            piece[r][0].load(row + h * a.dim + c, a.half);
            finish(piece[r][0], h, c);
        }
        // what no rotation reaches: the rest of the heads, and the values
        for (int j = threadIdx.x; j < all * copied; j += blockDim.x) {
            const int h = j / copied, c = 2 * a.half + (j - h * copied) * VEC;
            Elems<VEC, WIDE> e;
            e.load(row + h * a.dim + c);
            if (h < a.heads || keep) e.store(target(h, c));
        }
        if (keep) {
            bf16* v_row = a.v_cache + static_cast<long long>(slot[r]) * kv_dim;
            for (int j = v0 + blockDim.x * VEC; j < kv_dim; j += blockDim.x * VEC) {
                value[r].load(row + all * a.dim + j);
                value[r].store(v_row + j);
            }
        }
    }
}

}  // namespace

int rotary_max_pairs() { return MAX_HALF; }

void launch_rotary(const RotaryArgs& a, int rows, bool interleaved, cudaStream_t s) {
    if (rows <= 0) return;
    // the widest access that every piece's start allows
    auto bits = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
    auto fits = [&](int vec) {
        return a.dim % vec == 0 && (interleaved || a.half % vec == 0) && a.ld % vec == 0 && a.ldq % vec == 0 &&
               ((bits(a.qkv) | bits(a.q) | bits(a.k_cache) | bits(a.v_cache)) & (2 * vec - 1)) == 0;
    };
    const int vec = fits(8) ? 8 : fits(4) ? 4 : (interleaved || fits(2)) ? 2 : 1;
    const bool wide = fits(vec);
    const int pieces = (a.heads + 2 * a.kv_heads) * a.dim / vec;
    const int threads = pieces >= 256 ? 256 : (pieces + 31) / 32 * 32;
    const int sms = runtime().num_sms;
    // two rows per CTA once there are several CTAs for every SM: their loads and tables overlap (TWO_ROWS figures at the top)
    const bool two = rows >= 8 * sms;
    auto go = [&](auto kernel, int per_cta) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(ceil_div(rows, per_cta));
        cfg.blockDim = dim3(threads);
        cfg.dynamicSmemBytes = static_cast<size_t>(per_cta) * a.half * sizeof(float2);
        cfg.stream = s;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = runtime().pdl ? 1 : 0;
        CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, a, rows));
    };
    if (interleaved) {
        if (vec == 8 && two) go(rotary_kernel<8, true, true, 2>, 2);
        else if (vec == 8) go(rotary_kernel<8, true, true, 1>, 1);
        else if (vec == 4) go(rotary_kernel<4, true, true, 1>, 1);
        else if (wide) go(rotary_kernel<2, true, true, 1>, 1);
        else go(rotary_kernel<2, true, false, 1>, 1);
    } else {
        if (vec == 8 && two) go(rotary_kernel<8, false, true, 2>, 2);
        else if (vec == 8) go(rotary_kernel<8, false, true, 1>, 1);
        else if (vec == 4) go(rotary_kernel<4, false, true, 1>, 1);
        else if (vec == 2) go(rotary_kernel<2, false, true, 1>, 1);
        else go(rotary_kernel<1, false, false, 1>, 1);
    }
}
