// Rows to 8-bit integers, sm_100a:  q = round(127 v / top), scale = top / 127, with top the largest magnitude of the row, alone or
// behind a residual sum and an RMS norm; and the packing of 8-bit weights.
//
// A norm multiplies a whole row by 1 / rms, which cancels in v / top: the integers are those of t * w, a product of two bf16 values and
// exact in fp32, and the factor goes into the scale.  So the sum of squares and the largest magnitude are found in the same pass, and the integers
// do not depend on the order of any sum.
//
// Bound: bytes.  One CTA per row, which stays in registers between the pass that finds the maximum and the one that rounds; rows too
// long for that are read twice.  A row with an infinity or a NaN gets the scale NaN and integers 0, a row of zeros the scale 0.
// 4096 rows of 16384: 35.4 us (5.7 TB/s), of 4096: 9.1 (5.5); 60 rows of 16384: 2.7, of 4096: 1.5.  Alone and cold (every launch by itself, from HBM): 4096 rows of 4096
// 11.0, behind a norm 18.6, behind a residual sum and a norm 21.7; of 8192 17.6, 29.6, 37.0; 2000 rows of 5121 11.7 (with rows of q in whole vectors), 20.1, 40.9.
// Behind a norm it is not the bytes: each row reads the norm's weights again, from L2, and meets twice.  Element by element it is the number of accesses, of 2 bytes.
#include <algorithm>

#include "w8a8_rows.cuh"

namespace w8 {
namespace {

constexpr int CLEARING = 1 << 16;   // CTAs that clear counters
struct QuantizeArgs {
    RowSource src;
    int K, pad_to;
    int8_t* q;
    long long ldq;
    bool q_wide;     // rows of q are 8-byte aligned and have room for whole vectors
    float* scale;
    int* clear;
    int n_clear, clear_step;   // step: the threads that clear
};

// VPT > 0: a thread's VPT pieces of eight elements stay in registers; 0: the row is read twice.
// Lets its successor start behind its own wait: a product may then fetch weights, which are older than this launch's predecessor.
template <int VPT>
constexpr int MOST_THREADS = VPT == 1 || VPT == 2 ? 1024 : VPT == 4 ? 512 : 256;
template <Source SRC, int VPT, bool WIDE>
__global__ void __launch_bounds__(MOST_THREADS<VPT>) quantize_kernel(const QuantizeArgs a) {
    __shared__ uint32_t sh_top[32];
    __shared__ float sh_sum[32];
    const size_t row = blockIdx.x;
    if (static_cast<int>(threadIdx.x) * 8 < a.K && threadIdx.x % 8 == 0) Values<SRC, WIDE>::ask(a.src, row, a.K, threadIdx.x * 8);
    grid_dep_wait();
    grid_dep_trigger();
    if (blockIdx.x < static_cast<unsigned>(CLEARING)) {   // not by all: numbers of 2^31 threads do not fit 32 bits
#pragma unroll 1
        for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < a.n_clear; i += a.clear_step) a.clear[i] = 0;
    }
    Values<SRC, WIDE> kept[VPT > 0 ? VPT : 1];
    float ss = 0.f;
    uint32_t top = 0u;
    const int step = blockDim.x * 8;
    if constexpr (VPT > 0) {
        // every load of the row is in flight before the first sum is stored
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int c = threadIdx.x * 8 + j * step;
            if (c < a.K) kept[j].fetch(a.src, row, a.K, c);
        }
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int c = threadIdx.x * 8 + j * step;
            if (c < a.K) {
                kept[j].combine(a.src, row, a.K, c, true, top, ss);
            }
        }
    } else {
        for (int c = threadIdx.x * 8; c < a.K; c += step) {
            kept[0].fetch(a.src, row, a.K, c);
            kept[0].combine(a.src, row, a.K, c, true, top, ss);
        }
    }
    top = block_max(top, sh_top);
    float factor = 1.f;
    if constexpr (HAS_NORM<SRC>) factor = 1.f / sqrtf(block_total(ss, sh_sum) / a.K + a.src.eps);
    const RowRound round(top, HAS_NORM<SRC>, SRC != SRC_F32);
    int8_t* q = a.q + row * a.ldq;
    auto finish = [&](const Values<SRC, WIDE>& r, int c) {
        float v[8];
        r.values(v);
        const uint2 w = ints_of<HAS_NORM<SRC>>(round, v);
        if (WIDE || a.q_wide) {
            *reinterpret_cast<uint2*>(q + c) = w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (c + i < a.K) q[c + i] = static_cast<int8_t>((i < 4 ? w.x : w.y) >> (i % 4 * 8));
            }
        }
    };
    if constexpr (VPT > 0) {
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int c = threadIdx.x * 8 + j * step;
            if (c < a.K) finish(kept[j], c);
        }
    } else {
        for (int c = threadIdx.x * 8; c < a.K; c += step) {
            kept[0].fetch(a.src, row, a.K, c);
            uint32_t known = 0u;
            float squares = 0.f;
            kept[0].combine(a.src, row, a.K, c, false, known, squares);
            finish(kept[0], c);
        }
    }
    for (int c = a.K + threadIdx.x; c < a.pad_to; c += blockDim.x) q[c] = 0;
    if (threadIdx.x == 0) a.scale[row] = RowRound::scale(top, factor);
}

template <Source SRC, bool WIDE>
void run_quantize(const QuantizeArgs& a, int rows, cudaStream_t s) {
    // the kernel, and how many of a row's vectors a thread has
    auto go = [&](void (*kernel)(QuantizeArgs), int vectors, int each) {
        const int threads = (ceil_div(vectors, each) + 31) / 32 * 32;
        QuantizeArgs with = a;
        with.clear_step = std::min(rows, CLEARING) * threads;
        launch_on(kernel, rows, threads, 0, s, 1, true, with);
    };
    const int vectors = ceil_div(a.K, 8);
    if (rows <= 2 * runtime().num_sms) {
        // few rows: a row's own time counts, and the fewer vectors a thread has the shorter it is (60 x 16384: 4.2 us with eight on 256 threads, 2.9
        // with two on 1024)
        if (vectors <= 1024) go(quantize_kernel<SRC, 1, WIDE>, vectors, 1);
        else if (vectors <= 2048) go(quantize_kernel<SRC, 2, WIDE>, vectors, 2);
        else go(quantize_kernel<SRC, 0, WIDE>, 256, 1);
        return;
    }
    // Many rows: several CTAs beside one another on an SM; where they come in more than eight rounds, fewer threads with more vectors each (4096 rows of 4096: four
    // vectors 9.1 us, two 10.0; of 2048: two 5.5, one 6.2; but 400 of 4096: four 2.6, two 2.2).  With a product of 64 columns behind them: 4096 rows of 4096 behind
    // a norm four 23.1, two 25.2; 2000 of 1536 two 11.6, one 10.8; and element by element the fewest (2000 rows of 5121 behind a residual sum and a norm:
    // two 44.8, four 52.2).
    const bool rounds = rows > 8 * runtime().num_sms;
    if (vectors > 2048) {
        go(quantize_kernel<SRC, 0, WIDE>, 256, 1);
    } else if (vectors > 1024) {
        if constexpr (SRC == SRC_PLAIN) go(quantize_kernel<SRC, 8, WIDE>, vectors, 8);
        else go(quantize_kernel<SRC, 4, WIDE>, vectors, 4);
    } else if constexpr (WIDE) {
        if (vectors > (rounds ? 256 : 512)) go(quantize_kernel<SRC, 4, WIDE>, vectors, 4);
        else if (vectors > (SRC == SRC_PLAIN && rounds ? 128 : 256)) go(quantize_kernel<SRC, 2, WIDE>, vectors, 2);
        else go(quantize_kernel<SRC, 1, WIDE>, vectors, 1);
    } else {
        if (vectors > 512) go(quantize_kernel<SRC, 2, WIDE>, vectors, 2);
        else go(quantize_kernel<SRC, 1, WIDE>, vectors, 1);
    }
}
template <Source SRC>
void run_quantize(const QuantizeArgs& a, int rows, bool wide, cudaStream_t s) {
    if (wide) run_quantize<SRC, true>(a, rows, s);
    else run_quantize<SRC, false>(a, rows, s);
}

// one thread per 16 bytes of the packed blocks; R rows of a role per tile
__global__ void pack_kernel(const int8_t* __restrict__ q, const float* __restrict__ scale, int N, int K, int role, int kblocks, bool vec,
                            uint8_t* __restrict__ blocks, float* __restrict__ scales, size_t chunks) {
    const int R = role == ROLE_PLAIN ? TILE_ROWS : TILE_ROWS / 2;
    const size_t per_row = static_cast<size_t>(kblocks) * (BLOCK_COLS / 16);
    for (size_t i = static_cast<size_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < chunks; i += static_cast<size_t>(gridDim.x) * blockDim.x) {
        const int r = static_cast<int>(i / per_row), c = static_cast<int>(i - r * per_row) * 16;
        const int tile = r / R, slot = r % R + (role == ROLE_UP ? R : 0);
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (r < N && c < K) {
            const int8_t* src = q + static_cast<size_t>(r) * K + c;
            if (vec) {
                v = *reinterpret_cast<const uint4*>(src);
            } else {
                uint32_t w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    auto at = [&](int k) { return c + k < K ? static_cast<int>(src[k]) : 0; };
                    w[j] = RowRound::low_bytes(at(4 * j), at(4 * j + 1), at(4 * j + 2), at(4 * j + 3));
                }
                v = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
        *reinterpret_cast<uint4*>(blocks + (static_cast<size_t>(tile) * kblocks + c / BLOCK_COLS) * BLOCK_BYTES + slot * BLOCK_COLS + c % BLOCK_COLS) = v;
        if (c == 0) scales[tile * TILE_ROWS + slot] = r < N ? scale[r] : 0.f;
    }
    __threadfence();   // in L2 before this CTA ends, which may be when the next launch fetches its first weights
}

}  // namespace

size_t packed_bytes(int N, int K, bool gated) {
    const size_t tiles = tiles_of(N, gated);
    return tiles * (pad_cols(K) / BLOCK_COLS) * BLOCK_BYTES + tiles * TILE_ROWS * sizeof(float);
}

Packed packed_view(const void* p, int N, int K, bool gated) {
    Packed w;
    w.tiles = tiles_of(N, gated);
    w.kblocks = pad_cols(K) / BLOCK_COLS;
    w.blocks = static_cast<const uint8_t*>(p);
    w.scales = reinterpret_cast<const float*>(w.blocks + static_cast<size_t>(w.tiles) * w.kblocks * BLOCK_BYTES);
    return w;
}

void launch_pack(const int8_t* q, const float* scale, int N, int K, Role role, void* packed, cudaStream_t s) {
    const bool gated = role != ROLE_PLAIN;
    const Packed w = packed_view(packed, N, K, gated);
    const size_t chunks = static_cast<size_t>(w.tiles) * (gated ? TILE_ROWS / 2 : TILE_ROWS) * w.kblocks * (BLOCK_COLS / 16);
    const bool vec = K % 16 == 0 && (reinterpret_cast<uintptr_t>(q) & 15) == 0;
    const size_t want = (chunks + 255) / 256;
    // not programmatic, and the kernel lets no successor start early (w8a8.cuh)
    launch_on(pack_kernel, static_cast<int>(want < 148 * 32 ? want : 148 * 32), 256, 0, s, 1, false, q, scale, N, K, static_cast<int>(role), w.kblocks, vec,
           const_cast<uint8_t*>(w.blocks), const_cast<float*>(w.scales), chunks);
}

void launch_quantize(const RowSource& src, int rows, int K, int8_t* q, long long ldq, int pad_to, float* scale, int* clear, int n_clear, cudaStream_t s) {
    if (rows <= 0) return;
    QuantizeArgs a;
    a.src = src;
    a.K = K; a.pad_to = pad_to;
    a.q = q; a.ldq = ldq;
    a.scale = scale;
    a.clear = clear; a.n_clear = n_clear;
    a.q_wide = (reinterpret_cast<uintptr_t>(q) & 7) == 0 && ldq % 8 == 0;
    const bool wide = rows_in_vectors(src, K) && a.q_wide;
    if (src.x32 != nullptr) run_quantize<SRC_F32, true>(a, rows, s);
    else if (src.norm == nullptr) run_quantize<SRC_PLAIN>(a, rows, wide, s);
    else if (src.delta == nullptr) run_quantize<SRC_NORM>(a, rows, wide, s);
    else run_quantize<SRC_ADD_NORM>(a, rows, wide, s);
}

}  // namespace w8
