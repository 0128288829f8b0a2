// One row of an 8-bit linear layer, sm_100a:  y[N] = (q . W_n) * scale * scale_n + bias_n, with q made of the row inside the launch (w8a8_rows.cuh).
//
// Bound: the weights' bytes from HBM.  One CTA of 32 warps per SM makes the integers of the row once, in shared memory; the weights of a warp's
// first batch, eight 16-byte loads a lane, are on their way meanwhile: 128 KB per SM, so that a product of up to 19 MB is in flight
// as a whole before its integers are there.  Eight lanes read 128 consecutive bytes of one weight row, a warp four rows (512 bytes) per
// k-block; S warps share the k-blocks of a group of rows and meet in shared memory, S chosen so that the groups divide evenly among the SMs.
// dp4a sums four products: 4 of them per 16 bytes, far below what the lanes can do at the HBM rate.
#include <algorithm>

#include "w8a8_rows.cuh"

namespace w8 {
namespace {

constexpr int WARPS = 32, THREADS = WARPS * 32;
constexpr int BATCH = 8;                              // 16-byte loads per lane in flight
constexpr int MAX_STAGE_BYTES = 200 * 1024;

struct OneRowArgs {
    RowSource src;
    Packed w;
    int N, K, share, units, rounds;   // share: warps per group of rows; units: groups of 4 (gated: 4 + 4) rows
    int staged;                       // the row's fp32 values fit beside its integers
    const bf16* bias;
    bf16* y;
    float* act;
};

// past the first-level cache, and kept in its place: before the wait (w8a8.cuh)
__device__ __forceinline__ uint4 load_weights(const uint8_t* p) {
    uint4 v;
    asm volatile("ld.global.cg.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ int dot16(const uint4& a, const uint4& b, int acc) {
    acc = __dp4a(static_cast<int>(a.x), static_cast<int>(b.x), acc);
    acc = __dp4a(static_cast<int>(a.y), static_cast<int>(b.y), acc);
    acc = __dp4a(static_cast<int>(a.z), static_cast<int>(b.z), acc);
    return __dp4a(static_cast<int>(a.w), static_cast<int>(b.w), acc);
}

// Lets its successor start behind its own wait, so that the successor's weights are older than this launch's predecessor.
template <Source SRC, int VEC, bool GATED>
__global__ void __launch_bounds__(THREADS, 1) one_row_s8_kernel(const OneRowArgs a) {
    constexpr int SETS = GATED ? 2 : 1;               // gate and up rows of the same features
    constexpr int KB = BATCH / SETS;                  // k-blocks per batch
    constexpr int TILE_UNITS = (GATED ? TILE_ROWS / 2 : TILE_ROWS) / 4;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ uint32_t sh_top[32];
    __shared__ float sh_sum[32];
    __shared__ int part[2][WARPS][4 * SETS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int slots = WARPS / a.share, slot = warp / a.share, ks = warp % a.share;
    const int kblocks = a.w.kblocks;
    const int batches = ceil_div_dev(ceil_div_dev(kblocks, a.share), KB);

    uint4 wv[KB][SETS];
    auto unit_of = [&](int round) { return (blockIdx.x + round * gridDim.x) * slots + slot; };
    auto load = [&](int round, int batch) {
        const int unit = unit_of(round);
        const uint8_t* base = a.w.blocks + static_cast<size_t>(unit / TILE_UNITS) * kblocks * BLOCK_BYTES +
                              ((unit % TILE_UNITS) * 4 + (lane >> 3)) * BLOCK_COLS + (lane & 7) * 16;
#pragma unroll
        for (int u = 0; u < KB; ++u) {
            const int kb = ks + a.share * (batch * KB + u);
#pragma unroll
            for (int g = 0; g < SETS; ++g) {
                wv[u][g] = unit < a.units && kb < kblocks ? load_weights(base + static_cast<size_t>(kb) * BLOCK_BYTES + g * (TILE_ROWS / 2) * BLOCK_COLS)
                                                          : make_uint4(0u, 0u, 0u, 0u);
            }
        }
    };
    load(0, 0);
    grid_dep_wait();
    grid_dep_trigger();

    // ---- the row's integers
    int8_t* q = reinterpret_cast<int8_t*>(smem);
    float* stage = reinterpret_cast<float*>(smem + kblocks * BLOCK_COLS);
    uint32_t top = 0u;
    float ss = 0.f;
    for (int c = threadIdx.x * VEC; c < a.K; c += THREADS * VEC) {
        Values<SRC, VEC> r;
        r.fetch(a.src, 0, a.K, c);
        r.combine(a.src, 0, a.K, c, ss, blockIdx.x == 0);
#pragma unroll
        for (int e = 0; e < VEC; ++e) top = max(top, magnitude(r.v[e]));
        if (a.staged) store_vec<VEC>(stage + c, r.v);
    }
    top = block_max(top, sh_top);
    float factor = 1.f;
    if constexpr (SRC == SRC_NORM || SRC == SRC_ADD_NORM) factor = 1.f / sqrtf(block_total(ss, sh_sum) / a.K + a.src.eps);
    const RowRound round8(top);
    for (int c = threadIdx.x * VEC; c < a.K; c += THREADS * VEC) {
        Values<SRC, VEC> r;
        if (a.staged) {
            load_vec<VEC>(stage + c, r.v);
        } else {
            float unused = 0.f;
            r.fetch(a.src, 0, a.K, c);
            r.combine(a.src, 0, a.K, c, unused, false);
        }
        store_ints<VEC>(q + c, round8, r.v);
    }
    for (int c = a.K + threadIdx.x; c < kblocks * BLOCK_COLS; c += THREADS) q[c] = 0;
    const float scale = RowRound::scale(top, factor);
    __syncthreads();

    // ---- products
    for (int round = 0; round < a.rounds; ++round) {
        int acc[SETS];
#pragma unroll
        for (int g = 0; g < SETS; ++g) acc[g] = 0;
        for (int batch = 0; batch < batches; ++batch) {
#pragma unroll
            for (int u = 0; u < KB; ++u) {
                const int kb = ks + a.share * (batch * KB + u);
                if (kb < kblocks) {
                    const uint4 x = *reinterpret_cast<const uint4*>(q + kb * BLOCK_COLS + (lane & 7) * 16);
#pragma unroll
                    for (int g = 0; g < SETS; ++g) acc[g] = dot16(wv[u][g], x, acc[g]);
                }
            }
            if (batch + 1 < batches) load(round, batch + 1);
            else if (round + 1 < a.rounds) load(round + 1, 0);
        }
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) {
#pragma unroll
            for (int g = 0; g < SETS; ++g) acc[g] += __shfl_xor_sync(0xffffffffu, acc[g], o);
        }
        if (a.share > 1) {
            if ((lane & 7) == 0) {
#pragma unroll
                for (int g = 0; g < SETS; ++g) part[round & 1][warp][g * 4 + (lane >> 3)] = acc[g];
            }
            // the warps of one group: at most eight groups
            asm volatile("bar.sync %0, %1;" ::"r"(1 + slot), "r"(a.share * 32) : "memory");
            if (ks == 0) {
#pragma unroll
                for (int g = 0; g < SETS; ++g) {
                    int sum = 0;
                    for (int w = lane & 7; w < a.share; w += 8) sum += part[round & 1][warp + w][g * 4 + (lane >> 3)];
#pragma unroll
                    for (int o = 4; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                    acc[g] = sum;
                }
            }
        }
        const int unit = unit_of(round);
        if (ks == 0 && (lane & 7) == 0 && unit < a.units) {
            const int tile = unit / TILE_UNITS, row = (unit % TILE_UNITS) * 4 + (lane >> 3);
            const int n = tile * (GATED ? TILE_ROWS / 2 : TILE_ROWS) + row;
            if (n < a.N) {
                const float* ws = a.w.scales + tile * TILE_ROWS + row;
                const float v = static_cast<float>(acc[0]) * scale * ws[0];
                if constexpr (GATED) {
                    a.act[n] = silu_f32(v) * (static_cast<float>(acc[SETS - 1]) * scale * ws[TILE_ROWS / 2]);
                } else {
                    a.y[n] = __float2bfloat16(v + (a.bias != nullptr ? __bfloat162float(a.bias[n]) : 0.f));
                }
            }
        }
    }
}

template <Source SRC, int VEC, bool GATED>
void run(const OneRowArgs& a, int grid, size_t smem, cudaStream_t s) {
    // the attribute belongs to the function on this device; setting it again costs a fraction of a launch and needs no flag that threads share
    CUDA_CHECK(cudaFuncSetAttribute(one_row_s8_kernel<SRC, VEC, GATED>, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_STAGE_BYTES));
    launch(one_row_s8_kernel<SRC, VEC, GATED>, grid, THREADS, smem, s, 1, true, a);
}
template <Source SRC, bool GATED>
void run(const OneRowArgs& a, int grid, size_t smem, bool vec, cudaStream_t s) {
    if (vec) run<SRC, 8, GATED>(a, grid, smem, s);
    else run<SRC, 1, GATED>(a, grid, smem, s);
}

}  // namespace

void launch_one_row(const RowSource& src, int N, int K, const Packed& w, const bf16* bias, bf16* y, float* act, cudaStream_t s) {
    const bool gated = act != nullptr;
    OneRowArgs a;
    a.src = src;
    a.w = w;
    a.N = N; a.K = K;
    a.bias = bias; a.y = y; a.act = act;
    a.units = w.tiles * (gated ? 16 : 32);
    // Warps per group: the fewest rounds times batches, the fewest warps of those (a shared group costs a barrier a round)
    const int sms = runtime().num_sms, per_batch = gated ? BATCH / 2 : BATCH;
    long long best = -1;
    for (int share = 1; share <= WARPS; share *= (share == 1 ? 4 : 2)) {
        const int slots = WARPS / share;
        const int rounds = ceil_div(ceil_div(a.units, slots), sms);
        const long long cost = static_cast<long long>(rounds) * ceil_div(ceil_div(w.kblocks, share), per_batch);
        if (best < 0 || cost < best) {
            best = cost;
            a.share = share;
            a.rounds = rounds;
        }
    }
    const int grid = std::min(sms, ceil_div(a.units, WARPS / a.share));
    const size_t ints = static_cast<size_t>(w.kblocks) * BLOCK_COLS, floats = (static_cast<size_t>(K) + 7) / 8 * 32;
    a.staged = ints + floats <= static_cast<size_t>(MAX_STAGE_BYTES);
    const size_t smem = ints + (a.staged ? floats : 0);
    const bool vec = rows_in_vectors(src, K);
    if (src.x32 != nullptr) run<SRC_F32, false>(a, grid, smem, vec, s);
    else if (src.norm == nullptr) gated ? run<SRC_PLAIN, true>(a, grid, smem, vec, s) : run<SRC_PLAIN, false>(a, grid, smem, vec, s);
    else if (src.delta == nullptr) gated ? run<SRC_NORM, true>(a, grid, smem, vec, s) : run<SRC_NORM, false>(a, grid, smem, vec, s);
    else gated ? run<SRC_ADD_NORM, true>(a, grid, smem, vec, s) : run<SRC_ADD_NORM, false>(a, grid, smem, vec, s);
}

}  // namespace w8
