// One row of an 8-bit linear layer, sm_100a:  y[N] = (q . W_n) * scale * scale_n + bias_n, with q made of the row inside the launch (w8a8_rows.cuh).
//
// Bound: the weights' bytes from HBM.  One CTA of 16 warps per SM makes the integers of the row once, in shared memory.  Weights come through
// asynchronous 16-byte copies into slots of shared memory that one lane writes and reads (no barriers): 96 or 128 KB per SM are in flight, the
// first of them before the wait for the predecessor and while the integers are made, and no registers hold them, so that the next launch's CTAs fit
// beside this one's and its weights are on their way before this one ends.  Eight lanes read 128 consecutive bytes of one weight row, a
// warp four rows (512 bytes) per k-block; S warps share the k-blocks of a group of rows and meet in shared memory, S chosen so
// that the groups divide evenly among the SMs.  dp4a sums four products: 4 of them per 16 bytes, far below what the lanes can do at
// the HBM rate.
// Back to back, weights from HBM: 4096 x 4096 4.8 us (3.5 TB/s), 16384 x 4096 13.2 (5.1), gate/up 4096 x 2 * 16384 21.5 (6.2).
#include <algorithm>

#include "ptx.cuh"
#include "w8a8_rows.cuh"

namespace w8 {
namespace {

constexpr int WARPS = 16, THREADS = WARPS * 32;
constexpr int MAX_STEP = 2;                           // k-blocks per step: 2, of gate/up pairs 1
// 16-byte copies per lane in flight.  Twelve, so that the next launch's CTA fits beside this one's; or, where the SM's share of the weights is more
// than sixteen hold, sixteen and the SM alone: (1 x 4096 x 4096, 1 x 16384 x 4096, 1 x 4096 x 32768) 4.84, 14.5, 23.1 us with twelve, 5.61, 13.2,
// 21.5 with sixteen; twenty and more gain nothing.
template <bool DEEP>
constexpr int SLOTS = DEEP ? 16 : 12;
template <bool DEEP>
constexpr int RING_BYTES = SLOTS<DEEP> * THREADS * 16;
constexpr int MAX_DYNAMIC_SMEM = 232448 - 2048;       // the static arrays are smaller than that

struct OneRowArgs {
    RowSource src;
    Packed w;
    int N, K, share, units, rounds;   // share: warps per group of rows; units: groups of 4 (gated: 4 + 4) rows
    int steps;                        // of a warp in a round
    const bf16* bias;
    bf16* y;
    float* act;
};

__device__ __forceinline__ int dot16(const uint4& a, const uint4& b, int acc) {
    acc = __dp4a(static_cast<int>(a.x), static_cast<int>(b.x), acc);
    acc = __dp4a(static_cast<int>(a.y), static_cast<int>(b.y), acc);
    acc = __dp4a(static_cast<int>(a.z), static_cast<int>(b.z), acc);
    return __dp4a(static_cast<int>(a.w), static_cast<int>(b.w), acc);
}

// Lets its successor start behind its own wait, so that the successor's weights are older than this launch's predecessor.
template <Source SRC, bool WIDE, bool GATED, bool DEEP>
__global__ void __launch_bounds__(THREADS, DEEP ? 1 : 2) one_row_s8_kernel(const OneRowArgs a) {
    constexpr int SETS = GATED ? 2 : 1;               // gate and up rows of the same features
    constexpr int STEP = MAX_STEP / SETS, PER_STEP = STEP * SETS, DEPTH = SLOTS<DEEP> / PER_STEP;   // copies of a lane; steps in flight
    constexpr int KEEP = HAS_NORM<SRC> ? 2 : 4;       // vectors that a thread keeps of the row
    constexpr int TILE_UNITS = (GATED ? TILE_ROWS / 2 : TILE_ROWS) / 4;
    extern __shared__ __align__(16) uint8_t smem[];   // ring, then the integers
    __shared__ uint32_t sh_top[32];
    __shared__ float sh_sum[32];
    __shared__ int part[2][WARPS][4 * SETS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int slots = WARPS / a.share, slot = warp / a.share, ks = warp % a.share;
    const int kblocks = a.w.kblocks;
    uint4* ring = reinterpret_cast<uint4*>(smem) + threadIdx.x;

    // ---- copies: steps in the order of their use.  Every warp has the same number of them in every round; what a step has no weights for is zeros.
    auto unit_of = [&](int round) { return (blockIdx.x + round * gridDim.x) * slots + slot; };
    const size_t stride = static_cast<size_t>(a.share) * STEP * BLOCK_BYTES;
    int load_round = 0, load_step = 0, load_at = 0, load_kb = 0;
    const uint8_t* load_from = a.w.blocks;
    auto seek = [&]() {
        const int unit = unit_of(load_round);
        const bool there = load_round < a.rounds && unit < a.units;
        load_kb = there ? ks * STEP : kblocks;
        load_from = a.w.blocks;
        if (there) load_from += (static_cast<size_t>(unit / TILE_UNITS) * kblocks + load_kb) * BLOCK_BYTES + ((unit % TILE_UNITS) * 4 + (lane >> 3)) * BLOCK_COLS + (lane & 7) * 16;
    };
    auto issue = [&]() {
#pragma unroll
        for (int u = 0; u < STEP; ++u) {
            const int bytes = load_kb + u < kblocks ? 16 : 0;   // 0: nothing is read
#pragma unroll
            for (int g = 0; g < SETS; ++g) {
                ptx::cp_async16(ring + (load_at * PER_STEP + u * SETS + g) * THREADS, load_from + u * BLOCK_BYTES + g * (TILE_ROWS / 2) * BLOCK_COLS, bytes);
            }
        }
        ptx::cp_async_commit();
        load_kb += a.share * STEP;
        load_from += stride;
        load_at = load_at + 1 == DEPTH ? 0 : load_at + 1;
        if (++load_step == a.steps) {
            load_step = 0;
            ++load_round;
            seek();
        }
    };
    // the row's lines first: behind the weights' they would be late
    if (static_cast<int>(threadIdx.x) * 8 < a.K && threadIdx.x % 8 == 0) Values<SRC, WIDE>::ask(a.src, 0, a.K, threadIdx.x * 8);
    seek();
#pragma unroll 1
    for (int i = 0; i < DEPTH; ++i) issue();
    grid_dep_wait();
    grid_dep_trigger();

    // ---- the row's integers
    int8_t* q = reinterpret_cast<int8_t*>(smem + RING_BYTES<DEEP>);
    uint32_t top = 0u;
    float ss = 0.f;
    Values<SRC, WIDE> kept[KEEP];
#pragma unroll
    for (int j = 0; j < KEEP; ++j) {
        const int c = (threadIdx.x + j * THREADS) * 8;
        if (c < a.K) kept[j].fetch(a.src, 0, a.K, c);
    }
#pragma unroll
    for (int j = 0; j < KEEP; ++j) {
        const int c = (threadIdx.x + j * THREADS) * 8;
        if (c < a.K) {
            kept[j].combine(a.src, 0, a.K, c, blockIdx.x == 0, top, ss);
        }
    }
    for (int c = (threadIdx.x + KEEP * THREADS) * 8; c < a.K; c += THREADS * 8) {   // of longer rows: read again below
        Values<SRC, WIDE> r;
        r.fetch(a.src, 0, a.K, c);
        r.combine(a.src, 0, a.K, c, blockIdx.x == 0, top, ss);
    }
    top = block_max(top, sh_top);
    float factor = 1.f;
    if constexpr (HAS_NORM<SRC>) factor = 1.f / sqrtf(block_total(ss, sh_sum) / a.K + a.src.eps);
    const RowRound round8(top, HAS_NORM<SRC>, SRC != SRC_F32);
#pragma unroll
    for (int j = 0; j < KEEP; ++j) {
        const int c = (threadIdx.x + j * THREADS) * 8;
        if (c < a.K) {
            float v[8];
            kept[j].values(v);
            *reinterpret_cast<uint2*>(q + c) = ints_of<HAS_NORM<SRC>>(round8, v);
        }
    }
    for (int c = (threadIdx.x + KEEP * THREADS) * 8; c < a.K; c += THREADS * 8) {
        Values<SRC, WIDE> r;
        float v[8], squares = 0.f;
        uint32_t known = 0u;
        r.fetch(a.src, 0, a.K, c);
        r.combine(a.src, 0, a.K, c, false, known, squares);
        r.values(v);
        *reinterpret_cast<uint2*>(q + c) = ints_of<HAS_NORM<SRC>>(round8, v);
    }
    for (int c = a.K + threadIdx.x; c < (kblocks + STEP - 1) / STEP * STEP * BLOCK_COLS; c += THREADS) q[c] = 0;
    const float scale = RowRound::scale(top, factor);
    __syncthreads();

    // ---- products
    int at = 0;
    for (int round = 0; round < a.rounds; ++round) {
        const int unit = unit_of(round);
        const int tile = unit / TILE_UNITS, row = (unit % TILE_UNITS) * 4 + (lane >> 3);
        const int n = tile * (GATED ? TILE_ROWS / 2 : TILE_ROWS) + row;
        const bool writes = ks == 0 && (lane & 7) == 0 && unit < a.units && n < a.N;
        float ws = 0.f, ws_up = 0.f, bias = 0.f;
        if (writes) {   // here before the sums are
            ws = __ldcg(a.w.scales + tile * TILE_ROWS + row);
            if constexpr (GATED) ws_up = __ldcg(a.w.scales + tile * TILE_ROWS + row + TILE_ROWS / 2);
            else if (a.bias != nullptr) bias = __bfloat162float(a.bias[n]);
        }
        int acc[SETS];
#pragma unroll
        for (int g = 0; g < SETS; ++g) acc[g] = 0;
        const int8_t* x_at = q + ks * STEP * BLOCK_COLS + (lane & 7) * 16;
#pragma unroll 1
        for (int step = 0; step < a.steps; ++step) {
            ptx::cp_async_wait<DEPTH - 1>();
            // steps behind the last k-block have zeros for weights; what they find for x does not matter, but has to be there
            const bool inside = (step * a.share + ks) * STEP < kblocks;
            uint4 x[STEP], wv[PER_STEP];
#pragma unroll
            for (int u = 0; u < STEP; ++u) x[u] = *reinterpret_cast<const uint4*>((inside ? x_at : q) + u * BLOCK_COLS);
#pragma unroll
            for (int i = 0; i < PER_STEP; ++i) wv[i] = ring[(at * PER_STEP + i) * THREADS];
#pragma unroll
            for (int i = 0; i < PER_STEP; ++i) acc[i % SETS] = dot16(wv[i], x[i / SETS], acc[i % SETS]);
            x_at += a.share * STEP * BLOCK_COLS;
            at = at + 1 == DEPTH ? 0 : at + 1;
            issue();
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
            ptx::named_bar_sync(1 + slot, a.share * 32);   // the warps of one group: at most eight groups
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
        if (writes) {
            const float v = static_cast<float>(acc[0]) * scale;
            if constexpr (GATED) a.act[n] = silu(v * ws) * (static_cast<float>(acc[SETS - 1]) * scale * ws_up);
            else a.y[n] = __float2bfloat16(fmaf(v, ws, bias));
        }
    }
    ptx::cp_async_wait<0>();
}

template <Source SRC, bool WIDE, bool GATED, bool DEEP>
void run(const OneRowArgs& a, int grid, size_t ints, cudaStream_t s) {
    static const bool allowed = [] {   // the library runs on one device
        CUDA_CHECK(cudaFuncSetAttribute(one_row_s8_kernel<SRC, WIDE, GATED, DEEP>, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_DYNAMIC_SMEM));
        return true;
    }();
    (void)allowed;
    launch_on(one_row_s8_kernel<SRC, WIDE, GATED, DEEP>, grid, THREADS, RING_BYTES<DEEP> + ints, s, 1, true, a);
}
template <Source SRC, bool GATED>
void run(const OneRowArgs& a, int grid, size_t ints, bool wide, bool deep, cudaStream_t s) {
    if constexpr (SRC != SRC_F32) {   // activations come in whole vectors
        if (!wide) { run<SRC, false, GATED, false>(a, grid, ints, s); return; }
    }
    if (deep) run<SRC, true, GATED, true>(a, grid, ints, s);
    else run<SRC, true, GATED, false>(a, grid, ints, s);
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
    // Warps per group: the fewest steps of a warp, with half a step for each round's meeting
    const int sms = runtime().num_sms, step_blocks = gated ? 1 : MAX_STEP, all_steps = ceil_div(w.kblocks, step_blocks);
    long long best = -1;
    for (int share = 1; share <= WARPS; share *= 2) {
        const int rounds = ceil_div(ceil_div(a.units, WARPS / share), sms), steps = ceil_div(all_steps, share);
        const long long cost = static_cast<long long>(rounds) * (2 * steps + (share > 1 ? 1 : 0));
        if (best < 0 || cost < best) {
            best = cost;
            a.share = share;
            a.rounds = rounds;
            a.steps = steps;
        }
    }
    const int grid = std::min(sms, ceil_div(a.units, WARPS / a.share));
    const size_t ints = static_cast<size_t>(all_steps) * step_blocks * BLOCK_COLS;
    const bool wide = rows_in_vectors(src, K);
    const bool deep = static_cast<size_t>(w.tiles) * w.kblocks * BLOCK_BYTES > static_cast<size_t>(sms) * RING_BYTES<true> && RING_BYTES<true> + ints <= MAX_DYNAMIC_SMEM;
    if (src.x32 != nullptr) run<SRC_F32, false>(a, grid, ints, wide, deep, s);
    else if (src.norm == nullptr) gated ? run<SRC_PLAIN, true>(a, grid, ints, wide, deep, s) : run<SRC_PLAIN, false>(a, grid, ints, wide, deep, s);
    else if (src.delta == nullptr) gated ? run<SRC_NORM, true>(a, grid, ints, wide, deep, s) : run<SRC_NORM, false>(a, grid, ints, wide, deep, s);
    else gated ? run<SRC_ADD_NORM, true>(a, grid, ints, wide, deep, s) : run<SRC_ADD_NORM, false>(a, grid, ints, wide, deep, s);
}

}  // namespace w8
