// Products of 8-bit integers, sm_100a:  Y[M,N] = (Q[M,K] W[N,K]^T) * xs[m] * ws[n] (+ bias[n]), int8 in, int32 sums in tensor memory, bf16 out; with
// gate/up weights silu(gate) * up in fp32 instead.
//
// Operand mapping as for the bf16 products (gemm_umma.cu): weights are the A operand (128 rows of a tile), token rows the B operand, the
// accumulator is Y^T.  A k-block is 128 integers, one 128-byte swizzle row, so a stage has the bytes of a bf16 stage and twice the products.
//   few tiles   clusters of 2 to 8 CTAs that cut a tile's k-blocks evenly and sum it in distributed shared memory, token tiles of 16 to 128
//   more        token tiles of 16 to 256 on single CTAs, or pairs of CTAs on tiles of 256 x 256 (tcgen05 cta_group::2: half of the operand bytes per
//               product); whole tiles in waves, and only those of the last wave are cut (stream-K), where that pays
// whichever find_division() expects to end first.
// Bound: the weights' bytes from HBM up to some 300 rows, the tensor pipe (and, with warm passes, the power cap) beyond.  60 x 16384 x 4096 14.2 us
// (5.8 TB/s between the first block and the last: 50 MB, 17 are asked for before), 4096 x 16384 x 4096 174 us (3.16 Pop/s), gate/up 4096 x 4096 x 2 * 16384
// 325 us (3.39, tensor pipe 91 % active).
//
// Cut tiles: each piece leaves its int32 sums in a workspace slot, and the one counted last adds them up.  Integer sums have no order, so the
// result does not depend on who is last, and no CTA waits for another one: the launch need not be resident as a whole, and may share the
// device with launches of other streams.  (Clusters are resident as a whole by definition.)
#include <algorithm>

#include "gemm_common.cuh"
#include "op_errors.cuh"
#include "row_ops.cuh"
#include "w8a8.cuh"

using gemm::SegIter;

namespace w8 {
namespace {

constexpr int UMMA_K = 32;
// Warp 0 TMA, warp 1 MMA + TMEM, then the epilogue: on each quarter of the tensor memory's lanes up to two warps, which take turns with batches of 16
// tokens.  (One alone waits for its own instructions most of the time: a gate/up tile of 256 tokens took 27000 cycles beside 16400 of products at
// K = 4096.  Four: 4096 x 128 x 4096 21.7 us, two 22.0; 60 x 128 x 38000 6.4, two 6.1.)
constexpr int BATCH = 16, MAX_PARTS = 2;
constexpr int EPI_BUF_BYTES = 1024;    // a warp's own: 16 tokens of 32 features in bf16, or 8 in 32 bits
constexpr int CLUSTER_THREADS = 192;   // of the cluster kernel, whose epilogue is short
constexpr int CTRL_BYTES = 256;

struct ProductArgs {
    gemm::LinearArgs sched;        // shape, raster and division of the work only
    int N;                         // output features
    const float *xs, *ws;
    const bf16* bias;
    bf16* y;
    long long ldy;
    float* act;
    int* partials;
    int* tickets;
    OpCount* errors;
};

// kind::i8, both operands signed, K-major, int32 accumulator: bits [4,6) D (2 = s32), [7,10) A (1 = s8), [10,13) B, [17,23) N>>3, [24,29) M>>4
__host__ __device__ constexpr uint32_t idesc_s8(int m, int n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}
template <bool PAIR>
__device__ __forceinline__ void umma_s8(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (PAIR) {
        asm volatile(
            "{\n\t"
            ".reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t"
            "}\n" ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
    } else {
        asm volatile(
            "{\n\t"
            ".reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t"
            "}\n" ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
    }
}
// one k-block
template <bool PAIR>
__device__ __forceinline__ void umma_block(uint32_t d, uint32_t wa, uint32_t xa, uint32_t idesc, bool first) {
#pragma unroll
    for (int j = 0; j < BLOCK_COLS / UMMA_K; ++j) {
        umma_s8<PAIR>(d, ptx::umma_desc_sw128(wa + j * UMMA_K, 16, 1024), ptx::umma_desc_sw128(xa + j * UMMA_K, 16, 1024), idesc, (!first || j > 0) ? 1u : 0u);
    }
}

// The end of a CTA, thread 0: a wait that ran out is reported, and copies still in flight, which arrive at this CTA's barriers, land before it retires.  (A partner's
// copies too: where a CTA's own waits all ended, the bytes of both have come.)
__device__ __forceinline__ void finish(volatile int* abort_flag, OpCount* errors) {
    if (*abort_flag == 0) return;
    report(errors, OP_TIMEOUT);
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000LL) {}
}

template <int MT>
constexpr int PARTS_OF = MT / BATCH < MAX_PARTS ? MT / BATCH : MAX_PARTS;   // epilogue warps on a quarter
template <int MT, bool PAIR>
struct Cfg {
    static constexpr int X_ROWS = PAIR ? MT / 2 : MT;           // token rows that this CTA loads
    static constexpr int STAGE_BYTES = BLOCK_BYTES + X_ROWS * BLOCK_COLS;
    static constexpr int STAGES = PAIR ? 6 : (MT <= 16) ? 10 : (MT <= 32) ? 9 : (MT <= 64) ? 8 : (MT <= 128) ? 6 : 4;
    static constexpr int TMEM_COLS = 2 * MT;
    static constexpr int PARTS = PARTS_OF<MT>, EPI_WARPS = 4 * PARTS, THREADS = 64 + EPI_WARPS * 32;
    static constexpr int TURNS = MT / (BATCH * PARTS);          // batches of an epilogue warp
    static constexpr int XCH_BYTES = EPI_WARPS * EPI_BUF_BYTES;
    static constexpr int SCALE_BYTES = EPI_WARPS * TURNS * BATCH * 4;   // per epilogue warp the scales of its tokens
    static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + CTRL_BYTES + XCH_BYTES + SCALE_BYTES + 1024;
    static_assert(SMEM_BYTES <= 232448, "shared memory budget");
};

// 16 sums of feature `lane` of this warp, tokens c0 .. c0 + 15, times the scales
__device__ __forceinline__ void scale16(const int (&r)[16], const float* xs, float ws, float bias, float (&v)[16]) {
#pragma unroll
    for (int c = 0; c < 16; c += 4) {
        const float4 s = *reinterpret_cast<const float4*>(xs + c);
        v[c] = fmaf(static_cast<float>(r[c]) * s.x, ws, bias);
        v[c + 1] = fmaf(static_cast<float>(r[c + 1]) * s.y, ws, bias);
        v[c + 2] = fmaf(static_cast<float>(r[c + 2]) * s.z, ws, bias);
        v[c + 3] = fmaf(static_cast<float>(r[c + 3]) * s.w, ws, bias);
    }
}

__device__ __forceinline__ void load16(uint32_t taddr, int (&r)[16]) {
    ptx::tmem_ld16(taddr, reinterpret_cast<uint32_t*>(r));
}

// 16 tokens' values of 32 features to rows of y, ldy apart (64 bits).  A lane has one feature: through `buf` eight features are one 16-byte store, where
// rows and widths allow that (vec).
__device__ __forceinline__ void store16(bf16* y, long long ldy, int N, long long y_row, int cnt, int n0, const float (&v)[16], uint8_t* buf, int lane, bool vec) {
    bf16* to = y + y_row * ldy;
    if (vec) {
        uint16_t* b = reinterpret_cast<uint16_t*>(buf);
        __syncwarp();   // the buffer's earlier contents have been read
#pragma unroll
        for (int c = 0; c < 16; c += 2) {
            const uint32_t two = two_bf16(v[c], v[c + 1]);
            b[c * 32 + lane] = static_cast<uint16_t>(two);
            b[(c + 1) * 32 + lane] = static_cast<uint16_t>(two >> 16);
        }
        __syncwarp();
        const int f = n0 + (lane & 3) * 8;
#pragma unroll
        for (int k = 0; k < 16; k += 8) {
            const int c = k + (lane >> 2);
            const uint4 w = *reinterpret_cast<const uint4*>(buf + c * 64 + (lane & 3) * 16);
            if (c < cnt && f < N) *reinterpret_cast<uint4*>(to + c * ldy + f) = w;
        }
    } else if (n0 + lane < N) {
#pragma unroll
        for (int c = 0; c < 16; ++c) {
            if (c < cnt) to[c * ldy + n0 + lane] = __float2bfloat16(v[c]);
        }
    }
}

// silu(gate) * up of a whole tile: lanes 0-63 hold the gate sums of 64 features, 64-127 the up sums of the same ones.  Warps q and q + 2 hand
// each other the sums of half of the tokens of a batch, so that both compute.  fp32: what is rounded next is the row of 8-bit integers.
// xs: the scales of this warp's batches, one after another.
template <int MT>
__device__ __forceinline__ void gate_tile(uint32_t t_addr, int m_cnt, float* act, long long ld, int N, long long row0, int n0, const float* xs, float ws_gate,
                                          float ws_up, uint8_t* xch, int q, int part, int lane) {
    constexpr int HB = BATCH / 2, PARTS = PARTS_OF<MT>;
    int* out = reinterpret_cast<int*>(xch + (part * 4 + q) * EPI_BUF_BYTES) + lane;
    const int* in = reinterpret_cast<const int*>(xch + (part * 4 + (q ^ 2)) * EPI_BUF_BYTES) + lane;
    const int pair_bar = 2 + part * 2 + (q & 1);
    const bool gates = q < 2;
    const bool column = n0 + lane < N;
    xs += gates ? 0 : HB;
#pragma unroll 1
    for (int c0 = part * BATCH; c0 < m_cnt; c0 += PARTS * BATCH, xs += BATCH) {   // the same in both warps
        uint32_t r[BATCH];
        ptx::tmem_ld16(t_addr + c0, r);
        ptx::tmem_wait_ld();
        // gate warps keep the first half of the tokens, up warps the second
#pragma unroll
        for (int c = 0; c < HB; ++c) out[c * 32] = static_cast<int>(gates ? r[HB + c] : r[c]);
        ptx::named_bar_sync(pair_bar, 64);
        const int first = c0 + (gates ? 0 : HB);
        float v[HB], gate[HB], up[HB], least = 0.f;
#pragma unroll
        for (int c = 0; c < HB; c += 4) {
            const float4 s4 = *reinterpret_cast<const float4*>(xs + c);
            const float s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int mine = static_cast<int>(gates ? r[c + e] : r[HB + c + e]), other = in[(c + e) * 32];
                gate[c + e] = static_cast<float>(gates ? mine : other) * s[e] * ws_gate;
                up[c + e] = static_cast<float>(gates ? other : mine) * s[e] * ws_up;
                v[c + e] = silu_above(gate[c + e]) * up[c + e];
                least = fminf(least, gate[c + e]);
            }
        }
        if (least <= SILU_LEAST) {
#pragma unroll
            for (int c = 0; c < HB; ++c) v[c] = silu(gate[c]) * up[c];
        }
        float* dst = act + (row0 + first) * ld + n0 + lane;
        if (column) {
#pragma unroll
            for (int c = 0; c < HB; ++c, dst += ld) {
                if (first + c < m_cnt) *dst = v[c];
            }
        }
        ptx::named_bar_sync(pair_bar, 64);   // the partner may write `in` again
    }
}

// The epilogue threads of one CTA walk the segments of `it`; rank: of a pair's CTA, which has 128 of the tile's 256 weight rows.
template <int MT, bool PAIR>
__device__ __forceinline__ void epilogue(const ProductArgs& a, SegIter it, uint32_t tmem_base, uint64_t* acc_full, uint64_t* acc_empty,
                                         volatile int* abort_flag, volatile int* s_last, int warp, int lane, int epi_tid, int g, int G, uint8_t* xch,
                                         float* scales, int rank) {
    using C = Cfg<MT, PAIR>;
    constexpr int CSZ = PAIR ? 2 : 1, STEP = C::PARTS * BATCH, MINE = C::TURNS * BATCH;   // tokens of this warp
    const gemm::LinearArgs& w = a.sched;
    const int q = warp & 3, row = q * 32 + lane, part = (warp - 2) >> 2;
    uint8_t* buf = xch + (part * 4 + q) * EPI_BUF_BYTES;
    float* xs = scales + (part * 4 + q) * MINE;
    const bool vec = a.act == nullptr && ((reinterpret_cast<uintptr_t>(a.y) | (static_cast<uintptr_t>(a.ldy) * 2) | (static_cast<uintptr_t>(a.N) * 2)) & 15) == 0;
    const int gt = w.tail_grid > 0 ? w.tail_grid : G;
    int acc = 0;
    uint32_t acc_phase = 0;
    // A tile's scales (and bias) are asked for while the tile before it is on its way out (4096 x 128 x 4096: 26.4 -> 22.0 us).
    struct Ahead {
        int tile, kb0, kb1, m_base, n_tile;
        float xs[(MINE + 31) / 32], ws, ws_up, bias;
    };
    auto look = [&](Ahead& t) {
        if (!it.next(t.tile, t.kb0, t.kb1)) return false;
        int m_tile, n_tile;
        gemm::tile_to_mn(w, t.tile, m_tile, n_tile);
        t.n_tile = n_tile * CSZ + rank;
        t.m_base = m_tile * MT;
#pragma unroll
        for (int i = 0; i < (MINE + 31) / 32; ++i) {
            const int l = lane + i * 32, m = t.m_base + l / BATCH * STEP + part * BATCH + l % BATCH;
            t.xs[i] = l < MINE && m < w.M ? a.xs[m] : 0.f;
        }
        const int n = t.n_tile * TILE_ROWS + row;
        t.ws = a.ws[a.act == nullptr ? n : t.n_tile * TILE_ROWS + (row & 63)];                       // gate/up tiles: of the gate
        t.ws_up = a.act == nullptr ? 0.f : a.ws[t.n_tile * TILE_ROWS + 64 + (row & 63)];
        t.bias = a.act == nullptr && a.bias != nullptr && n < a.N ? __bfloat162float(a.bias[n]) : 0.f;
        return true;
    };
    Ahead next;
    bool more = look(next);
    while (more) {
        const int tile = next.tile, kb0 = next.kb0, kb1 = next.kb1, m_base = next.m_base, n_tile = next.n_tile;
        const int m_cnt = min(w.M - m_base, MT);
        const float ws = next.ws, ws_up = next.ws_up, bias = next.bias;
        __syncwarp();   // the tile before has done with the scales
#pragma unroll
        for (int i = 0; i < (MINE + 31) / 32; ++i) {
            if (lane + i * 32 < MINE) xs[lane + i * 32] = next.xs[i];
        }
        __syncwarp();
        more = look(next);
        // A wait that ran out (the launch reports it) does not end the walk: the warps meet at barriers further down, and must all come to each of them.
        ptx::mbar_wait_warp(&acc_full[acc], acc_phase, abort_flag);
        ptx::tc_fence_after();
        const uint32_t t_addr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + acc * MT;
        const int n0 = n_tile * TILE_ROWS + q * 32;
        int* const slot = a.partials + (static_cast<size_t>(g * CSZ + rank) * 2 + (kb0 == 0 ? 1 : 0)) * (MT * TILE_ROWS);
        const bool whole = kb0 == 0 && kb1 == w.kblocks;
        int first = 0, pieces = 1;
        if (!whole) {
            const long long u0 = static_cast<long long>(tile - w.wave_tiles) * w.kblocks;
            first = gemm::unit_owner(u0, w.total_units, gt);
            pieces = gemm::unit_owner(u0 + w.kblocks - 1, w.total_units, gt) - first + 1;
        }
        if (a.act != nullptr) {
            gate_tile<MT>(t_addr, m_cnt, a.act, a.ldy, a.N, m_base, n_tile * 64 + (q & 1) * 32, xs, ws, ws_up, xch, q, part, lane);
        } else if (whole) {
            const float* s = xs;
#pragma unroll 1
            for (int c0 = part * BATCH; c0 < m_cnt; c0 += STEP, s += BATCH) {
                int r[16];
                float v[16];
                load16(t_addr + c0, r);
                ptx::tmem_wait_ld();
                scale16(r, s, ws, bias, v);
                store16(a.y, a.ldy, a.N, m_base + c0, m_cnt - c0, n0, v, buf, lane, vec);
            }
        } else {
#pragma unroll 1
            for (int c0 = part * BATCH; c0 < m_cnt; c0 += STEP) {
                int r[16];
                load16(t_addr + c0, r);
                ptx::tmem_wait_ld();
#pragma unroll
                for (int c = 0; c < 16; ++c) {
                    if (c0 + c < m_cnt) __stcg(slot + (c0 + c) * TILE_ROWS + row, r[c]);
                }
            }
        }
        ptx::tc_fence_before();
        if constexpr (PAIR) ptx::mbar_arrive_cluster(ptx::cluster_map(ptx::smem_u32(&acc_empty[acc]), 0));
        else ptx::mbar_arrive(&acc_empty[acc]);
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1;

        if (!whole) {
            __threadfence();   // this thread's sums are visible before the count
            ptx::named_bar_sync(1, C::EPI_WARPS * 32);
            if (epi_tid == 0) *s_last = atomicAdd(&a.tickets[tile * CSZ + rank], 1) == pieces - 1;
            ptx::named_bar_sync(1, C::EPI_WARPS * 32);
            const bool last = *s_last != 0;
            ptx::named_bar_sync(1, C::EPI_WARPS * 32);   // everyone has read s_last before it can change
            if (last) {
                __threadfence();
                const float* sc = xs;
#pragma unroll 1
                for (int c0 = part * BATCH; c0 < m_cnt; c0 += STEP, sc += BATCH) {
                    int sum[16];
#pragma unroll
                    for (int c = 0; c < 16; ++c) sum[c] = 0;
#pragma unroll 1
                    for (int p0 = 0; p0 < pieces; p0 += 2) {
                        int r[2][16];
#pragma unroll
                        for (int s = 0; s < 2; ++s) {
                            const int gg = first + p0 + s;
                            const int* from = a.partials + (static_cast<size_t>(gg * CSZ + rank) * 2 + (gg == first ? 1 : 0)) * (MT * TILE_ROWS) + c0 * TILE_ROWS + row;
#pragma unroll
                            for (int c = 0; c < 16; ++c) r[s][c] = p0 + s < pieces && c0 + c < m_cnt ? __ldcg(from + c * TILE_ROWS) : 0;
                        }
#pragma unroll
                        for (int s = 0; s < 2; ++s) {
#pragma unroll
                            for (int c = 0; c < 16; ++c) sum[c] += r[s][c];
                        }
                    }
                    float v[16];
                    scale16(sum, sc, ws, bias, v);
                    store16(a.y, a.ldy, a.N, m_base + c0, m_cnt - c0, n0, v, buf, lane, vec);
                }
            }
        }
    }
}

// Lets its successor start at once: what a successor fetches before its own wait are packed weights only.
template <int MT, bool PAIR>
__global__ void __launch_bounds__(Cfg<MT, PAIR>::THREADS, 1)
product_s8_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, const ProductArgs a) {
    using C = Cfg<MT, PAIR>;
    constexpr int CSZ = PAIR ? 2 : 1;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::STAGES * C::STAGE_BYTES);   // pairs: rank 0's count both CTAs' copies
    uint64_t* empty = full + C::STAGES;
    uint64_t* acc_full = empty + C::STAGES;
    uint64_t* acc_empty = acc_full + 2;                                                // pairs: rank 0's
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile int* s_last = abort_flag + 1;
    uint8_t* xch = smem + C::STAGES * C::STAGE_BYTES + CTRL_BYTES;
    float* scales = reinterpret_cast<float*>(xch + C::XCH_BYTES);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = PAIR ? static_cast<int>(ptx::cluster_ctarank()) : 0;
    const int G = gridDim.x / CSZ, g = blockIdx.x / CSZ;
    const gemm::LinearArgs& sched = a.sched;
    grid_dep_trigger();

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; ++s) {
            ptx::mbar_init(&full[s], 1);
            ptx::mbar_init(&empty[s], 1);
        }
        for (int s = 0; s < 2; ++s) {
            ptx::mbar_init(&acc_full[s], 1);
            ptx::mbar_init(&acc_empty[s], CSZ * C::EPI_WARPS * 32);
        }
        *abort_flag = 0;
        *s_last = 0;
        ptx::mbar_fence_init();
        ptx::prefetch_tensormap(&tm_w);
        ptx::prefetch_tensormap(&tm_x);
    }
    if (warp == 1) {
        if constexpr (PAIR) {
            ptx::tmem_alloc_pair(tmem_slot, C::TMEM_COLS);
        } else {
            ptx::tmem_alloc(tmem_slot, C::TMEM_COLS);
            ptx::tmem_relinquish();
        }
    }
    ptx::tc_fence_before();
    __syncthreads();
    if constexpr (PAIR) ptx::cluster_sync();   // both CTAs' barriers are there before either copies or arrives
    ptx::tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    SegIter it = gemm::make_seg_iter(sched, g, G);
    if (warp != 0) grid_dep_wait();

    if (warp == 0) {
        // ------------------------------------------------ TMA producer
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            int tile, kb0, kb1;
            bool ok = true;
            auto load_w = [&](int s, int kb, int n_tile) {
                uint8_t* dst = smem + s * C::STAGE_BYTES;
                const int y = ((CSZ * n_tile + rank) * sched.kblocks + kb) * TILE_ROWS;
                if (rank == 0) ptx::mbar_arrive_expect_tx(&full[s], CSZ * C::STAGE_BYTES);
                if constexpr (PAIR) ptx::tma_load_2d_pair(dst, &tm_w, ptx::cluster_map(ptx::smem_u32(&full[s]), 0), 0, y);
                else ptx::tma_load_2d(dst, &tm_w, &full[s], 0, y);
            };
            auto load_x = [&](int s, int kb, int m_tile) {
                uint8_t* dst = smem + s * C::STAGE_BYTES + BLOCK_BYTES;
                const int y = m_tile * MT + rank * C::X_ROWS;
                if constexpr (PAIR) ptx::tma_load_2d_pair(dst, &tm_x, ptx::cluster_map(ptx::smem_u32(&full[s]), 0), kb * BLOCK_COLS, y);
                else ptx::tma_load_2d(dst, &tm_x, &full[s], kb * BLOCK_COLS, y);
            };
            // the first stages' weights: older than the predecessor (w8a8.cuh)
            int pre = 0;
            {
                SegIter pit = it;
                while (pre < C::STAGES && pit.next(tile, kb0, kb1)) {
                    int m_tile, n_tile;
                    gemm::tile_to_mn(sched, tile, m_tile, n_tile);
                    for (int kb = kb0; kb < kb1 && pre < C::STAGES; ++kb, ++pre) load_w(pre, kb, n_tile);
                }
            }
            grid_dep_wait();
            int issued = 0;
            while (ok && it.next(tile, kb0, kb1)) {
                int m_tile, n_tile;
                gemm::tile_to_mn(sched, tile, m_tile, n_tile);
                for (int kb = kb0; kb < kb1; ++kb, ++issued) {
                    if (issued >= pre) {
                        if (!ptx::mbar_wait(&empty[stage], phase ^ 1, abort_flag)) { ok = false; break; }
                        load_w(stage, kb, n_tile);
                    }
                    load_x(stage, kb, m_tile);
                    if (++stage == C::STAGES) { stage = 0; phase ^= 1; }
                }
            }
        } else {
            grid_dep_wait();
        }
    } else if (warp == 1) {
        // ------------------------------------------------ MMA issuer (pairs: rank 0).  The whole warp walks the blocks and one lane issues: descriptors
        // that are the same in all lanes stay in uniform registers, where the instruction takes them.
        if (rank == 0) {
            constexpr uint32_t idesc = idesc_s8(CSZ * TILE_ROWS, MT);
            const bool leader = ptx::elect_one();
            int stage = 0;
            uint32_t phase = 0;
            int acc = 0;
            uint32_t acc_phase = 0;
            int tile, kb0, kb1;
            bool ok = true;
            while (ok && it.next(tile, kb0, kb1)) {
                if (!ptx::mbar_wait_warp(&acc_empty[acc], acc_phase ^ 1, abort_flag)) break;
                ptx::tc_fence_after();
                for (int kb = kb0; kb < kb1; ++kb) {
                    if (!ptx::mbar_wait_warp(&full[stage], phase, abort_flag)) { ok = false; break; }
                    ptx::tc_fence_after();
                    if (leader) {
                        const uint32_t wa = ptx::smem_u32(smem + stage * C::STAGE_BYTES);
                        umma_block<PAIR>(tmem_base + acc * MT, wa, wa + BLOCK_BYTES, idesc, kb == kb0);
                        if constexpr (PAIR) ptx::umma_commit_pair(&empty[stage]);
                        else ptx::umma_commit(&empty[stage]);
                    }
                    __syncwarp();
                    if (++stage == C::STAGES) { stage = 0; phase ^= 1; }
                }
                if (!ok) break;
                if (leader) {
                    if constexpr (PAIR) ptx::umma_commit_pair(&acc_full[acc]);
                    else ptx::umma_commit(&acc_full[acc]);
                }
                __syncwarp();
                acc ^= 1;
                if (acc == 0) acc_phase ^= 1;
            }
        }
    } else {
        epilogue<MT, PAIR>(a, it, tmem_base, acc_full, acc_empty, abort_flag, s_last, warp, lane, threadIdx.x - 64, g, G, xch, scales, rank);
    }

    ptx::tc_fence_before();
    __syncthreads();
    if constexpr (PAIR) {
        __syncwarp();
        ptx::cluster_sync();   // neither CTA leaves while the other may still read its memory or arrive at its barriers
    }
    if (warp == 1) {
        ptx::tc_fence_after();
        if constexpr (PAIR) ptx::tmem_dealloc_pair(tmem_base, C::TMEM_COLS);
        else ptx::tmem_dealloc(tmem_base, C::TMEM_COLS);
    }
    if (threadIdx.x == 0) finish(abort_flag, a.errors);
}

// A tile per cluster: CTA `rank` of CS has k-blocks [rank * kblocks / CS, (rank + 1) * kblocks / CS).  Each CTA sends each peer that peer's share of the tokens
// straight from tensor memory into a buffer beside the operand ring; one cluster barrier, and every CTA adds and stores its own share.  A first barrier only
// says that every CTA has started: arrived at on entry, waited for before the first write to a peer.  All threads reach both barriers whatever
// the bounded waits before returned.
template <int MT, int CS>
struct ClusterCfg {
    static constexpr int STAGE_BYTES = Cfg<MT, false>::STAGE_BYTES;
    static constexpr int STAGES = MT <= 64 ? Cfg<MT, false>::STAGES : 5;
    static constexpr int TPR = MT / CS + (MT % CS != 0);            // tokens summed and stored by each rank
    static constexpr int RED_BYTES = CS * TPR * TILE_ROWS * 4;
    static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + RED_BYTES + CTRL_BYTES + 1024;
    static_assert(SMEM_BYTES <= 232448, "shared memory budget");
};

template <int MT, int CS>
__global__ void __launch_bounds__(CLUSTER_THREADS, 1)
product_s8_cluster_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, const ProductArgs a) {
    using C = ClusterCfg<MT, CS>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    int* red = reinterpret_cast<int*>(smem + C::STAGES * C::STAGE_BYTES);   // [source][token][row]: peers write here, nothing else does
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::STAGES * C::STAGE_BYTES + C::RED_BYTES);
    uint64_t* empty = full + C::STAGES;
    uint64_t* acc_full = empty + C::STAGES;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 2);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    __shared__ float xs[C::TPR];   // scales of this CTA's tokens

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = static_cast<int>(ptx::cluster_ctarank());
    const int m_tile = blockIdx.x / CS / a.sched.n_tiles, tile = blockIdx.x / CS - m_tile * a.sched.n_tiles, kblocks = a.sched.kblocks;
    const int m_base = m_tile * MT;
    const int kb_begin = kblocks * rank / CS, kpc = kblocks * (rank + 1) / CS - kb_begin;
    grid_dep_trigger();
    ptx::cluster_arrive_relaxed();   // "this CTA runs"

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; ++s) {
            ptx::mbar_init(&full[s], 1);
            ptx::mbar_init(&empty[s], 1);
        }
        ptx::mbar_init(acc_full, 1);
        *abort_flag = 0;
        ptx::mbar_fence_init();
        ptx::prefetch_tensormap(&tm_w);
        ptx::prefetch_tensormap(&tm_x);
    }
    if (warp == 1) {
        ptx::tmem_alloc(tmem_slot, Cfg<MT, false>::TMEM_COLS);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    if (warp != 0) grid_dep_wait();

    const int q = warp & 3, row = q * 32 + lane;
    bool summed = false;   // epilogue threads: this CTA's sums are in tensor memory
    const int m_cnt = min(a.sched.M - m_base, MT), t0 = rank * C::TPR, cnt = min(m_cnt - t0, C::TPR);   // this CTA's share of the tile's tokens
    float ws = 0.f, bias = 0.f;
    if (warp == 0) {
        if (lane == 0) {
            const int pre = min(kpc, C::STAGES);
            for (int i = 0; i < pre; ++i) {   // weights: older than the predecessor
                ptx::mbar_arrive_expect_tx(&full[i], C::STAGE_BYTES);
                ptx::tma_load_2d(smem + i * C::STAGE_BYTES, &tm_w, &full[i], 0, (tile * kblocks + kb_begin + i) * TILE_ROWS);
            }
            grid_dep_wait();
            int stage = 0;
            uint32_t phase = 0;
            for (int i = 0; i < kpc; ++i) {
                uint8_t* dst = smem + stage * C::STAGE_BYTES;
                if (i >= pre) {
                    if (!ptx::mbar_wait(&empty[stage], phase ^ 1, abort_flag)) break;
                    ptx::mbar_arrive_expect_tx(&full[stage], C::STAGE_BYTES);
                    ptx::tma_load_2d(dst, &tm_w, &full[stage], 0, (tile * kblocks + kb_begin + i) * TILE_ROWS);
                }
                ptx::tma_load_2d(dst + BLOCK_BYTES, &tm_x, &full[stage], (kb_begin + i) * BLOCK_COLS, m_base);
                if (++stage == C::STAGES) { stage = 0; phase ^= 1; }
            }
        } else {
            grid_dep_wait();
        }
    } else if (warp == 1) {
        constexpr uint32_t idesc = idesc_s8(TILE_ROWS, MT);
        const bool leader = ptx::elect_one();
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int i = 0; i < kpc; ++i) {
            if (!ptx::mbar_wait_warp(&full[stage], phase, abort_flag)) { ok = false; break; }
            ptx::tc_fence_after();
            if (leader) {
                const uint32_t wa = ptx::smem_u32(smem + stage * C::STAGE_BYTES);
                umma_block<false>(tmem_base, wa, wa + BLOCK_BYTES, idesc, i == 0);
                ptx::umma_commit(&empty[stage]);
            }
            __syncwarp();
            if (++stage == C::STAGES) { stage = 0; phase ^= 1; }
        }
        if (ok && leader) ptx::umma_commit(acc_full);
        __syncwarp();
    } else {
        // scales while the sums are being made
        ws = a.ws[tile * TILE_ROWS + row];
        if (a.act == nullptr && a.bias != nullptr && tile * TILE_ROWS + row < a.N) bias = __bfloat162float(a.bias[tile * TILE_ROWS + row]);
        if (threadIdx.x - 64 < C::TPR) xs[threadIdx.x - 64] = static_cast<int>(threadIdx.x) - 64 < cnt ? a.xs[m_base + t0 + threadIdx.x - 64] : 0.f;
        summed = ptx::mbar_wait_warp(acc_full, 0, abort_flag);
        ptx::tc_fence_after();
    }
    __syncwarp();
    ptx::cluster_wait();   // every CTA has started: its shared memory may be written

    const uint32_t t_addr = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
    if (warp >= 2 && summed) {
        const uint32_t mine = ptx::smem_u32(red + rank * C::TPR * TILE_ROWS + row);
        // token t goes to rank t / TPR, place t % TPR
#pragma unroll 1
        for (int c0 = 0; c0 < m_cnt; c0 += 16) {
            int r[16];
            load16(t_addr + c0, r);
            ptx::tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 16; ++c) {
                const int t = c0 + c, d = t / C::TPR;
                if (t < m_cnt) {
                    const uint32_t at = ptx::cluster_map(mine, static_cast<uint32_t>(d)) + (t - d * C::TPR) * TILE_ROWS * 4;
                    asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(at), "r"(r[c]) : "memory");
                }
            }
        }
    }
    ptx::tc_fence_before();
    __syncwarp();
    ptx::cluster_sync();   // this CTA's share has arrived
    if (warp >= 2 && *abort_flag == 0) {
        if (a.act == nullptr) {
            const int n = tile * TILE_ROWS + row;
#pragma unroll 4
            for (int t = 0; t < cnt; ++t) {
                int sum = 0;
#pragma unroll
                for (int s = 0; s < CS; ++s) sum += red[(s * C::TPR + t) * TILE_ROWS + row];
                if (n < a.N) a.y[static_cast<long long>(m_base + t0 + t) * a.ldy + n] = __float2bfloat16(fmaf(static_cast<float>(sum) * xs[t], ws, bias));
            }
        } else {
            // gate rows 0-63 and up rows 64-127 meet in the first source's place, scaled
            float* meet = reinterpret_cast<float*>(red);
#pragma unroll 4
            for (int t = 0; t < cnt; ++t) {
                int sum = 0;
#pragma unroll
                for (int s = 0; s < CS; ++s) sum += red[(s * C::TPR + t) * TILE_ROWS + row];
                meet[t * TILE_ROWS + row] = static_cast<float>(sum) * xs[t] * ws;
            }
            ptx::named_bar_sync(1, 128);
            const int f = row & 63, n = tile * 64 + f;
            for (int t = row >> 6; t < cnt; t += 2) {
                if (n < a.N) a.act[static_cast<long long>(m_base + t0 + t) * a.ldy + n] = silu(meet[t * TILE_ROWS + f]) * meet[t * TILE_ROWS + 64 + f];
            }
        }
    }

    __syncthreads();
    if (warp == 1) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem_base, Cfg<MT, false>::TMEM_COLS);
    }
    if (threadIdx.x == 0) finish(abort_flag, a.errors);
}

// ---------------------------------------------------------------- host
CUtensorMap map_rows(const void* base, long long rows, long long cols, int box_rows) {
    return make_tmap_2d_u8_sw128(base, cols, rows, cols, BLOCK_COLS, box_rows);
}

template <typename... A>
bool allow_smem(void (*kernel)(A...), int bytes) {
    CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    return true;
}

template <int MT, bool PAIR>
void run(const CUtensorMap& tw, const CUtensorMap& tx, const ProductArgs& a, int grid, cudaStream_t s) {
    using C = Cfg<MT, PAIR>;
    static const bool allowed = allow_smem(product_s8_kernel<MT, PAIR>, C::SMEM_BYTES);   // the library runs on one device
    (void)allowed;
    launch_on(product_s8_kernel<MT, PAIR>, grid, C::THREADS, C::SMEM_BYTES, s, PAIR ? 2 : 1, true, tw, tx, a);
}
template <int MT, int CS>
void run_cluster(const CUtensorMap& tw, const CUtensorMap& tx, const ProductArgs& a, int grid, cudaStream_t s) {
    using C = ClusterCfg<MT, CS>;
    static const bool allowed = allow_smem(product_s8_cluster_kernel<MT, CS>, C::SMEM_BYTES);
    (void)allowed;
    launch_on(product_s8_cluster_kernel<MT, CS>, grid, CLUSTER_THREADS, C::SMEM_BYTES, s, CS, true, tw, tx, a);
}
template <int MT>
void run_cluster(int cs, const CUtensorMap& tw, const CUtensorMap& tx, const ProductArgs& a, int grid, cudaStream_t s) {
    if (cs == 2) run_cluster<MT, 2>(tw, tx, a, grid, s);
    else if (cs == 3) run_cluster<MT, 3>(tw, tx, a, grid, s);
    else if (cs == 4) run_cluster<MT, 4>(tw, tx, a, grid, s);
    else run_cluster<MT, 8>(tw, tx, a, grid, s);
}
template <int MT, int CS>
int capacity_of() {
    static const int n = [] {
        allow_smem(product_s8_cluster_kernel<MT, CS>, ClusterCfg<MT, CS>::SMEM_BYTES);
        return max_active_clusters(product_s8_cluster_kernel<MT, CS>, dim3(CLUSTER_THREADS), ClusterCfg<MT, CS>::SMEM_BYTES, CS);
    }();
    return n;
}
// clusters the device runs at once; the kernels differ in their stages only by the token tile, and by less than a CTA's worth
template <int MT>
int capacity(int cs) { return cs == 2 ? capacity_of<MT, 2>() : cs == 3 ? capacity_of<MT, 3>() : cs == 4 ? capacity_of<MT, 4>() : capacity_of<MT, 8>(); }
int cluster_capacity(int mt, int cs) { return mt == 16 ? capacity<16>(cs) : mt == 32 ? capacity<32>(cs) : mt == 64 ? capacity<64>(cs) : capacity<128>(cs); }

// How a product is divided: by its sizes alone.
struct Division {
    int mt = 0, m_tiles = 0;
    int cluster = 0;       // CTAs per tile, one tile per cluster
    bool pair = false;
    bool cut = false;      // pieces of tiles, which are summed through the workspace
    int workers = 0;       // CTAs, pairs, or clusters
    int wave_tiles = 0, tail_grid = 0;
};
// Of all kinds of tiles the one that is expected to end first.  In cycles, fitted to runs of all kinds: block, a k-block of a CTA (the weights no sooner than
// HBM gives them); out, a tile's way out of tensor memory, where no other tile hides it (clusters: with the sum); next, what one tile takes at least
// where another one follows.
Division find_division(int M, int tiles, int kblocks, bool gated, int sms) {
    Division d;
    const int widest = linear_pick_mt(M), from_hbm = static_cast<int>(static_cast<long long>(tiles) * kblocks * BLOCK_BYTES / 3440);
    long long best = -1;
    auto better = [&](long long cost) {
        if (best >= 0 && cost >= best) return false;
        best = cost;
        return true;
    };
    // One tile per cluster, all clusters at once.  Rows x columns x outputs, single CTAs (whole or cut) and the best cluster: 95 x 2624 x 256 10.0, 4.6 us
    // (tiles of 16, 8 CTAs); 200 x 1024 x 1024 7.1, 5.7 (32, 2); 300 x 4096 x 1024 12.9, 10.3 (64, 3); 128 x 16384 x 4096 28.2, 19.9 (128, 4); but
    // 333 x 713 x 1001 7.7, 8.7 and 100 x 128 x 1024 whole (the rows' own kernel in all of them).
    struct Cluster { int mt, block, out; };
    constexpr Cluster clusters[] = {{16, 400, 2500}, {32, 420, 2800}, {64, 440, 5400}, {128, 490, 8900}};
    for (const Cluster& k : clusters) {
        const long long n = static_cast<long long>(tiles) * ceil_div(M, k.mt);
        if (k.mt > widest || 2 * n > sms) continue;
        for (int cs : {8, 4, 3, 2}) {
            if (kblocks < 2 * cs || n * cs > sms) continue;
            const long long cost = std::max(ceil_div(kblocks, cs) * k.block, from_hbm) + k.out;
            if ((best >= 0 && cost >= best) || cluster_capacity(k.mt, cs) < n) continue;
            best = cost;
            d.mt = k.mt;
            d.cluster = cs;
        }
    }
    // Single CTAs and pairs, and whether the tiles of the last wave are cut into equal pieces.  Whole tiles of 64, 128, 256 and pairs, with the rows' kernel:
    // 300 x 4096 x 4096 21.3, 14.4, 18.0, 18.0 us; 1000 x 4096 x 4608 37.3, 24.2, 19.6, 20.0; 2048 x 4096 x 4096 61.8, 42.1, 31.9, 30.8.  Of 16, 32, 64, 128,
    // 256 and pairs: 150 x 64 x 16384 13.3, 9.8, 7.9, 7.9, 6.7, 7.7; 250 x 74 x 3519 9.0, 6.5, 5.9, 6.9, 9.3, 10.2; 2000 x 512 x 2048 23.7, 16.1, 12.5,
    // 11.0, 10.5, 11.5.  Cut tiles, products alone: 4096 x 16384 x 4096 pairs 177, cut 174; but 2048 x 4096 x 4096 pairs 25.7, cut 36.6.
    // sum: over a cut tile's pieces, as far as whole tiles behind it do not hide it.
    struct Kind { int mt; bool pair; int block, out, next, sum; };
    constexpr Kind kinds[] = {{16, false, 420, 2200, 2000, 20000}, {32, false, 440, 2400, 2300, 20000}, {64, false, 420, 3200, 3200, 20000},
                              {128, false, 500, 4300, 5500, 30000}, {256, false, 580, 6800, 9000, 45000}, {256, true, 540, 9200, 10500, 45000}};
    for (const Kind& k : kinds) {
        if (k.mt > widest || (k.pair && tiles % 2 != 0)) continue;
        const long long n = static_cast<long long>(k.pair ? tiles / 2 : tiles) * ceil_div(M, k.mt);
        const int workers = k.pair ? sms / 2 : sms;
        const long long waves = n / workers, last = n - waves * workers, one = static_cast<long long>(kblocks) * k.block;
        const long long behind = last > 0 ? waves : waves - 1;    // waves that another one follows
        if (better(std::max<long long>(behind * std::max<long long>(one, k.next) + one, from_hbm) + k.out)) {
            d.mt = k.mt;
            d.pair = k.pair;
            d.cut = false;
            d.cluster = 0;
        }
        if (gated || last == 0 || last * kblocks < workers * 4) continue;   // gate/up tiles: the activation needs complete sums; pieces of four blocks at least
        const long long sum = std::max<long long>(0, k.sum - waves * one), share = (n * kblocks + workers - 1) / workers * k.block;
        if (better(std::max({share, waves * k.next, static_cast<long long>(from_hbm)}) + k.out + 6000 + sum)) {
            d.mt = k.mt;
            d.pair = k.pair;
            d.cut = true;
            d.cluster = 0;
        }
    }
    d.m_tiles = ceil_div(M, d.mt);
    if (d.cluster > 0) {
        d.workers = tiles * d.m_tiles;
        return d;
    }
    const int n_tiles = d.pair ? tiles / 2 : tiles, most = d.pair ? sms / 2 : sms;
    const long long all = static_cast<long long>(n_tiles) * d.m_tiles;
    if (!d.cut) {
        const long long rounds = (all + most - 1) / most;
        d.workers = static_cast<int>(std::min<long long>(d.m_tiles == 1 ? (all + rounds - 1) / rounds : most, all));
        d.wave_tiles = static_cast<int>(all);
        d.tail_grid = 1;
        return d;
    }
    d.workers = static_cast<int>(std::max<long long>(1, std::min<long long>(most, all * kblocks / 4)));
    if (d.m_tiles > 1) gemm::plan_waves(all, kblocks, d.workers, d.wave_tiles, d.tail_grid);
    return d;
}

// A call asks several times for the division of the same sizes (its workspace, its layout, its launch), and a model's layers repeat theirs: each thread keeps
// the last ones (0.3 us a search).
Division divide(int M, int tiles, int kblocks, bool gated) {
    struct Found {
        int M = -1, tiles = 0, kblocks = 0;
        bool gated = false;
        Division d;
    };
    thread_local Found found[16];
    Found& f = found[(static_cast<unsigned>(M) * 31u + static_cast<unsigned>(tiles) * 7u + static_cast<unsigned>(kblocks) * 3u + gated) % 16u];
    if (f.M != M || f.tiles != tiles || f.kblocks != kblocks || f.gated != gated) {
        f.M = -1;   // an exception leaves no entry
        f.d = find_division(M, tiles, kblocks, gated, runtime().num_sms);
        f.M = M;
        f.tiles = tiles;
        f.kblocks = kblocks;
        f.gated = gated;
    }
    return f.d;
}

}  // namespace

Scratch product_scratch(int M, int N, int K) {
    Scratch s;
    if (M <= 1) return s;
    const int tiles = tiles_of(N, false);
    const Division d = divide(M, tiles, pad_cols(K) / BLOCK_COLS, false);
    if (d.cut) {
        s.partial_bytes = static_cast<size_t>(d.workers) * (d.pair ? 2 : 1) * 2 * d.mt * TILE_ROWS * sizeof(int);
        s.tickets = tiles * d.m_tiles;
    }
    return s;
}

void product_division(int M, int N, int K, bool gated, int32_t (&out)[6]) {
    const Division d = divide(M, tiles_of(N, gated), pad_cols(K) / BLOCK_COLS, gated);
    const int32_t v[6] = {d.mt, d.m_tiles, d.cluster, d.pair, d.cut, d.workers};
    std::copy(v, v + 6, out);
}

void launch_product(const Product& p, cudaStream_t s) {
    const bool gated = p.act != nullptr;
    const Division d = divide(p.M, p.w.tiles, p.w.kblocks, gated);
    ProductArgs a;
    gemm::LinearArgs& w = a.sched;
    w = gemm::LinearArgs();
    w.M = p.M; w.N = p.N; w.K = p.K;
    w.n_tiles = d.pair ? p.w.tiles / 2 : p.w.tiles;
    w.m_tiles = d.m_tiles;
    w.kblocks = p.w.kblocks;
    w.wave_tiles = d.wave_tiles;
    w.tail_grid = d.tail_grid;
    w.total_units = (static_cast<long long>(w.n_tiles) * w.m_tiles - w.wave_tiles) * w.kblocks;
    w.band = gemm::raster_band(d.mt, p.w.kblocks * BLOCK_COLS / 2);   // bytes of a token row as the rule counts them
    a.N = p.N;
    a.xs = p.xs; a.ws = p.w.scales; a.bias = p.bias;
    a.y = p.y; a.ldy = p.ldy; a.act = p.act;
    a.partials = static_cast<int*>(p.partials);
    a.tickets = p.tickets;
    a.errors = op_counters(s);
    const CUtensorMap tw = map_rows(p.w.blocks, static_cast<long long>(p.w.tiles) * p.w.kblocks * TILE_ROWS, BLOCK_COLS, TILE_ROWS);
    const CUtensorMap tx = map_rows(p.q, p.M, static_cast<long long>(p.w.kblocks) * BLOCK_COLS, d.pair ? d.mt / 2 : d.mt);
    if (d.cluster > 0) {
        const int grid = d.workers * d.cluster;
        if (d.mt == 16) run_cluster<16>(d.cluster, tw, tx, a, grid, s);
        else if (d.mt == 32) run_cluster<32>(d.cluster, tw, tx, a, grid, s);
        else if (d.mt == 64) run_cluster<64>(d.cluster, tw, tx, a, grid, s);
        else run_cluster<128>(d.cluster, tw, tx, a, grid, s);
        return;
    }
    if (d.pair) {
        run<256, true>(tw, tx, a, 2 * d.workers, s);
        return;
    }
    switch (d.mt) {
        case 16: run<16, false>(tw, tx, a, d.workers, s); break;
        case 32: run<32, false>(tw, tx, a, d.workers, s); break;
        case 64: run<64, false>(tw, tx, a, d.workers, s); break;
        case 128: run<128, false>(tw, tx, a, d.workers, s); break;
        default: run<256, false>(tw, tx, a, d.workers, s); break;
    }
}

}  // namespace w8
