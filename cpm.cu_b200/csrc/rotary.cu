// Rotary positions, sm_100a:  pair i of every query and key head of a row becomes
//   (a cos - b sin, b cos + a sin),  angle = pos * inv_freq[i],  sines and cosines times a factor,
// with pair i = elements (2 i, 2 i + 1) (interleaved) or (i, i + half), on the first 2 * half elements of a head; the rest of it is copied.
// Rotated keys, and values as they are, go to the row's cache slot.
//
// The angle is a 64-bit product, reduced to a fraction of a turn before it becomes fp32: at position 10^6 an fp32 product is off by 0.03
// radians.
//
// Bound: every element in and out once.  Few rows: one CTA per row, whose loads are in flight while some threads make the row's `half` sines and
// cosines (60 rows of 32 + 2 * 2 heads of 128: 2.4 us, a launch).  Many: CTAs that stay, with rings of rows (8192 rows of 32 + 2 * 8 heads of 128:
// 34.6 us, 5.8 TB/s; 50 % of the DRAM's time cold and alone, half of the output still in L2 at the end).
#include <algorithm>

#include "ptx.cuh"
#include "row_ops.cuh"
#include "rotary.cuh"

namespace {

// VEC elements as they lie in memory; WIDE: in one access
template <int VEC, bool WIDE>
struct Elems {
    alignas(VEC > 1 ? 4 : 2) bf16 e[VEC];
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

// Two pairs (a.lo, b.lo), (a.hi, b.hi) of packed values.
__device__ __forceinline__ void turn_two(uint32_t& a, uint32_t& b, const float* cs, const float* sn) {
    const uint32_t x = a, y = b;
    a = two_bf16(fmaf(low(x), cs[0], -(low(y) * sn[0])), fmaf(high(x), cs[1], -(high(y) * sn[1])));
    b = two_bf16(fmaf(low(y), cs[0], low(x) * sn[0]), fmaf(high(y), cs[1], high(x) * sn[1]));
}
// One pair (lo, hi)
__device__ __forceinline__ void turn_within(uint32_t& a, float cs, float sn) {
    const uint32_t x = a;
    a = two_bf16(fmaf(low(x), cs, -(high(x) * sn)), fmaf(high(x), cs, low(x) * sn));
}
__device__ __forceinline__ void turn(bf16& a, bf16& b, float cs, float sn) {
    const float x = __bfloat162float(a), y = __bfloat162float(b);
    a = __float2bfloat16(fmaf(x, cs, -(y * sn)));
    b = __float2bfloat16(fmaf(y, cs, x * sn));
}

// Sines and cosines of a row: `padded` cosines, then the sines.
__host__ __device__ constexpr int padded(int half) { return (half + 7) / 8 * 8; }
// turns per position of a frequency
__device__ __forceinline__ double turns_of(float inv_freq) { return static_cast<double>(inv_freq) * 0.15915494309189533577; }
__device__ __forceinline__ void fill(float* table, int i, int half, int32_t pos, double per_pos, float factor) {
    const double turns = static_cast<double>(pos) * per_pos;
    float sn, cs;
    sincospif(2.f * static_cast<float>(turns - rint(turns)), &sn, &cs);
    table[i] = cs * factor;
    table[padded(half) + i] = sn * factor;
}
template <int N>
__device__ __forceinline__ void take(const float* p, float (&f)[N]) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) *reinterpret_cast<float4*>(f + i) = *reinterpret_cast<const float4*>(p + i);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = p[i];
    }
}

// A piece of a row: VEC elements and their partners `half` further on, or (interleaved) VEC elements that lie together.
template <int VEC, bool INTERLEAVED, bool WIDE>
struct Piece {
    Elems<VEC, WIDE> lo, hi;
    __device__ __forceinline__ void load(const bf16* p, int half) {
        lo.load(p);
        if constexpr (!INTERLEAVED) hi.load(p + half);
    }
    // c: first element in the head, a multiple of VEC
    __device__ __forceinline__ void rotate(int c, int half, const float* table) {
        constexpr int N = INTERLEAVED ? (VEC + 1) / 2 : VEC;   // pairs
        const int first = INTERLEAVED ? c >> 1 : c;
        alignas(16) float cs[N], sn[N];
        if (INTERLEAVED && first >= half) return;
        take<N>(table + first, cs);
        take<N>(table + padded(half) + first, sn);
        if constexpr (VEC == 1) {
            turn(lo.e[0], hi.e[0], cs[0], sn[0]);
        } else {
            uint32_t *a = reinterpret_cast<uint32_t*>(lo.e), *b = reinterpret_cast<uint32_t*>(hi.e);
#pragma unroll
            for (int j = 0; j < VEC / 2; ++j) {
                if constexpr (INTERLEAVED) {
                    if (first + j < half) turn_within(a[j], cs[j], sn[j]);
                } else {
                    turn_two(a[j], b[j], cs + 2 * j, sn + 2 * j);
                }
            }
        }
    }
    __device__ __forceinline__ void store(bf16* p, int half) const {
        lo.store(p);
        if constexpr (!INTERLEAVED) hi.store(p + half);
    }
};

constexpr int MAX_HALF = 512;

// One CTA per row: what has few rows, and what does not lie in 16-byte pieces.  A thread's first pieces are in flight before the table is made.
template <int VEC, bool INTERLEAVED, bool WIDE>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryArgs a) {
    __shared__ __align__(16) float table[2 * padded(MAX_HALF)];
    constexpr int AHEAD = 2;
    const int kv_dim = a.kv_heads * a.dim, all = a.heads + a.kv_heads;
    // pieces of a head that are rotated (interleaved: all of it, the unrotated pairs as they are), and that are copied
    const int turned = INTERLEAVED ? a.dim / VEC : a.half / VEC, copied = INTERLEAVED ? 0 : (a.dim - 2 * a.half) / VEC;
    const int items = all * turned;
    const int v0 = threadIdx.x * VEC;
    const long long r = blockIdx.x;
    const bf16* row = a.qkv + r * a.ld;
    bf16* q = a.q + r * a.ldq;
    grid_dep_wait();
    grid_dep_trigger();
    Piece<VEC, INTERLEAVED, WIDE> piece[AHEAD];
    Elems<VEC, WIDE> value;
    auto place = [&](int i, int& h, int& c) {
        h = i / turned;
        c = (i - h * turned) * VEC;
    };
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
        const int i = threadIdx.x + j * blockDim.x;
        if (i < items) {
            int h, c;
            place(i, h, c);
            piece[j].load(row + h * a.dim + c, a.half);
        }
    }
    if (v0 < kv_dim) value.load(row + all * a.dim + v0);
    long long slot = a.kv_heads > 0 ? a.slots[r] : -1;
    const int32_t pos = a.pos[r];
    for (int t = threadIdx.x; t < a.half; t += blockDim.x) fill(table, t, a.half, pos, turns_of(a.inv_freq[t]), a.factor);
    if (slot >= a.cache_rows) {   // memory stays intact; the host hears of it
        slot = -1;
        if (threadIdx.x == 0) report(a.errors, OP_KV_OVERFLOW);
    }
    const bool keep = slot >= 0;
    bf16 *k_row = a.k_cache + slot * kv_dim, *v_row = a.v_cache + slot * kv_dim;
    auto target = [&](int h, int c) { return h < a.heads ? q + h * a.dim + c : k_row + (h - a.heads) * a.dim + c; };
    if (keep && v0 < kv_dim) value.store(v_row + v0);
    __syncthreads();
    for (int i = threadIdx.x, j = 0; i < items; i += blockDim.x, ++j) {
        int h, c;
        place(i, h, c);
        Piece<VEC, INTERLEAVED, WIDE> e;
        if (j == 0) e = piece[0];
        else if (j == 1) e = piece[1];
        else e.load(row + h * a.dim + c, a.half);
        e.rotate(c, a.half, table);
        if (h < a.heads || keep) e.store(target(h, c), a.half);
    }
    // what no rotation reaches: the rest of the heads, and the values
    if constexpr (!INTERLEAVED) {
        for (int j = threadIdx.x; j < all * copied; j += blockDim.x) {
            const int h = j / copied, c = 2 * a.half + (j - h * copied) * VEC;
            Elems<VEC, WIDE> e;
            e.load(row + h * a.dim + c);
            if (h < a.heads || keep) e.store(target(h, c));
        }
    }
    if (keep) {
        for (int j = v0 + blockDim.x * VEC; j < kv_dim; j += blockDim.x * VEC) {
            value.load(row + all * a.dim + j);
            value.store(v_row + j);
        }
    }
}

// Many rows: CTAs that stay, each with a ring of groups of rows in shared memory.  Bulk copies bring a group; while the threads turn group i, some of them
// make the tables of group i + 1, and the copies of the next groups are on their way.  A row alone in a CTA spends a third of its time with loads in
// flight.
constexpr int RING_STAGES = 3, RING_GROUP_BYTES = 12 * 1024, RING_MAX_GROUP = 8, RING_MAX_ROW_BYTES = 24 * 1024, RING_CTAS = 4;
// i / d for i * d < 2^32
struct Divisor {
    uint32_t d = 1, m = 0;
    void set(int v) { d = v; m = v > 1 ? static_cast<uint32_t>(((1ull << 32) + v - 1) / v) : 0u; }
    __device__ __forceinline__ int operator()(int i) const { return d == 1 ? i : static_cast<int>(__umulhi(static_cast<uint32_t>(i), m)); }
};
struct RingArgs {
    RotaryArgs a;
    int rows, group, groups, row_bytes;
    int turned, copied;                       // pieces of rotated elements (two vectors, or one where interleaved heads have an odd number), and copied vectors, per head
    int apart;                                // of a piece's vectors: interleaved pairs lie in them, the others across them
    Divisor by_items, by_turned, by_copies, by_copied, by_values;
};
template <bool INTERLEAVED, int VEC, bool TWO = true>
__global__ void __launch_bounds__(256, RING_CTAS) rotary_ring_kernel(const RingArgs g) {
    const RotaryArgs& a = g.a;
    const int G = g.group, pad = 2 * padded(a.half), stage_bytes = G * g.row_bytes;
    extern __shared__ __align__(128) uint8_t smem[];   // stages of G rows, then two sets of G tables
    float* tables = reinterpret_cast<float*>(smem + RING_STAGES * stage_bytes);
    __shared__ uint64_t full[RING_STAGES];
    __shared__ int slots[2][RING_MAX_GROUP];
    __shared__ int abort_flag;
    const int kv_dim = a.kv_heads * a.dim, all = a.heads + a.kv_heads;
    const int items = all * g.turned, copies = all * g.copied, values = kv_dim / VEC;
    const int n = (g.groups - 1 - static_cast<int>(blockIdx.x)) / static_cast<int>(gridDim.x) + 1;   // groups of this CTA
    auto row_of = [&](int i, int r) { return (static_cast<long long>(blockIdx.x) + static_cast<long long>(i) * gridDim.x) * G + r; };
    auto rows_in = [&](int i) { return static_cast<int>(min(static_cast<long long>(G), g.rows - row_of(i, 0))); };
    if (threadIdx.x == 0) {
        for (int s = 0; s < RING_STAGES; ++s) ptx::mbar_init(&full[s], 1);
        abort_flag = 0;
        ptx::mbar_fence_init();
    }
    __syncthreads();
    grid_dep_wait();
    grid_dep_trigger();
    auto fetch = [&](int i, int s) {
        const int m = rows_in(i);
        ptx::mbar_arrive_expect_tx(&full[s], m * g.row_bytes);
        for (int r = 0; r < m; ++r) ptx::bulk_load(smem + s * stage_bytes + r * g.row_bytes, a.qkv + row_of(i, r) * a.ld, g.row_bytes, &full[s]);
    };
    if (threadIdx.x == 0) {
        for (int i = 0; i < RING_STAGES && i < n; ++i) fetch(i, i);
    }
    // A thread has one pair of one of the rows (or, of wide heads in groups of one, further ones); its frequency stays in a register, and positions
    // and slots are loaded two groups ahead: a table is arithmetic alone.
    const int my_row = a.half > 0 ? threadIdx.x / a.half : G, my_pair = a.half > 0 ? threadIdx.x - my_row * a.half : 0;
    const double mine = my_row < G ? turns_of(a.inv_freq[my_pair]) : 0.0;
    auto pos_of = [&](int i) { return my_row < G && i < n && my_row < rows_in(i) ? a.pos[row_of(i, my_row)] : 0; };
    auto slot_of = [&](int i) { return static_cast<int>(threadIdx.x) < G && a.kv_heads > 0 && i < n && static_cast<int>(threadIdx.x) < rows_in(i) ? a.slots[row_of(i, threadIdx.x)] : -1; };
    auto prepare = [&](int i, int32_t pos, int slot) {
        float* t = tables + (i & 1) * G * pad;
        if (my_row < G) fill(t + my_row * pad, my_pair, a.half, pos, mine, a.factor);
        for (int k = threadIdx.x + blockDim.x; k < a.half; k += blockDim.x) fill(t, k, a.half, pos, turns_of(a.inv_freq[k]), a.factor);
        if (static_cast<int>(threadIdx.x) < G) {
            if (slot >= a.cache_rows) {   // memory stays intact; the host hears of it
                slot = -1;
                report(a.errors, OP_KV_OVERFLOW);
            }
            slots[i & 1][threadIdx.x] = slot;
        }
    };
    prepare(0, pos_of(0), slot_of(0));
    int32_t next_pos = pos_of(1);
    int next_slot = slot_of(1);
    __syncthreads();
    int stage = 0;
    uint32_t phase = 0;
    for (int i = 0; i < n; ++i) {
        const int32_t pos = next_pos;
        const int slot = next_slot;
        next_pos = pos_of(i + 2);
        next_slot = slot_of(i + 2);
        if (i + 1 < n) prepare(i + 1, pos, slot);
        if (!ptx::mbar_wait(&full[stage], phase, &abort_flag)) break;
        const int m = rows_in(i);
        const float* table = tables + (i & 1) * G * pad;
        const bf16* from = reinterpret_cast<const bf16*>(smem + stage * stage_bytes);
        const int row_elems = g.row_bytes / 2;
        const long long r0 = row_of(i, 0);
        auto put = [&](auto& e, int r, int h, int c) {
            if (h < a.heads) {
                e(a.q + (r0 + r) * a.ldq + h * a.dim + c);
            } else {
                const long long at = slots[i & 1][r];
                if (at >= 0) e(a.k_cache + at * kv_dim + (h - a.heads) * a.dim + c);
            }
        };
        for (int j = threadIdx.x; j < m * items; j += blockDim.x) {
            const int r = g.by_items(j), k = j - r * items, h = g.by_turned(k), c = (k - h * g.turned) * VEC;
            const bf16* at = from + r * row_elems + h * a.dim + c;
            Piece<VEC, INTERLEAVED, true> e;
            e.load(at, a.half);
            if constexpr (INTERLEAVED) {
                Piece<VEC, true, true> e2;
                if constexpr (TWO) e2.load(at + g.apart, a.half);
                e.rotate(c, a.half, table + r * pad);
                if constexpr (TWO) e2.rotate(c + g.apart, a.half, table + r * pad);
                auto store = [&](bf16* to) {
                    e.store(to, a.half);
                    if constexpr (TWO) e2.store(to + g.apart, a.half);
                };
                put(store, r, h, c);
            } else {
                e.rotate(c, a.half, table + r * pad);
                auto store = [&](bf16* to) { e.store(to, a.half); };
                put(store, r, h, c);
            }
        }
        // values, and what no rotation reaches, from the other end of the threads
        const int back = blockDim.x - 1 - threadIdx.x;
        if constexpr (!INTERLEAVED) {
            for (int j = back; j < m * copies; j += blockDim.x) {
                const int r = g.by_copies(j), k = j - r * copies, h = g.by_copied(k), c = 2 * a.half + (k - h * g.copied) * VEC;
                Elems<VEC, true> e;
                e.load(from + r * row_elems + h * a.dim + c);
                auto store = [&](bf16* to) { e.store(to); };
                put(store, r, h, c);
            }
        }
        for (int j = back; j < m * values; j += blockDim.x) {
            const int r = g.by_values(j), c = (j - r * values) * VEC;
            const long long at = slots[i & 1][r];
            Elems<VEC, true> e;
            e.load(from + r * row_elems + all * a.dim + c);
            if (at >= 0) e.store(a.v_cache + at * kv_dim + c);
        }
        __syncthreads();   // the group has been read, the next tables are there
        if (threadIdx.x == 0 && i + RING_STAGES < n) {
            ptx::fence_proxy_async_smem();
            fetch(i + RING_STAGES, stage);
        }
        if (++stage == RING_STAGES) { stage = 0; phase ^= 1; }
    }
    if (abort_flag) {   // copies in flight land before the CTA retires
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000LL) {}
        if (threadIdx.x == 0) report(a.errors, OP_TIMEOUT);
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
    auto go = [&](auto kernel, int grid, int threads, size_t smem, const auto& args) { launch_on(kernel, grid, threads, smem, s, 1, true, args); };
    const int pieces = (a.heads + 2 * a.kv_heads) * a.dim / vec;
    const int sms = runtime().num_sms, row_bytes = (a.heads + 2 * a.kv_heads) * a.dim * 2;
    // Rings where every SM has eight rows, or three groups of several short rows: 8192 rows of 32 + 2 * 8 heads of 128 35.5 us (one CTA per row 45.0),
    // of 16 + 2 * 4 interleaved 19.1 (27.5), 2000 rows of 15 + 2 * 5 heads of 80 6.8 (7.3), 8000 rows of 4 + 2 heads of 64 6.3 (9.8); but
    // 1000 rows of 32 + 2 * 8 heads of 128 7.8 (7.4), 1000 of 12 + 2 * 4 heads of 64 3.8 (3.2).
    // (Narrower pieces where the halves of a head are no vectors of eight: 8192 rows of 3 + 2 * 3 heads of 72 7.3 (11.7), 4000 of 12 + 2 * 4 heads of 96, 24 elements
    // rotated, 9.2 (13.4).)
    const int group = std::max(1, std::min({RING_GROUP_BYTES / row_bytes, a.half > 0 ? 256 / a.half : RING_MAX_GROUP, RING_MAX_GROUP}));
    const int groups = ceil_div(rows, group);
    const bool bulk = (bits(a.qkv) & 15) == 0 && a.ld % 8 == 0 && row_bytes % 16 == 0;   // rows may be brought by bulk copies
    if (bulk && wide && vec >= (interleaved ? 8 : 2) && row_bytes <= RING_MAX_ROW_BYTES && groups >= (group > 1 ? 3 : 8) * sms) {
        RingArgs g;
        g.a = a;
        g.rows = rows;
        g.row_bytes = row_bytes;
        g.group = group;
        g.groups = groups;
        const bool two = a.dim % 16 == 0;
        g.apart = interleaved ? a.dim / 2 : a.half;
        g.turned = !interleaved ? a.half / vec : two ? a.dim / 16 : a.dim / 8;
        g.copied = interleaved ? 0 : (a.dim - 2 * a.half) / vec;
        const int all = a.heads + a.kv_heads;
        g.by_items.set(std::max(1, all * g.turned));
        g.by_turned.set(std::max(1, g.turned));
        g.by_copies.set(std::max(1, all * g.copied));
        g.by_copied.set(std::max(1, g.copied));
        g.by_values.set(std::max(1, a.kv_heads * a.dim / vec));
        const int smem = RING_STAGES * g.group * row_bytes + 2 * g.group * 2 * padded(a.half) * static_cast<int>(sizeof(float));
        auto* kernel = interleaved ? (two ? rotary_ring_kernel<true, 8> : rotary_ring_kernel<true, 8, false>) : vec == 8 ? rotary_ring_kernel<false, 8> : vec == 4 ? rotary_ring_kernel<false, 4> : rotary_ring_kernel<false, 2>;
        static const bool allowed = [] {   // the library runs on one device
            for (auto* k : {rotary_ring_kernel<true, 8>, rotary_ring_kernel<true, 8, false>, rotary_ring_kernel<false, 8>, rotary_ring_kernel<false, 4>, rotary_ring_kernel<false, 2>}) {
                CUDA_CHECK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, 96 * 1024));
            }
            return true;
        }();
        (void)allowed;
        const int per_sm = std::max(1, std::min(RING_CTAS, 227 * 1024 / (smem + 1280)));
        const int grid = std::min(g.groups, per_sm * sms);
        go(kernel, grid, 256, smem, g);
        return;
    }
    const int threads = pieces >= 256 ? 256 : (pieces + 31) / 32 * 32;
    if (interleaved) {
        if (vec == 8) go(rotary_kernel<8, true, true>, rows, threads, 0, a);
        else if (vec == 4) go(rotary_kernel<4, true, true>, rows, threads, 0, a);
        else if (wide) go(rotary_kernel<2, true, true>, rows, threads, 0, a);
        else go(rotary_kernel<2, true, false>, rows, threads, 0, a);
    } else {
        if (vec == 8) go(rotary_kernel<8, false, true>, rows, threads, 0, a);
        else if (vec == 4) go(rotary_kernel<4, false, true>, rows, threads, 0, a);
        else if (vec == 2) go(rotary_kernel<2, false, true>, rows, threads, 0, a);
        else go(rotary_kernel<1, false, false>, rows, threads, 0, a);
    }
}
