// Linear layers in 8-bit integers: y = (q W^T) * (scale of the token) * (scale of the channel) + bias, with q the rows rounded to
// integers in [-127, 127] (w8a8_rows.cu), W int8, sums exact in 32-bit integers.  Rows of one token go through w8a8_one_row.cu, more
// through the tensor cores (gemm_w8a8.cu).
//
// All launches here but the packing are programmatic, on the caller's stream.  A launch lets its successor start only where the note at its kernel
// says so; packed weights are the one thing that is fetched before the wait for the predecessor.  That is in order because the kernel that writes
// them (pack_kernel) lets no successor start before its CTAs have ended, with their writes in L2, and every later launch starts later still; the
// fetches go past the first-level cache.
#pragma once
#include "common.cuh"

namespace w8 {

constexpr int TILE_ROWS = 128;        // weight rows of a tile
constexpr int BLOCK_COLS = 128;       // int8 columns of a block: one 128-byte row
constexpr int BLOCK_BYTES = TILE_ROWS * BLOCK_COLS;
constexpr int MAX_COLS = 131072;      // 127 * 128 * MAX_COLS < 2^31

inline int pad_cols(int K) { return (K + BLOCK_COLS - 1) / BLOCK_COLS * BLOCK_COLS; }

// Packed weights: ceil(N / 128) x ceil(K / 128) blocks of 128 rows x 128 bytes, blocks of a tile consecutive along K (one sequential burst of 16 KB
// for each copy, as for the bf16 weights), zeros beyond N and K; then the fp32 scales of the tiles' rows.  A gate/up pair has 64
// gate rows and the 64 up rows of the same features in every tile.
struct Packed {
    const uint8_t* blocks = nullptr;
    const float* scales = nullptr;
    int tiles = 0, kblocks = 0;
};
enum Role : int { ROLE_PLAIN = 0, ROLE_GATE = 1, ROLE_UP = 2 };
size_t packed_bytes(int N, int K, bool gated);
Packed packed_view(const void* p, int N, int K, bool gated);
inline int tiles_of(int N, bool gated) { return ceil_div(N, gated ? TILE_ROWS / 2 : TILE_ROWS); }
void launch_pack(const int8_t* q, const float* scale, int N, int K, Role role, void* packed, cudaStream_t s);

// What the integers of a row are made of.
struct RowSource {
    const bf16* x = nullptr;        // rows of K values, ldx apart; or
    const float* x32 = nullptr;     // fp32 rows of whole vectors: K and ldx multiples of 8, 16-byte aligned
    long long ldx = 0;
    // norm != null: integers of t * norm, t = bf16(x + delta_scale * delta) (delta may be null: t = x), whose scale carries 1 / rms(t)
    const bf16* norm = nullptr;
    const bf16* delta = nullptr;    // [rows, K]
    bf16* total = nullptr;          // [rows, K]: t, where there is a delta
    float delta_scale = 1.f, eps = 0.f;
};
// q [rows, ldq] (zeros from K to pad_cols(K)), scale [rows]; also clears n_clear counters for the product behind it
void launch_quantize(const RowSource& src, int rows, int K, int8_t* q, long long ldq, int pad_to, float* scale, int* clear, int n_clear, cudaStream_t s);

struct Product {
    int M = 0, N = 0, K = 0;
    Packed w;
    const int8_t* q = nullptr;      // [M, pad_cols(K)]
    const float* xs = nullptr;      // [M], readable up to the next multiple of 256
    const bf16* bias = nullptr;
    bf16* y = nullptr;              // [M, ldy]
    long long ldy = 0;
    float* act = nullptr;           // gate/up weights: silu(gate) * up instead of y, fp32, N features, ldy floats apart
    void* partials = nullptr;
    int* tickets = nullptr;         // zero
};
struct Scratch {                    // what cut tiles need; gate/up tiles are never cut
    size_t partial_bytes = 0;
    int tickets = 0;
};
Scratch product_scratch(int M, int N, int K);
// How a product is divided: token tile, token tiles, CTAs of a cluster (0: none), pairs of CTAs, cut tiles, and clusters, pairs or CTAs (for tests)
void product_division(int M, int N, int K, bool gated, int32_t (&out)[6]);
void launch_product(const Product& p, cudaStream_t s);
// one row, straight from its source
void launch_one_row(const RowSource& src, int N, int K, const Packed& w, const bf16* bias, bf16* y, float* act, cudaStream_t s);

// silu in 32 bits, of exact sums: off by at most 5 * 2^-24 (the exponential 2; its product or the sum, the quotient 1 each).  An approximate exponential and
// quotient are off by 28 (|v| to 30), and put activations next to a border of the 8-bit integers on its other side.
// The quotient is that by an approximate reciprocal and one Newton step with its remainder, which needs no cases for divisors far from overflow; the general
// division has such cases, and tiles of activations take longer with it (60 x 2048 with 5632 inside 20.4 us, so 19.2; 4096 x 4096 with 16384 inside 585, 580).
__device__ __forceinline__ float quotient(float n, float d) {
    const float r = __fdividef(1.f, d), q = n * r;
    return fmaf(fmaf(-q, d, n), r, q);
}
constexpr float SILU_LEAST = -80.f;
__device__ __forceinline__ float silu_above(float v) { return quotient(v, 1.f + expf(-v)); }   // of v > SILU_LEAST
// v e^v / (1 + e^v) below 0: nothing overflows, and small results keep their digits.  (For all values it takes 587 us in place of 580.)
__device__ __forceinline__ float silu(float v) {
    const float t = expf(-fabsf(v));
    return quotient(v >= 0.f ? v : v * t, 1.f + t);
}

}  // namespace w8
