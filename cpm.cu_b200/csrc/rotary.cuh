// Rotation of fused q/k/v rows with their append to a cache, for any layout of the pairs (rotary.cu).
#pragma once
#include "op_errors.cuh"

struct RotaryArgs {
    const bf16* qkv = nullptr;        // rows of heads + 2 kv_heads heads of `dim`, ld elements apart
    long long ld = 0;
    int heads = 0, kv_heads = 0, dim = 0;
    int half = 0;                     // rotated pairs per head
    const float* inv_freq = nullptr;  // [half]
    float factor = 1.f;               // of sines and cosines
    const int32_t* pos = nullptr;
    bf16* q = nullptr;                // rows of `heads` heads, ldq elements apart
    long long ldq = 0;
    bf16 *k_cache = nullptr, *v_cache = nullptr;   // [cache_rows, kv_heads * dim]
    int cache_rows = 0;
    const int32_t* slots = nullptr;
    OpCount* errors = nullptr;
};
int rotary_max_pairs();
void launch_rotary(const RotaryArgs& a, int rows, bool interleaved, cudaStream_t s);
