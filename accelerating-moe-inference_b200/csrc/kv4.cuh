// Granule layout of the paged 4-bit cache (include/moe_b200.h): 16 tokens of
// one head, codes then (scale, minimum) pairs.
#pragma once

#include <cuda_runtime.h>

namespace moe {

// Bytes of a granule: codes of K and V (16 * D / 2 each), then their params.
__host__ __device__ constexpr int kv4_granule(int D) { return 16 * D + 128 * (D / 64); }

// Byte offset of the 32-bit word with dims [8 m, 8 m + 8) of token t's key:
// [16 tokens][4 j][G g][2 h], dims 64 g + 16 j + 8 h.
template <int D> __device__ __forceinline__ int kv4_k_word(int t, int m) {
    constexpr int G = D / 64;
    const int g = m >> 3, j = (m >> 1) & 3, h = m & 1;
    return t * (D / 2) + ((j * G + g) * 2 + h) * 4;
}

// The same for its value: [G p][8 n][4 j][4 / G v][G g], dims 64 g + 8 n.
template <int D> __device__ __forceinline__ int kv4_v_word(int t, int m) {
    constexpr int G = D / 64, V = 4 / G;
    const int g = m >> 3, n = m & 7;
    const int u = (t >> 3) * 2 + (t & 1), j = (t & 7) >> 1;
    return 8 * D + ((((u / V) * 8 + n) * 4 + j) * V + u % V) * G * 4 + g * 4;
}

}  // namespace moe
