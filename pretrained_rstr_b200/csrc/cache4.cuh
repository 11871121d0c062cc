// The paged cache held in 4 bits: where a page's bytes lie, and the small device functions its kernels share.
//
// Rows of head_dim channels go in groups of 32 (the last may be shorter).  A group keeps two bfloat16
// numbers, step = (largest - smallest) / 15 and middle = smallest + 8 step, and a code c of 4 bits a channel,
// the nearest with value middle + step * (c - 8).  The middle is kept rather than the smallest number: it is
// nearer to zero, so its rounding to 8 bits of mantissa is worth less against the step.
//
// A page of one key/value head is one tile of page_size * (head_dim / 2 + 4 * groups) bytes: group by group the
// rows' codes (16 bytes a row, 8 in a group of 16 channels; channel i of the group in bits 4 (i % 8) of its word
// i / 8), then for every row its groups' (step, middle) pairs.  One tile is one stretch of memory, so a bulk copy
// fetches it whole; with 16 bytes between rows, the 8 rows x 4 words that a warp reads at a time as a matrix
// operand lie in the 32 banks of shared memory without a conflict, at every head size.
#pragma once
#include "common.cuh"

namespace cache4 {
constexpr int GROUP = 32;                 // channels that share a step and a middle
constexpr int MAX_HEAD_DIM = 128;

__host__ __device__ __forceinline__ int groups_of(int head_dim) { return (head_dim + GROUP - 1) / GROUP; }
__host__ __device__ __forceinline__ int tile_bytes(int head_dim, int page_size) {
    return page_size * (head_dim / 2 + 4 * groups_of(head_dim));
}
// Where word `w` (channels 8 w to 8 w + 7) of row `at` lies in a tile.
__device__ __forceinline__ int code_word(int head_dim, int page_size, int at, int w) {
    const int g = w >> 2, row = head_dim - g * GROUP >= GROUP ? 16 : (head_dim - g * GROUP) / 2;
    return g * page_size * 16 + at * row + (w & 3) * 4;
}
// Head sizes are multiples of 16 (a matrix instruction's reduction) up to 128, pages multiples of 16
// positions: every piece of a tile is then a multiple of 16 bytes.
__host__ __device__ __forceinline__ bool takes(int head_dim, int page_size) {
    return head_dim >= 16 && head_dim <= MAX_HEAD_DIM && head_dim % 16 == 0 && page_size >= 16 && page_size % 16 == 0 &&
           page_size <= 1024;
}
}  // namespace cache4
