// Layout of the 4-bit K/V cache pages, shared by the store and attention kernels.
//
// A page holds page_size positions of one request (page_size a multiple of 16), per K/V head
// as page_size / 16 tiles of 16 positions.  Every K or V vector of hd values is cut into
// groups of 64 dims (the last one shorter); a group is stored as 4-bit codes c with an fp16
// scale s and an fp16 bias b and stands for s c + b.  Dim 8 w + i of a vector is in bits
// 4 i .. 4 i + 3 of its code word w < nw = hd / 8.  In 32-bit words, a tile is
//   K codes:  word w of position r at 64 j + 2 (min(4, nw - 4 j) (r % 8) + w % 4) + r / 8, j = w / 4
//   V codes:  word w of position r at 16 nw + 16 w + 4 ((r % 8) / 2) + 2 (r / 8) + r % 2
//   (s, b) of group n (one word, s in the low half) at 32 nw + 32 n + 4 (r % 8) + 2 (V: 1, K: 0) + r / 8
// so that in the matrix instruction's fragment order (lane 4 g + t) a lane's K words of
// positions g and g + 8 are one 8-byte load, its V words of positions 2 t, 2 t + 1, 2 t + 8 and
// 2 t + 9 one 16-byte load and its K and V (s, b) of positions g and g + 8 another, each warp
// load covering whole 128-byte lines.
#pragma once

#include "common.cuh"

namespace msb {

constexpr int KV4_GROUP = 64;  // dims per (scale, bias)
constexpr int KV4_TILE = 16;   // positions per tile

__host__ __device__ __forceinline__ int kv4_words(int hd) { return hd >> 3; }
__host__ __device__ __forceinline__ int kv4_groups(int hd) { return (hd + KV4_GROUP - 1) / KV4_GROUP; }
__host__ __device__ __forceinline__ int kv4_tile_words(int hd) { return 32 * kv4_words(hd) + 32 * kv4_groups(hd); }

__host__ __device__ __forceinline__ int kv4_k_word(int nw, int w, int r) {
    const int j = w >> 2, left = nw - 4 * j, tw = left < 4 ? left : 4;
    return 64 * j + 2 * (tw * (r & 7) + (w & 3)) + (r >> 3);
}
__host__ __device__ __forceinline__ int kv4_v_word(int nw, int w, int r) {
    return 16 * nw + 16 * w + 4 * ((r & 7) >> 1) + 2 * (r >> 3) + (r & 1);
}
__host__ __device__ __forceinline__ int kv4_meta_word(int nw, int n, int r, int v) {
    return 32 * nw + 32 * n + 4 * (r & 7) + 2 * v + (r >> 3);
}

}  // namespace msb
