// q4.hpp -- the 4-bit pages of the paged K/V cache: what a record holds, and
// how a wave turns it into matrix operands.
//
// A block of 32 neighbouring channels stands for codes -8 .. 7 times a step of 8
// significant bits, held as fp16: every product has at most 11 bits and is exact
// in fp16, so rows of 4-bit pages multiply on the fp16 matrix cores without a
// rounding of their own. Sixteen positions of a head are one record of 9 DH
// bytes, 8 DH of codes + 8 (two to a byte), then DH of steps; a page is
// [2 = K, V][Hkv][page_size / 16] records. 4.5 bits a value.
//
// Within a record the codes lie as the lanes of a wave want them (lane = 16 p + b
// below): a lane's 16 bytes at 1024 h + 16 lane are its share of a product, so
// every load is 1 KB in one piece.
//   keys    [DH / 128 = h][16 positions][4 = p][4 = a][4 bytes]: a word holds
//           channels 128 h + 32 a + 8 p + j; its fields, lowest first, are j = 0, 2,
//           4, 6, 1, 3, 5, 7, so that masking a word (and the word >> 8) leaves two
//           neighbours in its halves. Steps [16 positions][DH / 32].
//   values  [DH / 128 = h][4 = p][16 = b][4 = i][4 bytes]: position 4 p + i, field
//           m is channel 128 h + 16 m + b. Steps [4 = p][DH / 32][4 = i].
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "hero/kernels.hpp"

namespace hero {

typedef _Float16 q4_h2 __attribute__((ext_vector_type(2)));
typedef _Float16 q4_h8 __attribute__((ext_vector_type(8)));

constexpr int kQ4Tile = 16;  // positions of a record

template <int DH>
__device__ __forceinline__ uint8_t* q4_record(const PagedRows& c, int64_t page, int kv, int g, int tile) {
    const int64_t tiles = c.page_size / kQ4Tile;
    return reinterpret_cast<uint8_t*>(c.pages) + ((page * 2 + kv) * c.Hkv + g) * tiles * (9 * DH) + int64_t(tile) * (9 * DH);
}

}  // namespace hero
