// paged.hpp -- device-side addressing of the paged K/V cache for kernels that
// work on rows of many sequences (PagedRows): positions, sequences and page
// ids come from device memory and are checked before anything is addressed
// with them.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "hero/device.hpp"
#include "hero/kernels.hpp"

namespace hero {

// the row's position, or -1 where the row is left out; its sequence in *seq
__device__ __forceinline__ int row_position(const PagedRows& c, int r, int* seq) {
    const int pos = c.positions[r], s = c.row_seq ? c.row_seq[r] : r;
    *seq = s;
    return (pos >= 0 && int64_t(pos) < int64_t(c.max_pages) * c.page_size && s >= 0 && s < c.seqs) ? pos : -1;
}
// the pool page of logical page lp (in range) of a sequence, or -1
__device__ __forceinline__ int64_t pool_page(const PagedRows& c, int seq, int lp) {
    const int64_t id = c.page_table[int64_t(seq) * c.max_pages + lp];
    return id >= 0 && id < c.pool_pages ? id : -1;
}

// rows of a page in units of DH values: K (kv = 0) or V (kv = 1) of head g, slot t
__device__ __forceinline__ int64_t page_row_index(const PagedRows& c, int kv, int g, int t) { return (int64_t(kv) * c.Hkv + g) * c.page_size + t; }
template <int DH>
__device__ __forceinline__ const _Float16* f16_page(const PagedRows& c, int64_t page) {
    return reinterpret_cast<const _Float16*>(c.pages) + page * (2 * int64_t(c.Hkv) * c.page_size * DH);
}
// Q8_0 pages: the int8 rows, and behind them the fp16 scales (DH / 32 a row)
template <int DH>
__device__ __forceinline__ uint8_t* q8_page(const PagedRows& c, int64_t page) {
    return reinterpret_cast<uint8_t*>(c.pages) + page * (2 * int64_t(c.Hkv) * c.page_size * (DH + DH / 16));
}
template <int DH>
__device__ __forceinline__ int64_t q8_scales_at(const PagedRows& c) { return 2 * int64_t(c.Hkv) * c.page_size * DH; }

// Between the stores and the reads by which the lanes of one wave exchange values
// through shared memory that is the wave's own, and before it is written again.
// The hardware keeps a wave's shared-memory operations in order; to the compiler
// the lanes are threads, and this is what keeps it from moving them.
__device__ __forceinline__ void wave_exchange() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// x >= 0 to 11 significant bits, halves away from zero (the fp16 encoder's
// rounding without fp16's range): products of an integer below 2^24 and two
// such values are exact in 64 bits
__device__ __forceinline__ float round11(float x) { return __uint_as_float((__float_as_uint(x) + 0x1000u) & ~0x1FFFu); }

// roundf(x) for |x| < 2^22 in three instructions: 0.5 less half an ulp carries
// exactly the values whose nearest integer (halves away from zero) is one more
__device__ __forceinline__ int round_code(float x) { return int(x + __builtin_copysignf(0.49999997f, x)); }

}  // namespace hero
