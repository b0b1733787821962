// kv4.hip -- rows of many sequences into the 4-bit pages of the paged K/V cache
// and back: query / key norms, rotary positions of one to four axes, 4-bit blocks.
//
// A block of 32 channels: m its value of largest magnitude (of two such the
// positive one), d = -m / 8 as fp16 (to nearest even), its magnitude then rounded to 8
// significant bits (halves up; below fp16's normal range to multiples of 2^-21), codes
// clamp(round(x / d), -8, 7), halves to even. The sign of the step puts m on the code
// -8, which has no counterpart. NaN counts as 0, what lies past +-65280 as that.
//
// Codes jump where x / d crosses a half, so a key that is off by an fp32 rounding
// may get another code than the formulas give. Norm and rotation are therefore
// formed in 64 bits and rounded to fp32 once, and the codes are decided on exact
// remainders: what is stored does not depend on the order of a sum.
#include "hero/device.hpp"
#include "hero/kernels.hpp"
#include "hero/paged.hpp"
#include "hero/q4.hpp"

namespace hero {

namespace {

// Sixteen lanes of a wave work on one head of one row.
template <int CTRL>
__device__ __forceinline__ float dpp_f32(float v) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, false)); }
template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
    const int2 x = __builtin_bit_cast(int2, v);
    return __builtin_bit_cast(double, make_int2(__builtin_amdgcn_update_dpp(0, x.x, CTRL, 0xF, 0xF, false), __builtin_amdgcn_update_dpp(0, x.y, CTRL, 0xF, 0xF, false)));
}
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t v) { return uint32_t(__builtin_amdgcn_update_dpp(0, int(v), CTRL, 0xF, 0xF, false)); }
constexpr int kXor1 = 0xB1, kXor2 = 0x4E, kHalfMirror = 0x141, kMirror = 0x140, kRor8 = 0x128, kXor3 = 0x1B;

__device__ __forceinline__ double sum16(double v) {
    v += dpp_f64<kXor1>(v);
    v += dpp_f64<kXor2>(v);
    v += dpp_f64<kHalfMirror>(v);
    return v + dpp_f64<kMirror>(v);
}

// the step of a block with largest value hi and smallest lo, as fp16 bits (0 without a sign)
__device__ __forceinline__ uint16_t q4_step(float hi, float lo) {
    const _Float16 h = _Float16((hi >= -lo ? hi : lo) * -0.125f);
    const uint16_t b = __builtin_bit_cast(uint16_t, h);
    const uint32_t size = ((b & 0x7FFFu) + 4u) & 0x7FF8u;
    return uint16_t(size ? size | (b & 0x8000u) : 0u);
}
// Eight values of a block (four lanes hold it) to codes + 8, a nibble each, and the block's step.
__device__ __forceinline__ uint32_t q4_codes(float (&x)[8], uint16_t* step) {
    float hi, lo, zero = 0.f;
    auto bounds = [&] {
        hi = lo = x[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) hi = fmaxf(hi, x[j]), lo = fminf(lo, x[j]);
    };
    bounds();
#pragma unroll
    for (int j = 0; j < 8; ++j) zero = __builtin_fmaf(x[j], 0.f, zero);
    if (!(zero == 0.f && hi <= 65280.f && lo >= -65280.f)) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = x[j] == x[j] ? fminf(fmaxf(x[j], -65280.f), 65280.f) : 0.f;
        bounds();
    }
    hi = fmaxf(hi, dpp_f32<kXor1>(hi)), lo = fminf(lo, dpp_f32<kXor1>(lo));
    hi = fmaxf(hi, dpp_f32<kXor2>(hi)), lo = fminf(lo, dpp_f32<kXor2>(lo));
    *step = q4_step(hi, lo);
    const float d = half_bits_to_f32(*step), inv = d != 0.f ? 1.f / d : 0.f;
    // 1.5 * 2^23 + 8 + q has q + 8 in its lowest bits, rounded to the nearest (halves to even)
    constexpr float kBig = 12582920.f;
    uint32_t word = 0;
    float far = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float q = __builtin_amdgcn_fmed3f(x[j] * inv, -8.f, 7.f), to = q + kBig;
        far = fmaxf(far, fabsf(q - (to - kBig)));
        word += (__float_as_uint(to) - 0x4B400000u) << (4 * j);
    }
    // The quotient is off by up to 2^-23 of itself, 2^-20 here: where one is that near to a half, the remainder
    // x - q d, which is exact there, decides.
    if (far >= 0.499998f) {
        word = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float q = __builtin_rintf(x[j] * inv);
            const float e = __builtin_fmaf(-q, d, x[j]), half = 0.5f * fabsf(d);
            const bool odd = int(q) & 1;
            if (fabsf(e) > half || (fabsf(e) == half && odd)) q += (e < 0.f) == (d < 0.f) ? 1.f : -1.f;
            word |= uint32_t(int(fminf(fmaxf(q, -8.f), 7.f)) + 8) << (4 * j);
        }
    }
    return word;
}

// Nibbles 0 2 4 6 1 3 5 7 of a word.
__device__ __forceinline__ uint32_t gather_nibbles(uint32_t w) {
    uint32_t even = w & 0x0F0F0F0Fu, odd = w >> 4 & 0x0F0F0F0Fu;
    even = (even | even >> 4) & 0x00FF00FFu, odd = (odd | odd >> 4) & 0x00FF00FFu;
    return __builtin_amdgcn_perm(odd, even, 0x06040200u);
}
// Eight words of eight nibbles, of the lanes of one l & 1: afterwards nibble m of lane l is nibble l / 2 of lane 2 m + (l & 1).
__device__ __forceinline__ uint32_t transpose_nibbles(uint32_t w, int l) {
    w = __builtin_amdgcn_perm(dpp_u32<kRor8>(w), w, l & 8 ? 0x03020706u : 0x05040100u);
    w = __builtin_amdgcn_perm(dpp_u32<kXor3>(dpp_u32<kHalfMirror>(w)), w, l & 4 ? 0x03070105u : 0x06020400u);
    const uint32_t of = dpp_u32<kXor2>(w), mine = l & 2 ? 0xF0F0F0F0u : 0x0F0F0F0Fu;
    return (w & mine) | ((l & 2 ? of >> 4 : of << 4) & ~mine);
}

__device__ __forceinline__ void load8(float (&v)[8], const float* p) {  // at any float's address
    __builtin_memcpy(v, p, 16);
    __builtin_memcpy(v + 4, p + 4, 16);
}

// Sixteen lanes take N heads of a row, queries, keys or values, which share its positions, its angles and the norm's
// weights; a workgroup takes the same N heads of sixteen rows, so that the words of neighbouring positions, which lie side by side in a
// record, leave one L2 cache together (1000 rows with consecutive heads in a workgroup instead: 16.3 us, so 14.5). Lane l: channels
// 128 h + 8 l + j. What does not depend on the position is loaded beside it, and rows that are left out go through it
// all up to the stores.
//
// What bounds it: with many rows the memory: 4000 rows of 32 + 16 heads move 165 MB in 37 us, 4.4 TB/s; 1000 rows 14.5 us,
// of which about 5 are launch, first loads and last stores, and the vector units are busy for 6. One row: the chain
// position, page and angles, stores: 4.6 us.
template <int DH, int N>
__global__ __launch_bounds__(256) void kv4_append_kernel(Kv4AppendArgs a) {
    constexpr int H = DH / 128;
    const PagedRows& c = a.c;
    const int l = threadIdx.x & 15;
    const int of_q = (a.Hq + N - 1) / N, of_k = (c.Hkv + N - 1) / N;
    const int per = of_q + 2 * of_k, r = int(blockIdx.x / per) * 16 + int(threadIdx.x >> 4);
    if (r >= c.rows) return;
    const int part = int(blockIdx.x % per), kind = part < of_q ? 0 : part < of_q + of_k ? 1 : 2;
    int seq, at[kRopeAxes];
    const int pos = row_position(c, r, &seq);
#pragma unroll
    for (int k = 0; k < kRopeAxes; ++k) at[k] = k >= a.axes ? 0 : a.rope_pos ? a.rope_pos[int64_t(k) * c.rows + r] : pos;
    const int head = N * (kind == 0 ? part : kind == 1 ? part - of_q : part - of_q - of_k), n = min(N, (kind == 0 ? a.Hq : c.Hkv) - head);
    const int64_t step = kind == 0 ? 2 * DH : DH;
    const float* src = a.proj + int64_t(r) * a.proj_stride + (kind == 0 ? 0 : kind == 1 ? a.k_off : a.v_off) + head * step + 8 * l;
    const float* gamma = (kind == 0 ? a.q_gamma : a.k_gamma) + 8 * l;
    float x[N][H][8], weight[H][8];
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int h = 0; h < H; ++h) load8(x[i][h], src + min(i, n - 1) * step + 128 * h);
#pragma unroll
    for (int h = 0; h < H; ++h) load8(weight[h], gamma + 128 * h);
    bool stays = pos < 0;
#pragma unroll
    for (int k = 0; k < kRopeAxes; ++k) stays = stays || at[k] < 0 || at[k] >= a.rope_positions;
    const int64_t page = pool_page(c, stays ? 0 : seq, stays ? 0 : pos / c.page_size);
    stays = stays || (kind != 0 && page < 0);
    if (kind != 2) {
        const int planes = DH == 128 ? l & 7 : l;  // 8 planes + j: the other channel of a plane is half a head away
        uint32_t axes = a.axis_bits[0];
#pragma unroll
        for (int k = 1; k < DH / 32; ++k) axes = planes / 2 == k ? a.axis_bits[k] : axes;
        axes >>= 16 * (planes & 1);
        // norm weight and angle together: a channel turned is scale (own x + cross (the other x))
        double own[H][8], cross[H][8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int axis = axes >> (2 * j) & 3;
            int p = at[0];
#pragma unroll
            for (int k = 1; k < kRopeAxes; ++k) p = axis == k ? at[k] : p;
            float2 cs;
            __builtin_memcpy(&cs, a.rope_cs + int64_t(stays ? 0 : p) * DH + 2 * (8 * planes + j), 8);
            if constexpr (H == 1) {
                own[0][j] = double(cs.x) * double(weight[0][j]);
                cross[0][j] = double(l < 8 ? -cs.y : cs.y) * double(dpp_f32<kRor8>(weight[0][j]));
            } else {
                own[0][j] = double(cs.x) * double(weight[0][j]), own[1][j] = double(cs.x) * double(weight[1][j]);
                cross[0][j] = double(-cs.y) * double(weight[1][j]), cross[1][j] = double(cs.y) * double(weight[0][j]);
            }
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            double v[H][8], ss = 0.0;
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    v[h][j] = x[i][h][j];
                    ss = __builtin_fma(v[h][j], v[h][j], ss);
                }
            const double scale = rsqrt(sum16(ss) * (1.0 / DH) + double(a.eps));
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if constexpr (H == 1) {
                    x[i][0][j] = float(scale * __builtin_fma(v[0][j], own[0][j], double(dpp_f32<kRor8>(x[i][0][j])) * cross[0][j]));
                } else {
                    x[i][0][j] = float(scale * __builtin_fma(v[0][j], own[0][j], v[1][j] * cross[0][j]));
                    x[i][1][j] = float(scale * __builtin_fma(v[1][j], own[1][j], v[0][j] * cross[1][j]));
                }
            }
        }
    }
    if (stays) return;
    const int slot = pos % c.page_size, t = slot % kQ4Tile;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (i >= n) break;
        const int g = head + i;
        if (kind == 0) {
            float* out = a.q_rot + (int64_t(r) * a.Hq + g) * DH + 8 * l;
#pragma unroll
            for (int h = 0; h < H; ++h) __builtin_memcpy(__builtin_assume_aligned(out + 128 * h, 16), x[i][h], 32);
            continue;
        }
        uint8_t* rec = q4_record<DH>(c, page, kind - 1, g, slot / kQ4Tile);
#pragma unroll
        for (int h = 0; h < H; ++h) {
            uint16_t d;
            uint32_t word = q4_codes(x[i][h], &d);
            int at = ((h * 16 + t) * 16 + (l & 3) * 4 + l / 4) * 4, step_at = t * (DH / 32) + 4 * h + l / 4;
            if (kind == 1) {
                // nibble j to place j / 2 + 4 (j & 1)
                word = gather_nibbles(word);
            } else {
                word = transpose_nibbles(word, l);
                at = ((h * 4 + t / 4) * 16 + 8 * (l & 1) + l / 2) * 16 + t % 4 * 4;
                step_at = (t / 4 * (DH / 32) + 4 * h + l / 4) * 4 + t % 4;
            }
            *reinterpret_cast<uint32_t*>(rec + at) = word;
            if ((l & 3) == 0) *reinterpret_cast<uint16_t*>(rec + 8 * DH + 2 * step_at) = d;
        }
    }
}

// Items, 16 lanes each: of every row its key heads, then its value heads; a lane
// holds the channels of one word.
template <int DH, typename T>
__global__ __launch_bounds__(256) void kv4_read_kernel(KvReadArgs a) {
    const PagedRows& c = a.c;
    const int l = threadIdx.x & 15;
    const int64_t item = int64_t(blockIdx.x) * 16 + (threadIdx.x >> 4);
    if (item >= 2 * int64_t(c.Hkv) * c.rows) return;
    const int r = int(item / (2 * c.Hkv)), what = int(item % (2 * c.Hkv)) / c.Hkv, g = int(item % c.Hkv);
    T* out = static_cast<T*>(a.out[what]);
    int seq;
    const int pos = row_position(c, r, &seq);
    if (!out || pos < 0) return;
    const int64_t page = pool_page(c, seq, pos / c.page_size);
    if (page < 0) return;
    const int slot = pos % c.page_size, i = slot % kQ4Tile;
    const uint8_t* rec = q4_record<DH>(c, page, what, g, slot / kQ4Tile);
    out += (int64_t(r) * c.Hkv + g) * DH;
#pragma unroll
    for (int h = 0; h < DH / 128; ++h) {
        if (what == 0) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(rec + ((h * 16 + i) * 16 + (l & 3) * 4 + l / 4) * 4);
            const float d = half_bits_to_f32(*reinterpret_cast<const uint16_t*>(rec + 8 * DH + (i * (DH / 32) + 4 * h + l / 4) * 2));
            T y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = T(float(int(w >> (4 * (j / 2 + 4 * (j & 1))) & 15) - 8) * d);
            __builtin_memcpy(__builtin_assume_aligned(out + 128 * h + 8 * l, 16), y, sizeof(y));
        } else {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(rec + ((h * 4 + i / 4) * 16 + l) * 16 + i % 4 * 4);
#pragma unroll
            for (int m = 0; m < 8; ++m) {
                const float d = half_bits_to_f32(*reinterpret_cast<const uint16_t*>(rec + 8 * DH + ((i / 4 * (DH / 32) + 4 * h + m / 2) * 4 + i % 4) * 2));
                out[128 * h + 16 * m + l] = T(float(int(w >> (4 * m) & 15) - 8) * d);
            }
        }
    }
}

unsigned groups_of(int64_t items) { return unsigned((items + 15) / 16); }

}  // namespace

namespace {
template <int DH, int N>
void kv4_append_sized(const Kv4AppendArgs& a, hipStream_t s) {
    const int64_t groups = ((a.Hq + N - 1) / N + 2 * int64_t((a.c.Hkv + N - 1) / N)) * ((a.c.rows + 15) / 16);
    hipLaunchKernelGGL((kv4_append_kernel<DH, N>), dim3(unsigned(groups)), dim3(256), 0, s, a);
}
template <int DH, int N>
void kv4_append(const Kv4AppendArgs& a, hipStream_t s) {
    if ((a.Hq + 2 * int64_t(a.c.Hkv)) * a.c.rows < 24 * 1024)  // one head: 256 rows of 48 heads 6.9 us (four: 7.9), 1000 rows 17.0 (14.5)
        kv4_append_sized<DH, 1>(a, s);
    else
        kv4_append_sized<DH, N>(a, s);
}
}  // namespace

void launch_kv4_append(const Kv4AppendArgs& a, hipStream_t s) {
    if (a.c.Dh == 256)
        kv4_append<256, 2>(a, s);
    else
        kv4_append<128, 4>(a, s);
}

namespace {
template <int DH>
void kv4_read_typed(const KvReadArgs& a, hipStream_t s) {
    const dim3 grid(groups_of(2 * int64_t(a.c.Hkv) * a.c.rows));
    if (a.f16)
        hipLaunchKernelGGL((kv4_read_kernel<DH, _Float16>), grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((kv4_read_kernel<DH, float>), grid, dim3(256), 0, s, a);
}
}  // namespace

void launch_kv4_read(const KvReadArgs& a, hipStream_t s) {
    if (a.c.Dh == 256)
        kv4_read_typed<256>(a, s);
    else
        kv4_read_typed<128>(a, s);
}

}  // namespace hero
