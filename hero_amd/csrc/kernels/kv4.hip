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
constexpr int kXor1 = 0xB1, kXor2 = 0x4E, kHalfMirror = 0x141, kMirror = 0x140, kRor8 = 0x128;

__device__ __forceinline__ double sum16(double v) {
    v += dpp_f64<kXor1>(v);
    v += dpp_f64<kXor2>(v);
    v += dpp_f64<kHalfMirror>(v);
    return v + dpp_f64<kMirror>(v);
}

__device__ __forceinline__ float q4_clean(float x) { return x == x ? fminf(fmaxf(x, -65280.f), 65280.f) : 0.f; }

// the step of a block with largest value hi and smallest lo, as fp16 bits (0 without a sign)
__device__ __forceinline__ uint16_t q4_step(float hi, float lo) {
    const _Float16 h = _Float16((hi >= -lo ? hi : lo) * -0.125f);
    const uint16_t b = __builtin_bit_cast(uint16_t, h);
    const uint32_t size = ((b & 0x7FFFu) + 4u) & 0x7FF8u;
    return uint16_t(size ? size | (b & 0x8000u) : 0u);
}
// x / d to the nearest code (halves to even) + 8: the quotient's rounding may be off by
// one at a border, the remainder x - q d is exact there and decides
__device__ __forceinline__ uint32_t q4_code(float x, float d, float inv) {
    float q = __builtin_rintf(x * inv);
    const float e = __builtin_fmaf(-q, d, x), half = 0.5f * fabsf(d);
    const bool odd = int(q) & 1;
    if (fabsf(e) > half || (fabsf(e) == half && odd)) q += (e < 0.f) == (d < 0.f) ? 1.f : -1.f;
    return d != 0.f ? uint32_t(int(fminf(fmaxf(q, -8.f), 7.f)) + 8) : 8u;
}

__device__ __forceinline__ float4 load4(const float* p) {  // at any float's address
    float4 v;
    __builtin_memcpy(&v, p, 16);
    return v;
}

// Items, 16 lanes each: of every row its query heads, key heads, value heads.
template <int DH>
__global__ __launch_bounds__(256) void kv4_append_kernel(Kv4AppendArgs a) {
    constexpr int H = DH / 128;
    const PagedRows& c = a.c;
    const int l = threadIdx.x & 15;
    const int64_t per = a.Hq + 2 * int64_t(c.Hkv), item = int64_t(blockIdx.x) * 16 + (threadIdx.x >> 4);
    if (item >= per * c.rows) return;
    const int r = int(item / per), head = int(item % per), kind = head < a.Hq ? 0 : head < a.Hq + c.Hkv ? 1 : 2;
    int seq;
    const int pos = row_position(c, r, &seq);
    int at[kRopeAxes];
    bool turns = pos >= 0;
#pragma unroll
    for (int k = 0; k < kRopeAxes; ++k) {
        at[k] = k >= a.axes ? 0 : a.rope_pos ? a.rope_pos[int64_t(k) * c.rows + r] : pos;
        turns = turns && at[k] >= 0 && at[k] < a.rope_positions;
    }
    if (!turns) return;
    const int64_t page = kind == 0 ? 0 : pool_page(c, seq, pos / c.page_size);
    if (page < 0) return;
    const int g = kind == 0 ? head : kind == 1 ? head - a.Hq : head - a.Hq - c.Hkv;
    const float* src = a.proj + int64_t(r) * a.proj_stride + (kind == 0 ? int64_t(g) * 2 * DH : (kind == 1 ? a.k_off : a.v_off) + int64_t(g) * DH);
    const int slot = pos % c.page_size, i = slot % kQ4Tile;
    if (kind == 2) {  // lane b: channels 128 h + 16 m + b
        uint8_t* rec = q4_record<DH>(c, page, 1, g, slot / kQ4Tile);
#pragma unroll
        for (int h = 0; h < H; ++h) {
            float x[8];
#pragma unroll
            for (int m = 0; m < 8; ++m) x[m] = q4_clean(src[128 * h + 16 * m + l]);
            uint32_t word = 0;
            uint16_t mine = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float hi = fmaxf(x[2 * k], x[2 * k + 1]), lo = fminf(x[2 * k], x[2 * k + 1]);
                hi = fmaxf(hi, dpp_f32<kXor1>(hi)), lo = fminf(lo, dpp_f32<kXor1>(lo));
                hi = fmaxf(hi, dpp_f32<kXor2>(hi)), lo = fminf(lo, dpp_f32<kXor2>(lo));
                hi = fmaxf(hi, dpp_f32<kHalfMirror>(hi)), lo = fminf(lo, dpp_f32<kHalfMirror>(lo));
                hi = fmaxf(hi, dpp_f32<kMirror>(hi)), lo = fminf(lo, dpp_f32<kMirror>(lo));
                const uint16_t bits = q4_step(hi, lo);
                const float d = half_bits_to_f32(bits), inv = d != 0.f ? 1.f / d : 0.f;
                if (l == k) mine = bits;
                word |= q4_code(x[2 * k], d, inv) << (8 * k) | q4_code(x[2 * k + 1], d, inv) << (8 * k + 4);
            }
            *reinterpret_cast<uint32_t*>(rec + ((h * 4 + i / 4) * 16 + l) * 16 + i % 4 * 4) = word;
            if (l < 4) *reinterpret_cast<uint16_t*>(rec + 8 * DH + ((i / 4 * (DH / 32) + 4 * h + l) * 4 + i % 4) * 2) = mine;
        }
        return;
    }
    // lane l: channels 128 h + 8 l + j; the other channel of a plane is half a head away
    const float* gamma = kind == 0 ? a.q_gamma : a.k_gamma;
    double x[H][8], ss = 0.0;
#pragma unroll
    for (int h = 0; h < H; ++h) {
        const float4 u = load4(src + 128 * h + 8 * l), v = load4(src + 128 * h + 8 * l + 4);
        const float f[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            x[h][j] = f[j];
            ss = __builtin_fma(x[h][j], x[h][j], ss);
        }
    }
    const double scale = 1.0 / sqrt(sum16(ss) / DH + double(a.eps));
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
        for (int j = 0; j < 8; ++j) x[h][j] *= scale * double(gamma[128 * h + 8 * l + j]);
    const int part = DH == 128 ? l & 7 : l;  // planes 8 part + j
    uint32_t axes = a.axis_bits[0];
#pragma unroll
    for (int k = 1; k < DH / 32; ++k) axes = part / 2 == k ? a.axis_bits[k] : axes;
    axes >>= 16 * (part & 1);
    float y[H][8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int axis = axes >> (2 * j) & 3;
        int p = at[0];
#pragma unroll
        for (int k = 1; k < kRopeAxes; ++k) p = axis == k ? at[k] : p;
        float2 cs;
        __builtin_memcpy(&cs, a.rope_cs + int64_t(p) * DH + 2 * (8 * part + j), 8);
        if constexpr (H == 1) {
            const double other = dpp_f64<kRor8>(x[0][j]);
            y[0][j] = float(l < 8 ? x[0][j] * cs.x - other * cs.y : x[0][j] * cs.x + other * cs.y);
        } else {
            y[0][j] = float(x[0][j] * cs.x - x[H - 1][j] * cs.y);
            y[H - 1][j] = float(x[H - 1][j] * cs.x + x[0][j] * cs.y);
        }
    }
    if (kind == 0) {
        float* out = a.q_rot + (int64_t(r) * a.Hq + g) * DH + 8 * l;
#pragma unroll
        for (int h = 0; h < H; ++h) {
            *reinterpret_cast<float4*>(out + 128 * h) = make_float4(y[h][0], y[h][1], y[h][2], y[h][3]);
            *reinterpret_cast<float4*>(out + 128 * h + 4) = make_float4(y[h][4], y[h][5], y[h][6], y[h][7]);
        }
        return;
    }
    uint8_t* rec = q4_record<DH>(c, page, 0, g, slot / kQ4Tile);
#pragma unroll
    for (int h = 0; h < H; ++h) {
        float hi = -INFINITY, lo = INFINITY;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            y[h][j] = q4_clean(y[h][j]);
            hi = fmaxf(hi, y[h][j]), lo = fminf(lo, y[h][j]);
        }
        hi = fmaxf(hi, dpp_f32<kXor1>(hi)), lo = fminf(lo, dpp_f32<kXor1>(lo));
        hi = fmaxf(hi, dpp_f32<kXor2>(hi)), lo = fminf(lo, dpp_f32<kXor2>(lo));
        const uint16_t bits = q4_step(hi, lo);
        const float d = half_bits_to_f32(bits), inv = d != 0.f ? 1.f / d : 0.f;
        uint32_t word = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) word |= q4_code(y[h][j], d, inv) << (4 * (j / 2 + 4 * (j & 1)));
        *reinterpret_cast<uint32_t*>(rec + ((h * 16 + i) * 16 + (l & 3) * 4 + l / 4) * 4) = word;
        if ((l & 3) == 0) *reinterpret_cast<uint16_t*>(rec + 8 * DH + (i * (DH / 32) + 4 * h + l / 4) * 2) = bits;
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

void launch_kv4_append(const Kv4AppendArgs& a, hipStream_t s) {
    const dim3 grid(groups_of((a.Hq + 2 * int64_t(a.c.Hkv)) * a.c.rows));
    if (a.c.Dh == 256)
        hipLaunchKernelGGL(kv4_append_kernel<256>, grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL(kv4_append_kernel<128>, grid, dim3(256), 0, s, a);
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
