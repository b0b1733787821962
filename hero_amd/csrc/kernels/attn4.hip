// attn4.hip -- gated attention over the 4-bit pages of the paged K/V cache: single
// tokens of many sequences and chunks of prompts, with or without a sliding window
// behind which the first tokens stay visible.
//
// For a (row, query head) pair over the keys j that the row sees, in one pass with a running maximum m:
//   s_j = scale log2(e) q . k_j,   o = sum 2^(s_j - m) v_j,   l = sum 2^(s_j - m),   out = o / l * sigmoid(gate).
// A cached value is an fp16 number (a code times its block's step, exact), so both sums are products for the matrix
// instructions. What they multiply it with is split into two fp16 terms of 22 bits together, queries as well
// as weights, and each product is taken once for each term: results are those of fp32, at twice the products.
// Scores and sums are held in fp32; m lags the true maximum by up to kPSlack, which saves most rescalings.
//
// Three forms. One row of a sequence: the two terms fill the 16 columns of one product with up to 8
// query heads; what counts is the read of the cache (attn4_short_kernel). Chunks: 128 columns of a
// workgroup, 128 / group rows, share the work of turning records into operands, and the products bound it
// (attn4_chunk_kernel). Few rows, and runs of a few rows among chunks: the short kernel again, as the columns'
// other halves would be idle in a chunk's workgroup. Keys are split into ranges where there are few
// workgroups, and combined by a second launch.
//
// Measured, 32 query and 8 K/V heads of 128, in pages of 64 (where two figures stand, on different cards): sixteen tokens of 32000
// keys each 121 to 129 us, 4.9 TB/s of cache
// in the first launch (a copy of gigabytes: 5.1); the same over windows of 4096 26 us; one token of 32000 keys 19.9 us, of which
// about 3 are spent before the first records arrive, 2 after the last ones and 4 on the second launch, and 6 keep the vector units
// busy with turning codes into operands; one token of 300 keys 8.8 us, latencies and instruction fetches (12.1 us with a table of
// 32768 positions, whose 96 ranges are nearly all empty). 500 rows
// over 16000 keys 253 to 266 us, 1.05 to 1.00 PFLOP/s of products (fp16 matrix products of 8192^3 reach 1.17), the same of 16 heads of 256
// 274 us; 1000 rows of three
// sequences over windows of 1024 77 us: 250 workgroups of 34 units each, 44 us for these, about 16 from start to first and from
// last product to end, 5 for the launch that looks for short runs.
#include "hero/device.hpp"
#include "hero/kernels.hpp"
#include "hero/paged.hpp"
#include "hero/q4.hpp"

#include <type_traits>

namespace hero {

namespace {

typedef float f4_t __attribute__((ext_vector_type(4)));
typedef float f2_t __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.4426950408889634f, kLog2eLow = 1.92596303e-8f, kLn2 = 0.6931471805599453f;  // (log2(e) - float(log2(e)))
constexpr float kPOne = 8192.f;  // a weight's terms are of 2^13 2^(s - m); its part in the total is 2^(s - m)
constexpr float kPSlack = 2.f;   // m may lag the maximum by this: weights stay below 2^15
constexpr float kLowest = -3.402823466e38f;

__device__ __forceinline__ float column_other(float x) {  // the value of column c ^ 8
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x128, 0xF, 0xF, true));  // row_ror:8
}
__device__ __forceinline__ int max_of_wave(int x) {
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0xB1, 0xF, 0xF, true));   // quad_perm [1,0,3,2]
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x4E, 0xF, 0xF, true));   // quad_perm [2,3,0,1]
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x141, 0xF, 0xF, true));  // row_half_mirror
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x140, 0xF, 0xF, true));  // row_mirror
    return max(max(__builtin_amdgcn_readlane(x, 0), __builtin_amdgcn_readlane(x, 16)), max(__builtin_amdgcn_readlane(x, 32), __builtin_amdgcn_readlane(x, 48)));
}
__device__ __forceinline__ float max_over_p(float x) {
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float sum_over_p(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}
__device__ __forceinline__ float max_of_8(float x) {  // neighbouring lanes
    x = fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0xB1, 0xF, 0xF, true)));          // quad_perm [1,0,3,2]
    x = fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x4E, 0xF, 0xF, true)));          // quad_perm [2,3,0,1]
    return fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x141, 0xF, 0xF, true)));      // row_half_mirror
}
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }  // 1 ulp; 0 below its range
// 1 / (1 + exp(-x)), 4 ulp: x log2(e) as the product's rounding and what it left; beyond +-200 as there, 1 or 0. (The
// cache's values are 4-bit: nothing here has to replay a reference's rounding, as exp_f32 does.)
__device__ __forceinline__ float gate_of(float x) {
    const float at = -__builtin_amdgcn_fmed3f(x, -200.f, 200.f), t = at * kLog2e;
    const float rest = __builtin_fmaf(at, kLog2eLow, __builtin_fmaf(at, kLog2e, -t));
    const float gate = __builtin_amdgcn_rcpf(1.f + exp2_hw(t) * __builtin_fmaf(rest, kLn2, 1.f));
    return x == x ? gate : x;
}

// x as two fp16 terms; pinned first, so that both are formed from one rounding of it
__device__ __forceinline__ void split_f16(float x, _Float16& hi, _Float16& lo) {
    asm("" : "+v"(x));
    hi = _Float16(x);
    lo = _Float16(x - float(hi));
}

// Two neighbouring codes in the low (F = 0) or second (F = 1) fields of a word's halves, as fp16.
// The masks are kept in registers that the compiler does not see through: it then joins mask and
// or into one instruction, which takes no literals.
struct FieldMasks {
    uint32_t low = 0x000F000Fu, second = 0x00F000F0u, one = 0x64006400u;
    __device__ __forceinline__ FieldMasks() { asm("" : "+s"(low), "+s"(second), "+v"(one)); }
    template <int F>
    __device__ __forceinline__ q4_h2 codes(uint32_t w) const {
        if constexpr (F == 0)  // 0x6400 | c is 1024 + c
            return __builtin_bit_cast(q4_h2, (w & low) | one) - _Float16(1032.f);
        else                   // 0x6400 | c << 4 is 1024 + 16 c
            return __builtin_elementwise_fma(__builtin_bit_cast(q4_h2, (w & second) | one), q4_h2{_Float16(0.0625f), _Float16(0.0625f)},
                                             q4_h2{_Float16(-72.f), _Float16(-72.f)});
    }
};

__device__ __forceinline__ q4_h8 join(q4_h2 a, q4_h2 b, q4_h2 c, q4_h2 d) { return q4_h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]}; }

// A wave's ring of units (two records of keys and of values) in shared memory, filled by
// loads that go there directly: what is in flight takes no registers. Records arrive as
// they lie, 1 KB a load, but for the keys' 16-byte pieces: piece p of key b goes to place
// p ^ (b / 4) of the key's 64 bytes, so that the lanes that read one piece of sixteen keys
// meet every bank once.
template <int DH, int D>
struct Ring {
    static constexpr int H = DH / 128, kLoads = 2 * 3 * H;  // load instructions of a unit
    struct Slot {
        uint4 k[2][H][64], v[2][H][64];
        struct {
            uint8_t k[DH], v[DH];  // next to each other: one load where they are 128 bytes
        } steps[2];
    };
    Slot slot[D];
};
template <int DH, int D>
__device__ __forceinline__ void ring_fetch(typename Ring<DH, D>::Slot& s, int x, const uint8_t* krec, const uint8_t* vrec, int lane) {
    constexpr int H = DH / 128;
#pragma unroll
    for (int h = 0; h < H; ++h) {
        lds_dma_b128(krec + 1024 * h + (lane & ~3) * 16 + ((lane ^ lane >> 4) & 3) * 16, lds_offset(&s.k[x][h][0]));
        lds_dma_b128(vrec + 1024 * h + lane * 16, lds_offset(&s.v[x][h][0]));
    }
    if constexpr (H == 1) {
        const uint8_t* rec = lane < 32 ? krec : vrec - 128;
        lds_dma_b32(rec + 8 * DH + lane * 4, lds_offset(&s.steps[x].k[0]));
    } else {
        lds_dma_b32(krec + 8 * DH + lane * 4, lds_offset(&s.steps[x].k[0]));
        lds_dma_b32(vrec + 8 * DH + lane * 4, lds_offset(&s.steps[x].v[0]));
    }
}

// R rows of up to COLS (row, query head) pairs: pair i is row i / group, head i % group
template <int DH, int COLS>
struct Merge {
    float o[4][COLS][DH], m[4][COLS], l[4][COLS];
};

template <int DH>
__device__ __forceinline__ void store_out(const Attn4Args& a, int r, int h, int ch, float o, float l) {
    const int64_t width = int64_t(a.Hq) * DH, idx = int64_t(r) * width + int64_t(h) * DH + ch;
    const float gate = a.proj[int64_t(r) * a.proj_stride + int64_t(h) * 2 * DH + DH + ch];
    const float out = l == 0.f ? 0.f : (o / l) * gate_of(gate);
    if (a.out_f32) a.out_f32[idx] = out;
    if (a.act_out) {
        float amax = fabsf(out);
        for (int off = 16; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor(amax, off));
        const float d = amax / 127.f, id = d != 0.f ? 1.f / d : 0.f;
        int8_t* qs = static_cast<int8_t*>(a.act_out);
        qs[idx] = int8_t(round_code(out * id));
        if ((ch & 31) == 0) reinterpret_cast<float*>(qs + int64_t(a.c.rows) * width)[idx >> 5] = half_bits_to_f32(fp32_to_fp16_ref(d));
    }
}

// Four neighbouring channels, by neighbouring lanes: channel `at` of the outputs and the next. Returns the step of
// the lane's block of Q8_0, whose place is store_step's.
__device__ __forceinline__ float store_four(const Attn4Args& a, int64_t at, f4_t v, bool live) {
    if (a.out_f32 && live) *reinterpret_cast<f4_t*>(a.out_f32 + at) = v;
    if (!a.act_out) return 0.f;
    const float amax = max_of_8(fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3]))));
    const float d = amax / 127.f, id = d != 0.f ? 1.f / d : 0.f;
    uint32_t codes = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) codes |= uint32_t(round_code(v[i] * id) & 0xFF) << (8 * i);
    if (live) *reinterpret_cast<uint32_t*>(static_cast<int8_t*>(a.act_out) + at) = codes;
    return d;
}
__device__ __forceinline__ void store_step(const Attn4Args& a, int64_t block, float d) {
    reinterpret_cast<float*>(static_cast<int8_t*>(a.act_out) + int64_t(a.c.rows) * a.Hq * a.c.Dh)[block] = half_bits_to_f32(fp32_to_fp16_ref(d));
}

// a row's keys: those below `stay`, and from `first` (>= stay) to `pos`
struct Seen {
    int stay, first, pos;
};
__device__ __forceinline__ Seen row_sees(const Attn4Args& a, int pos) {
    const int first = a.window > 0 ? max(0, pos - a.window + 1) : 0;
    return {a.window > 0 ? min(a.sinks, first) : 0, first, pos};
}

// The four waves' results of `pairs` = rows x group pairs joined, and stored: as the row's where
// the keys were not split, else as this range's.
template <int DH, int COLS>
__device__ __forceinline__ void merge_waves(const Attn4Args& a, const Merge<DH, COLS>& sh, int r0, int rows, int g, int nsplit, int split) {
    const int group = a.Hq / a.c.Hkv;
    for (int idx = threadIdx.x; idx < rows * group * DH; idx += 256) {
        const int k = idx / DH, ch = idx % DH, row = r0 + k / group;
        if (row >= a.c.rows) break;
        float mx = sh.m[0][k];
#pragma unroll
        for (int w = 1; w < 4; ++w) mx = fmaxf(mx, sh.m[w][k]);
        float lt = 0.f, ot = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = exp2_hw(sh.m[w][k] - mx);
            lt += f * sh.l[w][k];
            ot += f * sh.o[w][k][ch];
        }
        ot *= 1.f / kPOne;
        if (nsplit == 1) {
            int s;
            if (row_position(a.c, row, &s) >= 0) store_out<DH>(a, row, g * group + k % group, ch, ot, lt);
        } else {
            float* rec = a.work + ((int64_t(row) * a.Hq + g * group + k % group) * nsplit + split) * (DH + 4);
            if (ch == 0) rec[0] = mx, rec[1] = lt;
            rec[4 + ch] = ot;
        }
    }
}

// The rows of a run: neighbours, of one sequence. A run is short where its (row, query head) pairs fit the 16
// columns of a product. The length of the one that starts in row r, 0 if none does or it is longer than `most`.
__device__ __forceinline__ int short_run(const PagedRows& c, int64_t r, int most) {
    int seq, other;
    if (r >= c.rows || row_position(c, int(r), &seq) < 0 || (r > 0 && row_position(c, int(r) - 1, &other) >= 0 && other == seq)) return 0;
    int n = 1;
    bool on = true;
#pragma unroll 4
    for (int d = 1; d <= most; ++d) {
        const int64_t i = min(r + d, int64_t(c.rows) - 1);
        on = on && row_position(c, int(i), &other) >= 0 && other == seq && r + d < c.rows;
        n += on;
    }
    return n <= most ? n : 0;
}

// One row (ONE), or the short runs of rows b, b + stride, ...: a workgroup of four waves takes one K/V head and
// one of nsplit equal ranges of the run's records, a wave two records (32 keys) at a time. A row alone (PAIR):
// the two terms of up to 8 query heads are the 16 columns, those of head h columns h and h + 8, added where both are
// done. Else the columns are the run's pairs, and each term has a product of its own.
template <int DH, int D, bool ONE>
__global__ __launch_bounds__(256, DH == 128 && ONE ? 3 : 2) void attn4_short_kernel(Attn4Args a, int nsplit, int stride) {
    constexpr int COLS = ONE ? 8 : 16, H = DH / 128, NS = DH / 32, NV = DH / 16;
    const PagedRows& c = a.c;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), p = lane >> 4, b = lane & 15;
    const int split = blockIdx.x % nsplit, g = blockIdx.x / nsplit % c.Hkv, first_row = blockIdx.x / nsplit / c.Hkv;
    const int group = a.Hq / c.Hkv, tpp = c.page_size / kQ4Tile;
    __shared__ union {
        Ring<DH, D> ring[4];
        Merge<DH, COLS> merge;
    } sh;
    const FieldMasks masks;

    auto attend = [&](auto pair, const int r, const int rows) __attribute__((always_inline)) {
        constexpr bool PAIR = decltype(pair)::value;
        const int col = PAIR ? b & 7 : b;
        const int mine = PAIR ? 0 : min(col / group, rows - 1);  // the column's row
        float x[NS][8];
        {
            const float* src = a.q_rot + (int64_t(r + mine) * a.Hq + g * group + (PAIR ? min(col, group - 1) : col % group)) * DH + 8 * p;
#pragma unroll
            for (int s = 0; s < NS; ++s) __builtin_memcpy(x[s], __builtin_assume_aligned(src + 32 * s, 16), 32);
        }
        int seq;
        const int pos0 = row_position(c, r, &seq);
        if (pos0 < 0) return;
        // the run's first and last position
        int pos = pos0, lo = pos0, hi = pos0;
        if constexpr (!PAIR) {
            int s;
            pos = row_position(c, r + mine, &s);
            lo = hi = pos;
            for (int off = 1; off < 16; off <<= 1) lo = min(lo, __shfl_xor(lo, off)), hi = max(hi, __shfl_xor(hi, off));
            lo = __builtin_amdgcn_readfirstlane(lo), hi = __builtin_amdgcn_readfirstlane(hi);
        }
        const Seen sees = row_sees(a, pos), most = row_sees(a, hi), least = row_sees(a, lo);
        // records: those of the first keys that stay, then from the earliest window's first key on
        const int first = least.first / kQ4Tile, stay = min((most.stay + kQ4Tile - 1) / kQ4Tile, first), last = hi / kQ4Tile;
        const int tiles = stay + last - first + 1, units = (tiles + 1) / 2;
        const int u0 = int(uint32_t(units) * uint32_t(split) / uint32_t(nsplit)), u1 = int(uint32_t(units) * uint32_t(split + 1) / uint32_t(nsplit));  // (units at most 2^19, ranges 768)
        // read as constant memory: through the scalar cache, apart from the counted vector loads
        const auto* table = (const __attribute__((address_space(4))) int32_t*)(c.page_table) + int64_t(seq) * c.max_pages;
        const uint32_t magic = (0x80000000u + tpp - 1) / tpp;  // x / tpp = x magic >> 31 for x < 2^23

        struct Place {
            int t;          // record of the sequence
            bool there;
            uint64_t krec;  // offset of the keys' record in the pool
        };
        const uint32_t rec_bytes = 9 * DH, head_bytes = uint32_t(tpp) * rec_bytes, half = head_bytes * c.Hkv;
        auto locate = [&](int k) {
            Place w;
            const int kk = min(k, tiles - 1);
            w.t = kk < stay ? kk : first + kk - stay;
            const int lp = int(uint64_t(w.t) * magic >> 31), id = __builtin_amdgcn_readfirstlane(table[lp]);
            w.there = k < tiles && id >= 0 && id < c.pool_pages;
            w.krec = uint64_t(w.there ? uint32_t(id) : 0u) * (2 * half) + uint32_t(g * head_bytes + (w.t - lp * tpp) * rec_bytes);
            return w;
        };
        Ring<DH, D>& ring = sh.ring[wave];
        auto fetch = [&](int at, const Place (&w)[2]) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const uint8_t* krec = reinterpret_cast<const uint8_t*>(c.pages) + w[x].krec;
                ring_fetch<DH, D>(ring.slot[at], x, krec, krec + half, lane);
            }
        };

        const int n = max(0, (u1 - u0 - wave + 3) / 4);  // the wave's units u0 + wave, + 4, ...
        Place ahead[D][2];
#pragma unroll
        for (int d = 0; d < D; ++d) {
#pragma unroll
            for (int x = 0; x < 2; ++x) ahead[d][x] = locate(2 * (u0 + wave + 4 * d) + x);
        }
        // The queries are in by now, for they wait for nothing; from here on the compiler, which does not see the records' loads, has
        // none of its own to wait for, and the queries turn into operands while the records are on their way.
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int j = 0; j < 8; ++j) asm volatile("" : "+v"(x[s][j]));
#pragma unroll
        for (int d = 0; d < D; ++d)
            if (d < n) fetch(d, ahead[d]);
        // the queries in units of log2, a power of two brings the head's largest channel below 2^14
        q4_h8 q[NS], q2[PAIR ? 1 : NS];
        float unit;
        {
            float amax = 0.f;
            const float k = a.score_scale * kLog2e;
#pragma unroll
            for (int s = 0; s < NS; ++s)
#pragma unroll
                for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(x[s][j] *= k));
            amax = max_over_p(amax);
            const int e = amax > 0.f && amax < INFINITY ? max(ilogbf(amax) + 1, -100) : 0;  // (128 at most: unit and slack are normal)
#pragma unroll
            for (int s = 0; s < NS; ++s)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    _Float16 hi, lo;
                    split_f16(ldexpf(x[s][j], 14 - e), hi, lo);
                    q[s][j] = PAIR && b >= 8 ? lo : hi;
                    if constexpr (!PAIR) q2[s][j] = lo;
                }
            unit = ldexpf(1.f, e - 14);
        }
        const float slack = kPSlack / unit;

        f4_t o[NV];
#pragma unroll
        for (int y = 0; y < NV; ++y) o[y] = f4_t{0.f, 0.f, 0.f, 0.f};
        float m = kLowest, m2 = kLowest, l = 0.f;  // m in units of the products, m2 = m unit

        // (One copy of the body: a wave has few units, and those of a call's first ones are spent on fetching instructions.)
        int at = 0;  // unit i's slot
#pragma unroll 1
        for (int i = 0; i < n; ++i) {
            const Place w[2] = {ahead[0][0], ahead[0][1]};
            const typename Ring<DH, D>::Slot& in = ring.slot[at];
            // the unit's loads are in when at most the ones behind it are outstanding
            if (i + D - 1 < n)
                wait_vmcnt<(D - 1) * Ring<DH, D>::kLoads>();
            else
                wait_vmcnt<0>();
            asm volatile("" ::: "memory");

            float s[8];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                _Float16 kd[NS];
                __builtin_memcpy(kd, __builtin_assume_aligned(in.steps[x].k + b * 2 * NS, 8), sizeof(kd));
                f4_t sum = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < NS; ++k) {
                    const uint4 w4 = in.k[x][k / 4][4 * b + (p ^ b >> 2)];
                    const uint32_t word = k % 4 == 0 ? w4.x : k % 4 == 1 ? w4.y : k % 4 == 2 ? w4.z : w4.w;
                    const q4_h2 d = {kd[k], kd[k]};
                    const q4_h8 f = join(masks.codes<0>(word) * d, masks.codes<1>(word) * d, masks.codes<0>(word >> 8) * d, masks.codes<1>(word >> 8) * d);
                    sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, q[k], sum, 0, 0, 0);
                    if constexpr (!PAIR) sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, q2[k], sum, 0, 0, 0);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) s[4 * x + j] = PAIR ? sum[j] + column_other(sum[j]) : sum[j];
            }
            uint4 v[2][H];
            q4_h2 vd[2][NV];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
#pragma unroll
                for (int h = 0; h < H; ++h) v[x][h] = in.v[x][h][lane];
                __builtin_memcpy(vd[x], __builtin_assume_aligned(in.steps[x].v + p * 4 * NV, 16), sizeof(vd[x]));
            }
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int k0 = kQ4Tile * w[x].t;
                if (!w[x].there || k0 + 15 > lo || (k0 < most.first && k0 + 15 >= least.stay)) {  // some row does not see all of it
                    bool none[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int key = k0 + 4 * p + j;
                        none[j] = !w[x].there || key > hi;
                        if (none[j] || key > pos || (key < sees.first && key >= sees.stay)) s[4 * x + j] = -INFINITY;
                    }
                    // slots past the last row may hold anything: their steps count as 0
#pragma unroll
                    for (int y = 0; y < NV; ++y)
#pragma unroll
                        for (int j = 0; j < 2; ++j)
                            if (none[2 * (y & 1) + j]) vd[x][y][j] = _Float16(0.f);
                }
            }
            // what the slot held is in registers: the next unit's loads may land there
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
            for (int d = 0; d + 1 < D; ++d) ahead[d][0] = ahead[d + 1][0], ahead[d][1] = ahead[d + 1][1];
            if (i + D < n) {
#pragma unroll
                for (int x = 0; x < 2; ++x) ahead[D - 1][x] = locate(2 * (u0 + wave + 4 * (i + D)) + x);
                fetch(at, ahead[D - 1]);
            }
            at = at + 1 == D ? 0 : at + 1;
            float best = s[0];
#pragma unroll
            for (int j = 1; j < 8; ++j) best = fmaxf(best, s[j]);
            if (__ballot(best > m + slack)) {
                const float to = fmaxf(m, max_over_p(best)), to2 = to == kLowest ? kLowest : to * unit, f = exp2_hw(m2 - to2);
                m = to, m2 = to2;
                l *= f;
#pragma unroll
                for (int y = 0; y < NV; ++y) o[y] *= f;
            }
            // Two weights at a time, as two terms of one value (the scaling is exact). Conversions in pairs and
            // remainders in fp32: instructions that round to one half of a register (fma_mixlo) take twice as
            // long. Pinned, or the compiler makes those of them.
            q4_h8 w8, w8l;
            float weights = 0.f;  // (a unit's weights first: roundings of thousands of equal ones would go the same way)
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const float e0 = exp2_hw(__builtin_fmaf(s[j], unit, -m2)), e1 = exp2_hw(__builtin_fmaf(s[j + 1], unit, -m2));
                weights += e0;
                weights += e1;
                const q4_h2 h2 = __builtin_convertvector((f2_t{e0 * kPOne, e1 * kPOne}), q4_h2);
                float d0 = __builtin_fmaf(e0, kPOne, -float(h2[0])), d1 = __builtin_fmaf(e1, kPOne, -float(h2[1]));
                asm volatile("" : "+v"(d0), "+v"(d1));
                const q4_h2 l2 = __builtin_convertvector((f2_t{d0, d1}), q4_h2);
                if constexpr (PAIR) {
                    const q4_h2 t = b < 8 ? h2 : l2;
                    w8[j] = t[0], w8[j + 1] = t[1];
                } else {
                    w8[j] = h2[0], w8[j + 1] = h2[1], w8l[j] = l2[0], w8l[j + 1] = l2[1];
                }
            }
            l += weights;
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
                for (int y = 0; y < 4; ++y) {  // byte y of the words: channels 128 h + 32 y + b and + 16
                    // 16-bit halves: that byte of two neighbouring keys
                    const uint32_t pick = 0x0C040C00u + 0x00010001u * y;
                    const uint32_t w0 = __builtin_amdgcn_perm(v[0][h].y, v[0][h].x, pick), w1 = __builtin_amdgcn_perm(v[0][h].w, v[0][h].z, pick);
                    const uint32_t w2 = __builtin_amdgcn_perm(v[1][h].y, v[1][h].x, pick), w3 = __builtin_amdgcn_perm(v[1][h].w, v[1][h].z, pick);
                    const q4_h2 d0 = vd[0][2 * (4 * h + y)], d1 = vd[0][2 * (4 * h + y) + 1];
                    const q4_h2 d2 = vd[1][2 * (4 * h + y)], d3 = vd[1][2 * (4 * h + y) + 1];
                    f4_t& oa = o[8 * h + 2 * y];
                    f4_t& ob = o[8 * h + 2 * y + 1];
                    const q4_h8 fa = join(masks.codes<0>(w0) * d0, masks.codes<0>(w1) * d1, masks.codes<0>(w2) * d2, masks.codes<0>(w3) * d3);
                    const q4_h8 fb = join(masks.codes<1>(w0) * d0, masks.codes<1>(w1) * d1, masks.codes<1>(w2) * d2, masks.codes<1>(w3) * d3);
                    oa = __builtin_amdgcn_mfma_f32_16x16x32_f16(fa, w8, oa, 0, 0, 0);
                    if constexpr (!PAIR) oa = __builtin_amdgcn_mfma_f32_16x16x32_f16(fa, w8l, oa, 0, 0, 0);
                    ob = __builtin_amdgcn_mfma_f32_16x16x32_f16(fb, w8, ob, 0, 0, 0);
                    if constexpr (!PAIR) ob = __builtin_amdgcn_mfma_f32_16x16x32_f16(fb, w8l, ob, 0, 0, 0);
                }
        }
        __syncthreads();

        // the four waves' results
        l = sum_over_p(l);
#pragma unroll
        for (int y = 0; y < NV; ++y) {
            f4_t v = o[y];
            if constexpr (PAIR) {
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] += column_other(v[i]);
            }
            if (!PAIR || b < 8) *reinterpret_cast<f4_t*>(&sh.merge.o[wave][col][16 * y + 4 * p]) = v;
        }
        if (p == 0 && (!PAIR || b < 8)) sh.merge.m[wave][col] = m2, sh.merge.l[wave][col] = l;
        __syncthreads();
        merge_waves<DH, COLS>(a, sh.merge, r, rows, g, nsplit, split);
    };

    if constexpr (ONE) {
        attend(std::true_type{}, first_row, 1);
    } else {
        for (int64_t base = first_row; base < c.rows; base += 64 * int64_t(stride)) {
            const int found = short_run(c, base + int64_t(lane) * stride, 16 / group);  // by a lane each
            for (uint64_t left = __ballot(found > 0); left; left &= left - 1) {
                const int at = __ffsll((unsigned long long)left) - 1;
                __syncthreads();  // the last run's results are read
                const int r = int(base + int64_t(at) * stride), rows = __builtin_amdgcn_readlane(found, at);
                if (rows == 1)
                    attend(std::true_type{}, r, 1);
                else
                    attend(std::false_type{}, r, rows);
            }
        }
    }
}

// Many rows: a workgroup takes 128 columns, (row, query head) pairs of consecutive rows and one K/V head, 32
// for each of its four waves, and one of nsplit ranges of their keys. The products are of
// 32 x 32 x 16 (lane = 32 f + x below):
//   scores   S^T[key][column]: lane (f, x) brings channels 16 s + 8 f .. + 7 of key x for step s, and gets keys 8 y +
//            4 f + i (register 4 y + i) of column x.
//   values   O^T[channel][column] over the 16 keys of a record: a lane's scores of the record, in order of
//            their registers, are its operand, so lane (f, x) brings keys 4 f + i and 8 + 4 f + i of channel x.
// The waves share the work of turning a unit's records (32 keys) into fp16 operands in shared memory. A unit
// passes in steps: its loads, its operands, its scores, its weights and values, a barrier apart, and
// an iteration holds one step of each of several units: the matrix cores multiply
// the next unit's scores while the vector units form this one's weights, and this
// one's values while they form operands.
constexpr int kListed = 256, kRing = 5;
struct Listed {
    uint64_t krec;   // offset of the keys' record in the pool
    int key, edge;   // its first position (-1: not there); whether some row does not see all of it
};

template <int DH>
__global__ __launch_bounds__(256, DH == 128 ? 2 : 1) void attn4_chunk_kernel(Attn4Args a, int R, int nsplit, int parts) {
    constexpr int H = DH / 128, NS = DH / 16, NB = DH / 32;
    constexpr int WK = NB / 2, WV = 2 * H;  // words of keys, and bytes of words of values, that a lane turns into operands
    typedef float f16_t __attribute__((ext_vector_type(16)));
    const PagedRows& c = a.c;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), f = lane >> 5, p = lane >> 4, b = lane & 15;
    // neighbouring workgroups, which go to different XCDs, take different heads: each L2 holds the records of its own
    const int g = blockIdx.x % c.Hkv, split = blockIdx.x / c.Hkv % nsplit;
    const int tiles_r = (c.rows + R - 1) / R, part = blockIdx.x / c.Hkv / nsplit / tiles_r, r0 = blockIdx.x / c.Hkv / nsplit % tiles_r * R;
    const int group = a.Hq / c.Hkv, tpp = c.page_size / kQ4Tile;
    const uint32_t magic = (0x80000000u + tpp - 1) / tpp;  // x / tpp = x magic >> 31 for x < 2^23
    const uint32_t rec_bytes = 9 * DH, head_bytes = uint32_t(tpp) * rec_bytes, half = head_bytes * c.Hkv;
    const FieldMasks masks;
    const uint8_t* const pool = reinterpret_cast<const uint8_t*>(c.pages);
    struct Units {
        uint4 ops_k[2][NS][64];      // operands, a lane's 16 bytes each
        uint2 ops_v[2][NB][2][64][2];
        struct {
            uint4 codes[2][2][H][64];  // keys, values; record; as they lie
            uint8_t steps[2][2][DH];
        } raw[kRing];
        Listed list[kListed];
    };
    __shared__ union {
        Units units;
        float out[4][32][DH + 4];    // a wave's columns
    } sh;
    auto& ops_k = sh.units.ops_k;
    auto& ops_v = sh.units.ops_v;
    auto& raw = sh.units.raw;
    auto& list = sh.units.list;

    // the workgroup's rows, two a lane
    int row_pos[2], row_of[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int i = lane + 64 * k;
        row_pos[k] = i < R && r0 + i < c.rows ? row_position(c, r0 + i, &row_of[k]) : -1;
    }
    int near_pos[3] = {}, near_seq[3] = {};  // of rows r0 - 16 + lane + 64 k
    if (parts > 1)
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            const int r = r0 - 16 + lane + 64 * k, at = min(max(r, 0), c.rows - 1);
            const int at_pos = row_position(c, at, &near_seq[k]);
            near_pos[k] = r == at ? at_pos : -1;
        }
    // the lane's column, and its query in units of log2, two terms; a power of two brings the head's largest channel below 2^14
    const int col = wave * 32 + (lane & 31), i_row = min(min(col / group, R - 1), c.rows - 1 - r0);
    const int row = col < R * group && r0 + col / group < c.rows ? i_row : -1, head = g * group + col % group;
    q4_h8 qh[NS], ql[NS];
    float unit;
    {
        const float* src = a.q_rot + (int64_t(r0 + i_row) * a.Hq + head) * DH + 8 * f;
        const float k = a.score_scale * kLog2e;
        f4_t x[NS][2];
        float amax = 0.f;
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int j = 0; j < 2; ++j) x[s][j] = *reinterpret_cast<const f4_t*>(src + 16 * s + 4 * j) * k;
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(x[s][j / 4][j % 4]));
        amax = fmaxf(amax, __shfl_xor(amax, 32));
        const int e = amax > 0.f && amax < INFINITY ? max(ilogbf(amax) + 1, -100) : 0;  // (128 at most: unit and slack are normal)
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                _Float16 hi, lo;
                split_f16(ldexpf(x[s][j / 4][j % 4], 14 - e), hi, lo);
                qh[s][j] = hi, ql[s][j] = lo;
            }
        unit = ldexpf(1.f, e - 14);
    }
    const float slack = kPSlack / unit;
    uint64_t valid[2] = {__ballot(row_pos[0] >= 0), __ballot(row_pos[1] >= 0)};
    if (parts > 1) {
        // Rows of short runs are not this kernel's. Bit i of `on`: row r0 - 16 + i goes on the run of the row before
        // it; `most` such bits in a row are a run of more rows than that, and it holds all of them.
        const int most = 16 / group;
        uint64_t on[3], all_on[3], bits[3], in[3];
        int s_last = -1;  // (of row r0 - 17: no window reaches back to it)
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            const int s = near_pos[k] >= 0 ? near_seq[k] : -1, before = __builtin_amdgcn_update_dpp(s_last, s, 0x138, 0xF, 0xF, false);  // wave_shr:1
            on[k] = all_on[k] = bits[k] = __ballot(s >= 0 && s == before);
            s_last = __builtin_amdgcn_readlane(s, 63);
        }
        auto down = [](uint64_t (&v)[3]) { v[0] = v[0] >> 1 | v[1] << 63, v[1] = v[1] >> 1 | v[2] << 63, v[2] >>= 1; };
        auto up = [](uint64_t (&v)[3]) { v[2] = v[2] << 1 | v[1] >> 63, v[1] = v[1] << 1 | v[0] >> 63, v[0] <<= 1; };
        for (int d = 1; d < most; ++d) {
            down(bits);
#pragma unroll
            for (int k = 0; k < 3; ++k) all_on[k] &= bits[k];
        }
#pragma unroll
        for (int k = 0; k < 3; ++k) in[k] = bits[k] = all_on[k];
        for (int d = 1; d < most; ++d) {
            up(bits);
#pragma unroll
            for (int k = 0; k < 3; ++k) in[k] |= bits[k];
        }
        down(all_on);
        valid[0] &= (in[0] | all_on[0]) >> 16 | (in[1] | all_on[1]) << 48;
        valid[1] &= (in[1] | all_on[1]) >> 16 | (in[2] | all_on[2]) << 48;
#pragma unroll
        for (int k = 0; k < 2; ++k)
            if (!(valid[k] >> lane & 1)) row_pos[k] = -1;
    }
    if (!(valid[0] | valid[1])) return;
    const uint64_t all[2] = {valid[0], valid[1]};
    uint64_t done[2] = {0, 0};  // rows of the runs that this workgroup takes
    auto of_row = [&](const int (&v)[2], int i) {
        const int x = __shfl(v[0], i & 63), y = __shfl(v[1], i & 63);  // by all lanes
        return i < 64 ? x : y;
    };
    const int pos = of_row(row_pos, i_row);
    const Seen sees = row_sees(a, pos);
    float m = kLowest, m2 = kLowest, l = 0.f;  // m in units of the products, m2 = m unit
    const f16_t zero = {};
    f16_t o[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n) o[n] = zero;

    // shared memory alone: loads stay in flight across it
    auto barrier = [] {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };

    // The rows of one sequence at a time: mostly there is one. Where a second sequence begins among a workgroup's rows
    // another workgroup (part 1) takes what is not the first's.
    for (int run = 0; (valid[0] | valid[1]) && (parts == 1 || part == 1 || run == 0); ++run) {
        const int lead = valid[0] ? __ffsll((unsigned long long)valid[0]) - 1 : 63 + __ffsll((unsigned long long)valid[1]);
        const int seq = __builtin_amdgcn_readfirstlane(of_row(row_of, lead));
        uint64_t mine[2];
        int lo = 0x7FFFFFFF, hi = -1;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const bool in = row_of[k] == seq && (valid[k] >> lane & 1);
            mine[k] = __ballot(in);
            valid[k] &= ~mine[k];
            if (part == 0 || run > 0) done[k] |= mine[k];
            if (in) lo = min(lo, row_pos[k]), hi = max(hi, row_pos[k]);
        }
        if (part == 1 && run == 0) continue;
        lo = -max_of_wave(-lo), hi = max_of_wave(hi);
        // (columns of rows that this workgroup does not store may hold anything: none of them touches another)
        const bool whole = (mine[0] == all[0] && mine[1] == all[1]) || (parts > 1 && (part == 0 || (run == 1 && !(valid[0] | valid[1]))));
        const bool here = row >= 0 && ((row < 64 ? mine[0] : mine[1]) >> (row & 63) & 1);

        // records: those of the first keys that stay, then from the earliest window to the last row
        const Seen most = row_sees(a, hi), least = row_sees(a, lo);
        const int first = least.first / kQ4Tile, stay = min((most.stay + kQ4Tile - 1) / kQ4Tile, first);
        const int tiles = stay + hi / kQ4Tile - first + 1, units = (tiles + 1) / 2;
        const int u0 = int(uint32_t(units) * uint32_t(split) / uint32_t(nsplit)), u1 = int(uint32_t(units) * uint32_t(split + 1) / uint32_t(nsplit));  // (units at most 2^19, ranges 768)
        if (u0 >= u1) continue;

        // The range's records are looked up by all lanes, kListed at a time: where each is, and whether some row
        // does not see all of it. In the loop that is a read of shared memory and one branch.
        auto look_up = [&](int from) {
            const int k = 2 * from + int(threadIdx.x), at_t = k < stay ? k : first + min(k, tiles - 1) - stay, lp = int(uint64_t(at_t) * magic >> 31), in = at_t - lp * tpp;
            const int id = c.page_table[int64_t(seq) * c.max_pages + lp], k0 = kQ4Tile * at_t;
            const bool there = k < tiles && id >= 0 && id < c.pool_pages;
            Listed e;
            e.krec = uint64_t(there ? uint32_t(id) : 0u) * (2 * half) + uint32_t(g) * head_bytes + uint32_t(in) * rec_bytes;
            e.key = there ? k0 : -1;
            e.edge = !whole || !there || k0 + 15 > lo || (k0 < most.first && k0 + 15 >= least.stay);
            list[threadIdx.x] = e;
        };
        struct Two {
            uint64_t krec0, krec1;
            int at;  // in the list
            bool edge;
        };
        int listed = u0;  // the list's first unit
        auto locate = [&](int u) __attribute__((always_inline)) {
            Two w;
            w.at = 2 * (u - listed);
            const Listed e0 = list[w.at], e1 = list[w.at + 1];
            auto uniform = [](uint64_t v) {
                return uint64_t(uint32_t(__builtin_amdgcn_readfirstlane(int(v >> 32)))) << 32 | uint32_t(__builtin_amdgcn_readfirstlane(int(v)));
            };
            w.krec0 = uniform(e0.krec), w.krec1 = uniform(e1.krec);
            w.edge = __builtin_amdgcn_readfirstlane(e0.edge | e1.edge);
            return w;
        };

        // A unit's records go to shared memory as they lie, five units ahead: each wave moves one record.
        constexpr int kLoads = H + 1;  // instructions of a wave
        auto fetch = [&](uint64_t krec0, uint64_t krec1, int slot) __attribute__((always_inline)) {
            const int kv = wave >> 1, x = wave & 1;
            const uint8_t* rec = pool + (x ? krec1 : krec0) + (kv ? half : 0u);
#pragma unroll
            for (int h = 0; h < H; ++h) lds_dma_b128(rec + 1024 * h + uint32_t(lane * 16), lds_offset(&raw[slot].codes[kv][x][h][0]));
            if (lane < DH / 4) lds_dma_b32(rec + 8 * DH + uint32_t(lane * 4), lds_offset(&raw[slot].steps[kv][x][0]));
        };
        // a wave's share of a unit: half of the words of one record of keys, one byte of every word of both records of values
        uint32_t raw_k[WK];
        _Float16 raw_kd[WK];
        uint4 raw_v[WV];
        q4_h2 raw_vd[WV][2];
        const int k_first = wave / 2 * WK;
        auto take = [&](int slot_k, int slot_v) __attribute__((always_inline)) {
            const uint8_t* codes = reinterpret_cast<const uint8_t*>(&raw[slot_k].codes[0][wave & 1][k_first / 4][0]) + b * 64 + p * 16 + k_first % 4 * 4;
            __builtin_memcpy(raw_k, __builtin_assume_aligned(codes, 4 * WK), sizeof(raw_k));
            __builtin_memcpy(raw_kd, __builtin_assume_aligned(&raw[slot_k].steps[0][wave & 1][(b * NB + k_first) * 2], 2 * WK), sizeof(raw_kd));
#pragma unroll
            for (int j = 0; j < WV; ++j) {
                const int x = j / H, h = j % H;
                raw_v[j] = raw[slot_v].codes[1][x][h][lane];
                __builtin_memcpy(raw_vd[j], __builtin_assume_aligned(&raw[slot_v].steps[1][x][(p * NB + 4 * h + wave) * 8], 8), 8);
            }
        };
        // slots past the last row may hold anything: their steps count as 0
        auto clean_v = [&](int at) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < WV; ++j) {
                const int k0 = list[at + j / H].key;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (k0 < 0 || k0 + 4 * p + i > hi) raw_vd[j][i / 2][i % 2] = _Float16(0.f);
            }
        };
        auto form_k = [&](int at, int s) __attribute__((always_inline)) {
            const uint32_t word = raw_k[s];
            const q4_h2 d = {raw_kd[s], raw_kd[s]};
            ops_k[at][2 * (k_first + s) + p / 2][32 * (p & 1) + 16 * (wave & 1) + b] =
                __builtin_bit_cast(uint4, join(masks.codes<0>(word) * d, masks.codes<1>(word) * d, masks.codes<0>(word >> 8) * d, masks.codes<1>(word >> 8) * d));
        };
        const uint32_t pick = 0x0C040C00u + 0x00010001u * wave;  // a byte of two neighbouring keys, in 16-bit halves
        auto form_v = [&](int at, int j) __attribute__((always_inline)) {
            const int x = j / H, h = j % H;
            const uint32_t w0 = __builtin_amdgcn_perm(raw_v[j].y, raw_v[j].x, pick), w1 = __builtin_amdgcn_perm(raw_v[j].w, raw_v[j].z, pick);
            const q4_h2 d0 = raw_vd[j][0], d1 = raw_vd[j][1];
            uint2(*to)[2] = &ops_v[at][4 * h + wave][x][32 * (p & 1) + b];
            to[0][p / 2] = make_uint2(__builtin_bit_cast(uint32_t, masks.codes<0>(w0) * d0), __builtin_bit_cast(uint32_t, masks.codes<0>(w1) * d1));
            to[16][p / 2] = make_uint2(__builtin_bit_cast(uint32_t, masks.codes<1>(w0) * d0), __builtin_bit_cast(uint32_t, masks.codes<1>(w1) * d1));
        };
        // piece i of WK + WV: the unit's next but one keys, the next values
        auto form = [&](int k_at, int v_at, int i) __attribute__((always_inline)) {
            if (i < WK)
                form_k(k_at, i);
            else
                form_v(v_at, i - WK);
        };
        auto operand_k = [&](int at, int k) __attribute__((always_inline)) { return __builtin_bit_cast(q4_h8, ops_k[at][k][lane]); };
        auto operand_v = [&](int at, int n, int x) __attribute__((always_inline)) { return *reinterpret_cast<const q4_h8*>(&ops_v[at][n][x][lane][0]); };
        barrier();  // the last run's list and operands are done with
        look_up(u0);
        barrier();
        // (units behind the range's last one are read and not used; records behind the last one are page 0's)
        Two w1 = locate(u0 + 1);
        bool edge = false;
        int slot = 0;  // of the unit that comes next
        {
            const Two w0 = locate(u0);
            edge = w0.edge;
            const Two w2 = locate(u0 + 2), w3 = locate(u0 + 3), w4 = locate(u0 + 4);
            fetch(w0.krec0, w0.krec1, 0);
            fetch(w1.krec0, w1.krec1, 1);
            fetch(w2.krec0, w2.krec1, 2);
            fetch(w3.krec0, w3.krec1, 3);
            fetch(w4.krec0, w4.krec1, 4);
        }
        wait_vmcnt<2 * kLoads>();
        barrier();
        take(0, 0);
        if (edge) clean_v(0);
#pragma unroll
        for (int i = 0; i < WK + WV; ++i) form(0, 0, i);
        take(1, 0);
#pragma unroll
        for (int i = 0; i < WK; ++i) form_k(1, i);
        barrier();
        f16_t s = zero;
#pragma unroll
        for (int k = 0; k < NS; ++k) {
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(operand_k(0, k), qh[k], s, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(operand_k(0, k), ql[k], s, 0, 0, 0);
        }
        barrier();
        auto hide = [&](f16_t& s, int at) __attribute__((always_inline)) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int k0 = list[at + x].key;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int key = k0 + 8 * (i / 4) + 4 * f + i % 4;
                    if (!(here && k0 >= 0 && key <= pos && (key >= sees.first || key < sees.stay))) s[8 * x + i] = -INFINITY;
                }
            }
        };
        auto rescale = [&](float best) __attribute__((always_inline)) {
            if (__builtin_expect(__ballot(best > m + slack) != 0, 0)) {
                const float to = fmaxf(m, fmaxf(best, __shfl_xor(best, 32))), to2 = to == kLowest ? kLowest : to * unit, x = exp2_hw(m2 - to2);
                m = to, m2 = to2;
                l *= x;
#pragma unroll
                for (int n = 0; n < NB; ++n) o[n] *= x;
            }
        };
        if (edge) hide(s, 0);
        {
            float best = s[0];
#pragma unroll
            for (int i = 1; i < 16; ++i) best = fmaxf(best, s[i]);
            rescale(best);
        }
        // here: the scores of unit u and their maxima, the keys of u + 1 and the values of u as operands, units u + 1 and
        // u + 2 in shared memory, u + 3 and u + 4 on the way
        auto iterate = [&](const int u, const int now) __attribute__((always_inline)) {
            // The next unit's scores, and between their products this one's weights, ... (The order is kept: the
            // compiler's own has the vector instructions first and the products behind them.)
            f16_t ahead = zero;
            float weights = 0.f;  // (a unit's weights first: roundings of thousands of equal ones would go the same way)
            uint32_t terms_h[8], terms_l[8];
            q4_h8 x_now = operand_k(now ^ 1, 0), x_next = operand_k(now ^ 1, 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int k = 0; k < NS; ++k) {
                const q4_h8 x_then = operand_k(now ^ 1, k + 2 < NS ? k + 2 : k);
                __builtin_amdgcn_sched_barrier(0);
                ahead = __builtin_amdgcn_mfma_f32_32x32x16_f16(x_now, qh[k], ahead, 0, 0, 0);
                if (k % (NS / 8) == 0) {  // two weights, as two terms; pinned to their place in the order
                    const int i = k / (NS / 8);
                    const float e0 = exp2_hw(__builtin_fmaf(s[2 * i], unit, -m2)), e1 = exp2_hw(__builtin_fmaf(s[2 * i + 1], unit, -m2));
                    weights += e0;
                    weights += e1;
                    // Conversions in pairs and remainders in fp32: instructions that round to one half of a
                    // register (fma_mixlo) take twice as long. Pinned, or the compiler makes those of them.
                    const q4_h2 hi = __builtin_convertvector((f2_t{e0 * kPOne, e1 * kPOne}), q4_h2);
                    float d0 = __builtin_fmaf(e0, kPOne, -float(hi[0])), d1 = __builtin_fmaf(e1, kPOne, -float(hi[1]));
                    asm volatile("" : "+v"(d0), "+v"(d1));
                    const q4_h2 lo = __builtin_convertvector((f2_t{d0, d1}), q4_h2);
                    terms_h[i] = __builtin_bit_cast(uint32_t, hi), terms_l[i] = __builtin_bit_cast(uint32_t, lo);
                    asm volatile("" : "+v"(terms_h[i]), "+v"(terms_l[i]));
                }
                ahead = __builtin_amdgcn_mfma_f32_32x32x16_f16(x_now, ql[k], ahead, 0, 0, 0);
                x_now = x_next, x_next = x_then;
                __builtin_amdgcn_sched_barrier(0);
            }
            l += weights;
            q4_h8 wh[2], wl[2];
            __builtin_memcpy(wh, terms_h, 32);
            __builtin_memcpy(wl, terms_l, 32);
            // ... this unit's values, and between their products operands of the units to come and the next unit's maxima
            const int slot1 = slot == kRing - 1 ? 0 : slot + 1, slot2 = slot1 == kRing - 1 ? 0 : slot1 + 1;
            take(slot2, slot1);
            const Two w5 = locate(u + 5), w2 = locate(u + 2);
            fetch(w5.krec0, w5.krec1, slot);  // (unit u's records have been operands since the last barrier)
            q4_h8 v_now[2] = {operand_v(now, 0, 0), operand_v(now, 0, 1)};
            if (__builtin_expect(w1.edge, 0)) {
                clean_v(w1.at);
                hide(ahead, w1.at);
            }
            float best = -INFINITY;
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                const int j = min(i + 1, NB - 1);
                const q4_h8 v_next[2] = {operand_v(now, j, 0), operand_v(now, j, 1)};
                __builtin_amdgcn_sched_barrier(0);
                // (products of one accumulator behind each other: it is passed on, not read again)
                o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v_now[0], wh[0], o[i], 0, 0, 0);
                o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v_now[0], wl[0], o[i], 0, 0, 0);
                form(now, now ^ 1, i);
#pragma unroll
                for (int y = 0; y < 16 / NB; ++y) best = fmaxf(best, ahead[i * (16 / NB) + y]);
                o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v_now[1], wh[1], o[i], 0, 0, 0);
                o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v_now[1], wl[1], o[i], 0, 0, 0);
                v_now[0] = v_next[0], v_now[1] = v_next[1];
                __builtin_amdgcn_sched_barrier(0);
            }
            w1 = w2;
            slot = slot1;
            rescale(best);
            wait_vmcnt<2 * kLoads>();
            barrier();
            s = ahead;
        };
        for (int u = u0; u < u1; u += 2) {
            if (u + 6 >= listed + kListed / 2) {  // the two units' locate would leave the list
                barrier();
                look_up(u);
                w1.at -= 2 * (u - listed);
                listed = u;
                barrier();
            }
            iterate(u, 0);
            if (u + 1 < u1) iterate(u + 1, 1);
        }
    }

    // Results by way of shared memory: register 4 y + i of block n is channel 32 n + 8 y + 4 f + i of the column, and then
    // a lane takes four neighbouring channels of one column (or, of 128, of every other) after another. Stores of whole
    // rows, and a short loop where the columns' own order unrolls to 24 KB of instructions that every call fetches anew.
    const float total = l + __shfl_xor(l, 32);
    const bool live = row >= 0 && ((row < 64 ? done[0] : done[1]) >> (row & 63) & 1);
    wait_vmcnt<0>();
    barrier();
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int y = 0; y < 4; ++y)
            *reinterpret_cast<f4_t*>(&sh.out[wave][lane & 31][32 * n + 8 * y + 4 * f]) = f4_t{o[n][4 * y], o[n][4 * y + 1], o[n][4 * y + 2], o[n][4 * y + 3]};
    if (f == 0) {  // behind a column its (row, query head), -1: none, and what else is known of it
        const int r = live ? r0 + row : r0;
        const float pair = __int_as_float(live ? r * a.Hq + head : -1), share = total == 0.f ? 0.f : 1.f / (total * kPOne);
        *reinterpret_cast<f4_t*>(&sh.out[wave][lane][DH]) = nsplit > 1 ? f4_t{pair, m2, total, 0.f} : f4_t{pair, share, __int_as_float(r), __int_as_float(head)};
    }
    wave_exchange();
    constexpr int kAtOnce = 8, kColumns = 256 / DH;
    const int ch = 4 * lane % DH;
#pragma unroll 1
    for (int k = 4 * lane / DH; k < 32; k += kAtOnce * kColumns) {
        f4_t of[kAtOnce], gate[kAtOnce];
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) of[j] = *reinterpret_cast<const f4_t*>(&sh.out[wave][k + j * kColumns][DH]);
        if (nsplit == 1)  // a round's loads together: one by one they were half of the time of a short call
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j)
                __builtin_memcpy(&gate[j], a.proj + int64_t(__float_as_int(of[j][2])) * a.proj_stride + int64_t(__float_as_int(of[j][3])) * 2 * DH + DH + ch, 16);
        float step = 0.f;  // of every eighth column, by its eight lanes one each
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {
            const int64_t pair = __float_as_int(of[j][0]);
            f4_t v = *reinterpret_cast<const f4_t*>(&sh.out[wave][k + j * kColumns][ch]);
            if (nsplit > 1) {
                if (pair >= 0) {
                    float* rec = a.work + (pair * nsplit + split) * (DH + 4);
                    if (ch == 0) rec[0] = of[j][1], rec[1] = of[j][2];
                    *reinterpret_cast<f4_t*>(rec + 4 + ch) = v * (1.f / kPOne);
                }
                continue;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = of[j][1] == 0.f ? 0.f : v[i] * of[j][1] * gate_of(gate[j][i]);
            const float d = store_four(a, pair * DH + ch, v, pair >= 0);
            step = (lane & 7) == j ? d : step;
        }
        if (nsplit == 1 && a.act_out)
            if (const int64_t pair = __float_as_int(sh.out[wave][k + (lane & 7) * kColumns][DH]); pair >= 0) store_step(a, pair * (DH / 32) + ch / 32, step);
    }
}

// Few ranges: DH / 4 lanes for a (row, query head), four channels each
constexpr int kFewRanges = 8;
template <int DH, int N>
__global__ __launch_bounds__(256) void attn4_combine_few_kernel(Attn4Args a, int nsplit) {
    constexpr int LN = DH / 4, kRec = DH + 4;
    const int64_t item = int64_t(blockIdx.x) * (256 / LN) + threadIdx.x / LN;
    const int ch = threadIdx.x % LN * 4;
    if (item >= int64_t(a.c.rows) * a.Hq) return;
    const int r = int(item / a.Hq), h = int(item % a.Hq);
    int seq;
    if (row_position(a.c, r, &seq) < 0) return;
    const float* rec = a.work + item * nsplit * kRec;
    f4_t v[N];
    float m[N], l[N], mx = kLowest;
#pragma unroll
    for (int s = 0; s < N; ++s) {
        const float* at = rec + min(s, nsplit - 1) * kRec;
        m[s] = at[0], l[s] = at[1];
        v[s] = *reinterpret_cast<const f4_t*>(at + 4 + ch);
    }
    const float* gates = a.proj + int64_t(r) * a.proj_stride + int64_t(h) * 2 * DH + DH + ch;
    float gate[4];
    __builtin_memcpy(gate, gates, 16);
#pragma unroll
    for (int s = 0; s < N; ++s) mx = fmaxf(mx, m[s]);
    float total = 0.f;
    f4_t o = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < N; ++s) {
        const float f = s < nsplit ? exp2_hw(m[s] - mx) : 0.f;
        total += f * l[s];
        o += s < nsplit ? f * v[s] : f4_t{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = total == 0.f ? 0.f : o[i] / total * gate_of(gate[i]);
    const int64_t at = (int64_t(r) * a.Hq + h) * DH + ch;
    const float d = store_four(a, at, o, true);
    if (a.act_out && ch % 32 == 0) store_step(a, at / 32, d);
}

// A workgroup per (row, query head): DH / 4 lanes for four channels each read a range's result, and
// 1024 / DH such groups take the ranges in turn.
template <int DH>
__global__ __launch_bounds__(256) void attn4_combine_kernel(Attn4Args a, int nsplit) {
    constexpr int LN = DH / 4, GR = 256 / LN, kRec = DH + 4, kPass = 4;
    const int r = blockIdx.x / a.Hq, h = blockIdx.x % a.Hq, t = threadIdx.x, grp = t / LN, ln = t % LN;
    int seq;
    if (row_position(a.c, r, &seq) < 0) return;
    __shared__ float part[GR][DH], total[4], most[4];
    extern __shared__ float share[];  // a range's factor
    const float* rec = a.work + int64_t(blockIdx.x) * nsplit * kRec;
    float mx = kLowest;
    for (int s = t; s < nsplit; s += 256) mx = fmaxf(mx, rec[int64_t(s) * kRec]);
    for (int off = 32; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off));
    if ((t & 63) == 0) most[t >> 6] = mx;
    __syncthreads();
    mx = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
    float l = 0.f;
    for (int s = t; s < (nsplit + GR * kPass - 1) / (GR * kPass) * (GR * kPass); s += 256) {
        float f = 0.f;
        if (s < nsplit) {
            f = exp2_hw(rec[int64_t(s) * kRec] - mx);
            l += f * rec[int64_t(s) * kRec + 1];
        }
        share[s] = f;
    }
    for (int off = 32; off > 0; off >>= 1) l += __shfl_xor(l, off);
    if ((t & 63) == 0) total[t >> 6] = l;
    __syncthreads();
    f4_t o = f4_t{0.f, 0.f, 0.f, 0.f};
    for (int s = grp; s < nsplit; s += GR * kPass) {
        f4_t v[kPass];
#pragma unroll
        for (int k = 0; k < kPass; ++k) v[k] = *reinterpret_cast<const f4_t*>(rec + int64_t(min(s + GR * k, nsplit - 1)) * kRec + 4 + 4 * ln);
#pragma unroll
        for (int k = 0; k < kPass; ++k) o += share[s + GR * k] * v[k];
    }
    *reinterpret_cast<f4_t*>(&part[grp][4 * ln]) = o;
    __syncthreads();
    if (t < DH) {
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < GR; ++k) v += part[k][t];
        store_out<DH>(a, r, h, t, v, (total[0] + total[1]) + (total[2] + total[3]));
    }
}

// Rows a workgroup takes, and into how many ranges their keys are split. Tokens and few rows: as many workgroups as are
// there at once, three per CU of single rows of 128-wide heads and else two (with three, eight rows over 16000 keys of 256-wide
// heads take 46 us instead of 42, four rows of one sequence over 32000 34 instead of 26), eight units of 32 keys each at least. Chunks: one workgroup per CU with at least eight units; two (of 128-wide heads, of which two
// fit) where one would have 45 units or more: two that share a CU are ahead of one in the long run, but the ranges'
// combination costs 5 to 10 us. 500 rows over 16000 keys, 258 units: 284 us in two ranges, 262 in four; 300 rows over
// 4000, 45 units: 65 in four, 63 in six; 1000 rows over 2500, 94 units: 127 in one, 123 in two; over windows of 1024, 34 units: 52 and
// 61; 500 rows of two sequences over 2250, 35 units: 82 in two, 89 in four. All of this goes by what the table has room for, which the host knows, and
// not by the rows' positions, which are the device's.
enum class Form { token, few, chunk };
struct Plan {
    int R, nsplit;
    int64_t tiles, groups, most;  // groups of rows; workgroups at most where keys are split; ranges that the keys allow
};
Plan attn4_plan(Form form, int64_t rows, int64_t seqs, int64_t group, int64_t Hkv, int64_t Dh, int64_t span, int64_t window, int64_t sinks) {
    Plan p;
    p.R = form == Form::token ? 1 : int((form == Form::few ? 16 : 128) / group);
    p.groups = form != Form::token || Dh == 256 ? 512 : 768;
    const int64_t keys = window > 0 ? std::min(span, window + sinks + p.R + 2 * kQ4Tile) : span, units = (keys + 31) / 32;
    p.tiles = form == Form::few && seqs > 1 ? rows : (rows + p.R - 1) / p.R;  // (rows of several sequences are mostly alone)
    p.most = std::max<int64_t>(1, units / 8);
    const int64_t each = p.tiles * Hkv;
    if (form != Form::chunk) {
        p.nsplit = int(std::max<int64_t>(1, std::min(p.groups / each, p.most)));
    } else {
        const int64_t one = std::max<int64_t>(1, std::min(256 / each, p.most)), two = Dh == 128 ? std::min(p.groups / each, p.most) : 1;
        p.nsplit = int(units >= 45 * one ? std::max(one, two) : one);
    }
    return p;
}
// rows that belong to sequences of their own have no keys in common; few rows are short runs, however they stand (four rows of one
// sequence over 16000 keys 23.6 us, as a chunk 32.2; over 1000 keys 16.8 and 23.0)
Form attn4_form(bool row_seq, int64_t rows, int64_t group) { return !row_seq || rows == 1 ? Form::token : rows * group <= 16 ? Form::few : Form::chunk; }

}  // namespace

// Room for any call of up to `rows` rows, of any form: where there are several ranges, the workgroups are
// at most p.groups, of R * group results each.
int64_t attn4_work_bytes(int64_t rows, int64_t Hq, int64_t Hkv, int64_t Dh, int64_t span, int64_t window, int64_t sinks) {
    int64_t slots = 0;
    for (const Form form : {Form::token, Form::few, Form::chunk}) {
        const Plan p = attn4_plan(form, rows, 1, Hq / Hkv, Hkv, Dh, span, window, sinks);
        if (p.most > 1) slots = std::max(slots, std::min(p.groups, p.tiles * Hkv * p.most) * p.R * (Hq / Hkv));
    }
    return slots * (Dh + 4) * 4;
}

namespace {
template <int DH>
void attn4_sized(const Attn4Args& a, hipStream_t s) {
    const int64_t rows = a.c.rows, Hkv = a.c.Hkv, group = a.Hq / Hkv;
    const Form form = attn4_form(a.c.row_seq, rows, group);
    const Plan p = attn4_plan(form, rows, a.c.seqs, group, Hkv, DH, int64_t(a.c.max_pages) * a.c.page_size, a.window, a.sinks);
    const bool runs = form == Form::few || (form == Form::chunk && a.c.seqs > 1);  // short ones, to be found
    if (form == Form::token)
        hipLaunchKernelGGL((attn4_short_kernel<DH, 2, true>), dim3(unsigned(rows * Hkv * p.nsplit)), dim3(256), 0, s, a, p.nsplit, 1);
    if (runs) {
        // two workgroups per CU are there at once: with three, 64 tokens of 8000 keys take 220 us instead of 210
        const int64_t stride = std::min(rows, std::max<int64_t>(1, 512 / (Hkv * p.nsplit)));
        hipLaunchKernelGGL((attn4_short_kernel<DH, 2, false>), dim3(unsigned(stride * Hkv * p.nsplit)), dim3(256), 0, s, a, p.nsplit, int(stride));
    }
    if (form == Form::chunk) {
        const int parts = runs ? 2 : 1;
        hipLaunchKernelGGL(attn4_chunk_kernel<DH>, dim3(unsigned(p.tiles * Hkv * p.nsplit * parts)), dim3(256), 0, s, a, p.R, p.nsplit, parts);
    }
    if (p.nsplit == 1) return;
    const int64_t heads = rows * a.Hq;
    const dim3 few(unsigned((heads * (DH / 4) + 255) / 256));
    if (p.nsplit <= kFewRanges / 2)
        hipLaunchKernelGGL((attn4_combine_few_kernel<DH, kFewRanges / 2>), few, dim3(256), 0, s, a, p.nsplit);
    else if (p.nsplit <= kFewRanges)
        hipLaunchKernelGGL((attn4_combine_few_kernel<DH, kFewRanges>), few, dim3(256), 0, s, a, p.nsplit);
    else
        hipLaunchKernelGGL(attn4_combine_kernel<DH>, dim3(unsigned(heads)), dim3(256), size_t(p.nsplit + 31) / 32 * 128, s, a, p.nsplit);
}
}  // namespace

void launch_attn4(const Attn4Args& a, hipStream_t s) {
    a.c.Dh == 256 ? attn4_sized<256>(a, s) : attn4_sized<128>(a, s);
}

}  // namespace hero
