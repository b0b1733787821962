// sparse.hip -- attention over selected pages of the paged K/V cache.
//
// Selection: the page summaries (kvcache.hip) bound every stored key, so
//   sum_c max(q_c max_c, q_c min_c)
// bounds a query's dot product with any key of the page. It is formed on 8-bit
// codes: the query of a head as round(q / d), d = amax / 127, the bounds as
// stored; with q+ = max(q, 0) and q- = max(-q, 0) it is the integer product
// [q+ | q-] . [max | -min]. Both steps are kept to 11 bits, so
// step_q * step_page * integer is exact in 64 bits and the order of the scores
// does not depend on any order of summation. A page's score for a K/V head is
// the largest of its query heads'. The first `sink` and the last `recent`
// pages a row sees are always taken; of the others the best, equal scores by
// ascending page; NaN scores (non-finite keys or queries) rank last.
//
// Attention: softmax(scale * q . k) over the positions of the selected pages
// up to the row's own, then the sum of the values, the sigmoid gate and the
// Q8_0 quantization (nm/src/qwen35.hpp:387-393). A row nothing is selected for
// gets zeros.
#include "hero/device.hpp"
#include "hero/kernels.hpp"
#include "hero/paged.hpp"

namespace hero {

namespace {

// ---- selection ----------------------------------------------------------------------
// order-preserving key of a score; 0 is kept for pages that cannot be taken
__device__ __forceinline__ uint64_t score_key(double s) {
    if (s != s) return 1;
    const int64_t b = __double_as_longlong(s + 0.0);  // -0 counts as 0
    return b < 0 ? ~uint64_t(b) : uint64_t(b) | (uint64_t(1) << 63);
}

// a workgroup per (row, K/V head, 256 pages), a lane per page
template <int DH>
__global__ __launch_bounds__(256) void page_scores_kernel(SelectArgs a) {
    const PagedRows& c = a.c;
    const int tid = threadIdx.x, r = blockIdx.x / c.Hkv, g = blockIdx.x % c.Hkv, group = a.Hq / c.Hkv;
    int seq;
    const int pos = row_position(c, r, &seq);
    if (pos < 0) return;
    const int visible = pos / c.page_size + 1;
    if (visible <= a.top || int(blockIdx.y) * 256 >= visible) return;
    __shared__ int8_t q[8][DH];
    __shared__ float step[8];
    for (int h = tid >> 6; h < group; h += 4) {
        const float* x = a.q_rot + (int64_t(r) * a.Hq + g * group + h) * DH;
        float amax = 0.f;
        for (int j = tid & 63; j < DH; j += 64) amax = fmaxf(amax, fabsf(x[j]));
        for (int off = 32; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor(amax, off));
        const float d = amax / 127.f, id = d != 0.f ? 1.f / d : 0.f;
        for (int j = tid & 63; j < DH; j += 64) q[h][j] = int8_t(int(roundf(x[j] * id)));
        if ((tid & 63) == 0) step[h] = round11(d);
    }
    __syncthreads();
    const int page = blockIdx.y * 256 + tid;
    if (page >= visible) return;
    const int64_t id = pool_page(c, seq, page);
    double s = -INFINITY;
    if (id >= 0) {
        const int8_t* b = reinterpret_cast<const int8_t*>(c.summaries + id * kv_summary_page_bytes(c.Hkv, DH));
        const float d = reinterpret_cast<const float*>(b + int64_t(c.Hkv) * 2 * DH)[g];
        b += int64_t(g) * 2 * DH;
        for (int h = 0; h < group; ++h) {
            int sum = 0;
            for (int j = 0; j < DH; ++j) sum += q[h][j] > 0 ? int(q[h][j]) * b[j] : -int(q[h][j]) * b[DH + j];
            s = fmax(s, double(sum) * double(step[h]));
        }
        s *= double(d);
    } else {
        s = __longlong_as_double(0x7ff8000000000000ll);
    }
    a.keys[(int64_t(r) * c.Hkv + g) * c.max_pages + page] = score_key(s);
}

// a wave per (row, K/V head): the top-th largest key bit by bit, then the
// pages above it and the first of its equals, in order
__global__ __launch_bounds__(64) void page_select_kernel(SelectArgs a) {
    const PagedRows& c = a.c;
    const int lane = threadIdx.x, r = blockIdx.x / c.Hkv, g = blockIdx.x % c.Hkv;
    int32_t* out = a.selected + (int64_t(r) * c.Hkv + g) * a.top;
    int seq;
    const int pos = row_position(c, r, &seq);
    const int visible = pos < 0 ? 0 : pos / c.page_size + 1;
    if (visible <= a.top) {
        for (int i = lane; i < a.top; i += 64) out[i] = i < visible ? i : -1;
        return;
    }
    const uint64_t* keys = a.keys + (int64_t(r) * c.Hkv + g) * c.max_pages;
    auto key = [&](int i) { return i >= visible ? 0 : i < a.sink || i >= visible - a.recent ? ~uint64_t(0) : keys[i]; };
    uint64_t t = 0;  // the largest t with at least top keys >= t
    for (int bit = 63; bit >= 0; --bit) {
        const uint64_t u = t | (uint64_t(1) << bit);
        int n = 0;
        for (int i = lane; i - lane < visible; i += 64) n += __popcll(__ballot(key(i) >= u));
        if (n >= a.top) t = u;
    }
    int above = 0;
    for (int i = lane; i - lane < visible; i += 64) above += __popcll(__ballot(key(i) > t));
    int equal = a.top - above, at = 0;
    const uint64_t below = (uint64_t(1) << lane) - 1;
    for (int i = lane; i - lane < visible && at < a.top; i += 64) {
        const uint64_t k = key(i), eq = __ballot(k == t);
        const bool take = k > t || (k == t && __popcll(eq & below) < equal);
        const uint64_t m = __ballot(take);
        if (take) out[at + __popcll(m & below)] = i;
        at += __popcll(m);
        equal -= min(equal, int(__popcll(eq)));
    }
}

// ---- attention ----------------------------------------------------------------------
// A workgroup of four waves per (row, K/V head, range of its list); a wave
// takes 32 key slots at a time, two halves of 16 that each lie in one page.
//
// Both products run on the matrix cores with every operand where its load or
// the product before put it, nothing through shared memory and no lane
// exchanged (lane = 16 g + c below):
//   scores   S^T[key][column] = K Q^T, 16 keys x 16 columns x 32 channels. Lane
//            (g, c) loads 16 bytes of key c, and gets the scores of keys 4 g ..
//            4 g + 3 for column c.
//   values   O^T[channel][column] += V^T P^T, 16 channels x 16 columns x 32
//            keys. The order of the 32 keys is free as long as both operands
//            agree, so a lane's eight scores (keys 4 g .. 4 g + 3 of both
//            halves) are its operand, and lane (g, c) loads those keys'
//            channels 8 c .. 8 c + 7: whole rows per load, transposed in the
//            lane's registers. Product e covers channels 8 c + e, and a lane
//            ends with 32 consecutive channels of its column's head.
// The matrix cores multiply fp16; queries and weights are fp32. Each is split
// into two fp16 terms (22 bits). A head's query is scaled by a power of two to
// at most 1 first, and a weight is 2^13 e^(s - m) with m at most 2 (base 2) below
// the running maximum, so that neither term leaves fp16's range: terms are
// dropped below 2^-38 of the largest. Keys and values of fp16 pages are exact, and
// the up to eight heads of a group times two terms are the 16 columns (head h
// in columns h and h + 8, added at the end).
// Q8_0 pages: codes are exact in fp16. A key block's product is scaled by the
// block's step afterwards. A value block's step goes into the weights: column
// (block, head) holds weights times that block's steps, for four heads at a
// time, and of its result the 32 channels of that block count. The steps'
// power of two is kept apart per column (`ve`), as theirs range as widely as
// fp16 does.
typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
typedef float f4_t __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kPShift = 13.f;  // weights are 2^13 2^(s - m)
constexpr float kPSlack = 2.f;   // m may lag the maximum by this: weights stay below 2^15

__device__ __forceinline__ float column_other(float x) {  // the value of column c ^ 8
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x128, 0xF, 0xF, false));  // row_ror:8
}
__device__ __forceinline__ float max_over_rows(float x) {  // over the four g of a column
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float sum_over_rows(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}
// 2^x for x <= 15 (the hardware's, good to 1 ulp; 0 below its range)
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// x as two fp16 terms. The value is pinned first: the compiler otherwise rounds
// a product that ends in x straight to fp16 for one use (v_fma_mixlo_f16) and by
// way of fp32 for the other, and where the two round apart lo no longer belongs
// to hi (seen as 2^-11 of one key's weight in every 2^13).
__device__ __forceinline__ void split_f16(float x, _Float16& hi, _Float16& lo) {
    asm("" : "+v"(x));
    hi = _Float16(x);
    lo = _Float16(x - float(hi));
}

// int8 codes to fp16, exact: 0x6400 | (b ^ 0x80) is 1024 + 128 + b
__device__ __forceinline__ h2_t codes_to_half(uint32_t zero_extended) {
    return __builtin_bit_cast(h2_t, zero_extended ^ 0x64806480u) - _Float16(1152.f);
}
__device__ __forceinline__ h8_t codes8_to_half(uint2 w) {
    h8_t r;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const h2_t h = codes_to_half(__builtin_amdgcn_perm(0u, k < 2 ? w.x : w.y, (k & 1) ? 0x0c030c02u : 0x0c010c00u));
        r[2 * k] = h[0];
        r[2 * k + 1] = h[1];
    }
    return r;
}

// rows of the lists of a range, in shared memory: the pool page and how many of
// its keys the row sees (0: none)
struct ListEntry {
    int32_t page, keys;
};

template <int DH>
struct SparseMerge {  // the four waves' results
    float m[4][8], l[4][8], o[4][8][DH];
};

template <int DH>
__device__ __forceinline__ void sparse_store(const SparseAttnArgs& a, int r, int h, int ch, float o, float l) {
    const int64_t width = int64_t(a.Hq) * DH, idx = int64_t(r) * width + int64_t(h) * DH + ch;
    const float gate = a.proj[int64_t(r) * a.proj_stride + int64_t(h) * 2 * DH + DH + ch];
    const float out = l == 0.f ? 0.f : (o / l) * sigmoid_f32(gate);
    if (a.out_f32) a.out_f32[idx] = out;
    if (a.act_out) {
        float amax = fabsf(out);
        for (int off = 16; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor(amax, off));
        const float d = amax / 127.f, id = d != 0.f ? 1.f / d : 0.f;
        int8_t* qs = static_cast<int8_t*>(a.act_out);
        qs[idx] = int8_t(int(roundf(out * id)));
        if ((ch & 31) == 0) reinterpret_cast<float*>(qs + int64_t(a.c.rows) * width)[idx >> 5] = half_bits_to_f32(fp32_to_fp16_ref(d));
    }
}

// GQ: quads of query heads (Q8_0 pages), 1 otherwise
template <int DH, bool Q8, int GQ>
__global__ __launch_bounds__(256) void attn_sparse_kernel(SparseAttnArgs a, int per, int nsplit) {
    constexpr int KB = DH / 32, VH = DH / 128;  // 32-channel blocks, 128-channel halves
    const PagedRows& c = a.c;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, g4 = lane >> 4, c16 = lane & 15;
    // K/V head fastest: with eight of them each XCD's L2 holds one head's pages
    const int g = blockIdx.x % c.Hkv, r = blockIdx.x / c.Hkv % c.rows, split = blockIdx.x / c.Hkv / c.rows;
    const int group = a.Hq / c.Hkv, ps = c.page_size;
    int seq;
    const int pos = row_position(c, r, &seq);
    if (pos < 0) return;
    extern __shared__ __align__(16) ListEntry list[];
    __shared__ __align__(16) SparseMerge<DH> mg;
    const int e0 = split * per, ne = min(per, a.top - e0);
    for (int i = tid; i < ne; i += 256) {
        const int lp = a.selected[(int64_t(r) * c.Hkv + g) * a.top + e0 + i];
        ListEntry e{0, 0};
        if (lp >= 0 && lp <= pos / ps) {
            const int64_t page = pool_page(c, seq, lp);
            if (page >= 0) e = {int32_t(page), min(ps, pos + 1 - lp * ps)};
        }
        list[i] = e;
    }

    // the column's head and its query terms: fp16 pages take term c / 8 of head
    // c % 8; Q8_0 pages both terms of head 4 quad + c % 4
    const float* q_row = a.q_rot + (int64_t(r) * a.Hq + int64_t(g) * group) * DH;
    h8_t qf[GQ][Q8 ? 2 : 1][KB];
    float qscale[GQ];
#pragma unroll
    for (int x = 0; x < GQ; ++x) {
        const int h = Q8 ? 4 * x + (c16 & 3) : c16 & 7;
        const bool have = h < group;
        float q[KB][8], amax = 0.f;
#pragma unroll
        for (int k = 0; k < KB; ++k)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                q[k][j] = have ? q_row[h * DH + 32 * k + 8 * g4 + j] : 0.f;
                amax = fmaxf(amax, fabsf(q[k][j]));
            }
        amax = max_over_rows(amax);
        const int e = __builtin_amdgcn_frexp_expf(amax);  // amax <= 2^e
        qscale[x] = ldexpf(a.score_scale * kLog2e, e);
#pragma unroll
        for (int k = 0; k < KB; ++k)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                _Float16 hi, lo;
                split_f16(ldexpf(q[k][j], -e), hi, lo);
                if constexpr (Q8) {
                    qf[x][0][k][j] = hi;
                    qf[x][1][k][j] = lo;
                } else {
                    qf[x][0][k][j] = c16 < 8 ? hi : lo;
                }
            }
    }
    float m[GQ], l[GQ];
    f4_t o[GQ][8 * VH];
#pragma unroll
    for (int x = 0; x < GQ; ++x) {
        m[x] = -INFINITY;
        l[x] = 0.f;
#pragma unroll
        for (int e = 0; e < 8 * VH; ++e) o[x][e] = f4_t{0.f, 0.f, 0.f, 0.f};
    }
    int ve = -200;  // Q8_0: the column's accumulators are in units of 2^ve
    __syncthreads();

    const int hp = ps / 16, halves = ne * hp;
    for (int u = w; 2 * u < halves; u += 4) {
        int page[2], off[2], nv[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int hf = min(2 * u + s, halves - 1), e = hf / hp;
            const ListEntry le = list[e];
            off[s] = (hf - e * hp) * 16;
            page[s] = __builtin_amdgcn_readfirstlane(le.page);
            nv[s] = 2 * u + s < halves ? __builtin_amdgcn_readfirstlane(max(0, min(16, le.keys - off[s]))) : 0;
        }
        if (nv[0] + nv[1] == 0) continue;
        if (nv[0] == 0) page[0] = page[1], off[0] = off[1];  // an entry of none names no page: read what is there, use nothing
        if (nv[1] == 0) page[1] = page[0], off[1] = off[0];
        const bool full = nv[0] + nv[1] == 32;

        f4_t s[GQ][2];
        if constexpr (!Q8) {
            h8_t kf[2][KB], vf[VH][8];
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                const _Float16* p = f16_page<DH>(c, page[hf]) + page_row_index(c, 0, g, off[hf] + c16) * DH + 8 * g4;
#pragma unroll
                for (int k = 0; k < KB; ++k) kf[hf][k] = *reinterpret_cast<const h8_t*>(p + 32 * k);
            }
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                const _Float16* p = f16_page<DH>(c, page[hf]) + page_row_index(c, 1, g, off[hf] + 4 * g4) * DH + 8 * c16;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int v = 0; v < VH; ++v) vf[v][4 * hf + i] = *reinterpret_cast<const h8_t*>(p + i * DH + 128 * v);
            }
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                f4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < KB; ++k) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[hf][k], qf[0][0][k], acc, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; ++i) s[0][hf][i] = (acc[i] + column_other(acc[i])) * qscale[0];
            }
            if (!full) {
#pragma unroll
                for (int hf = 0; hf < 2; ++hf)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (4 * g4 + i >= nv[hf]) {
                            s[0][hf][i] = -INFINITY;
#pragma unroll
                            for (int v = 0; v < VH; ++v) vf[v][4 * hf + i] = h8_t{};
                        }
            }
            float top = s[0][0][0];
#pragma unroll
            for (int i = 1; i < 8; ++i) top = fmaxf(top, s[0][i >> 2][i & 3]);
            if (__any(top > m[0] + kPSlack)) {
                const float m2 = fmaxf(m[0], max_over_rows(top)), f = m2 == -INFINITY ? 1.f : exp2_hw(m[0] - m2);
                m[0] = m2;
                l[0] *= f;
#pragma unroll
                for (int e = 0; e < 8 * VH; ++e) o[0][e] *= f;
            }
            const float base = m[0] - kPShift;
            h8_t pf;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float p = exp2_hw(s[0][i >> 2][i & 3] - base);
                l[0] += p;
                _Float16 hi, lo;
                split_f16(p, hi, lo);
                pf[i] = c16 < 8 ? hi : lo;
            }
#pragma unroll
            for (int v = 0; v < VH; ++v)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    h8_t x;
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] = vf[v][i][e];
                    o[0][8 * v + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, pf, o[0][8 * v + e], 0, 0, 0);
                }
        } else {
            uint2 kq[2][KB], vq[8];
            uint4 kd[2][2], vd[2][2];
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                const uint8_t* pg = q8_page<DH>(c, page[hf]);
                const int64_t kr = page_row_index(c, 0, g, off[hf]), vr = page_row_index(c, 1, g, off[hf]);
                const uint8_t* kp = pg + (kr + c16) * DH + 8 * g4;
#pragma unroll
                for (int k = 0; k < KB; ++k) kq[hf][k] = *reinterpret_cast<const uint2*>(kp + 32 * k);
                const uint4* kdp = reinterpret_cast<const uint4*>(pg + q8_scales_at<DH>(c) + (kr + 4 * g4) * (2 * KB));
                kd[hf][0] = kdp[0];
                kd[hf][1] = kdp[1];
                const uint8_t* vp = pg + (vr + 4 * g4) * DH + 8 * c16;
#pragma unroll
                for (int i = 0; i < 4; ++i) vq[4 * hf + i] = *reinterpret_cast<const uint2*>(vp + i * DH);
                const uint4* vdp = reinterpret_cast<const uint4*>(pg + q8_scales_at<DH>(c) + (vr + 4 * g4) * (2 * KB));
                vd[hf][0] = vdp[0];
                vd[hf][1] = vdp[1];
            }
            // scores: a block's product, then the key's step of that block
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                h8_t steps[2] = {__builtin_bit_cast(h8_t, kd[hf][0]), __builtin_bit_cast(h8_t, kd[hf][1])};  // [key][block]
#pragma unroll
                for (int x = 0; x < GQ; ++x) s[x][hf] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < KB; ++k) {
                    const h8_t kf = codes8_to_half(kq[hf][k]);
#pragma unroll
                    for (int x = 0; x < GQ; ++x) {
                        f4_t acc = {0.f, 0.f, 0.f, 0.f};
                        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[x][1][k], acc, 0, 0, 0);
                        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[x][0][k], acc, 0, 0, 0);
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[x][hf][i] = __builtin_fmaf(float(steps[i >> 1][4 * (i & 1) + k]), acc[i], s[x][hf][i]);
                    }
                }
#pragma unroll
                for (int x = 0; x < GQ; ++x)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[x][hf][i] = 4 * g4 + i < nv[hf] ? s[x][hf][i] * qscale[x] : -INFINITY;
            }
            // the column's value steps, 2^-ve times, 0 past the keys
            float d[8], dmax = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint4 two = vd[i >> 2][(i & 3) >> 1];
                const uint64_t four = (i & 1) ? uint64_t(two.w) << 32 | two.z : uint64_t(two.y) << 32 | two.x;
                d[i] = 4 * g4 + (i & 3) < nv[i >> 2] ? half_bits_to_f32(uint16_t(four >> (16 * (c16 >> 2)))) : 0.f;
                dmax = fmaxf(dmax, d[i]);
            }
            const int top_e = __builtin_amdgcn_frexp_expf(dmax);
            if (__any(dmax > 0.f && top_e > ve)) {
                int e = dmax > 0.f ? top_e : -200;
                e = max(e, __shfl_xor(e, 16));
                e = max(e, __shfl_xor(e, 32));
                e = max(e, ve);
#pragma unroll
                for (int x = 0; x < GQ; ++x)
#pragma unroll
                    for (int n = 0; n < 8; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[x][n][i] = ldexpf(o[x][n][i], ve - e);
                ve = e;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] = ldexpf(d[i], -ve);
            h8_t ph[GQ], pl[GQ];
#pragma unroll
            for (int x = 0; x < GQ; ++x) {
                float top = s[x][0][0];
#pragma unroll
                for (int i = 1; i < 8; ++i) top = fmaxf(top, s[x][i >> 2][i & 3]);
                if (__any(top > m[x] + kPSlack)) {
                    const float m2 = fmaxf(m[x], max_over_rows(top)), f = m2 == -INFINITY ? 1.f : exp2_hw(m[x] - m2);
                    m[x] = m2;
                    l[x] *= f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) o[x][e] *= f;
                }
                const float base = m[x] - kPShift;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float p = exp2_hw(s[x][i >> 2][i & 3] - base);
                    l[x] += p;
                    _Float16 hi, lo;
                    split_f16(p * d[i], hi, lo);
                    ph[x][i] = hi;
                    pl[x][i] = lo;
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                h8_t v;
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const uint32_t lo = e < 4 ? vq[i].x : vq[i].y, hi = e < 4 ? vq[i + 1].x : vq[i + 1].y;
                    const h2_t t = codes_to_half(__builtin_amdgcn_perm(hi, lo, 0x0c040c00u + 0x00010001u * (e & 3)));
                    v[i] = t[0];
                    v[i + 1] = t[1];
                }
#pragma unroll
                for (int x = 0; x < GQ; ++x) {
                    o[x][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pl[x], o[x][e], 0, 0, 0);
                    o[x][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, ph[x], o[x][e], 0, 0, 0);
                }
            }
        }
    }

    // merge: a lane holds channels 128 v + 32 g4 + 8 i + e of its column's head
#pragma unroll
    for (int x = 0; x < GQ; ++x) {
        const float sum = sum_over_rows(l[x]);
        const int h = Q8 ? 4 * x + (c16 & 3) : c16 & 7;
#pragma unroll
        for (int n = 0; n < 8 * VH; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (Q8)
                    o[x][n][i] = ldexpf(o[x][n][i], ve);
                else
                    o[x][n][i] += column_other(o[x][n][i]);
            }
        if (h < group && (Q8 ? (c16 >> 2) == g4 : c16 < 8)) {
            if (Q8 || g4 == 0) mg.m[w][h] = m[x], mg.l[w][h] = sum;
#pragma unroll
            for (int v = 0; v < VH; ++v)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float4* to = reinterpret_cast<float4*>(&mg.o[w][h][128 * v + 32 * g4 + 8 * i]);
                    to[0] = make_float4(o[x][8 * v][i], o[x][8 * v + 1][i], o[x][8 * v + 2][i], o[x][8 * v + 3][i]);
                    to[1] = make_float4(o[x][8 * v + 4][i], o[x][8 * v + 5][i], o[x][8 * v + 6][i], o[x][8 * v + 7][i]);
                }
        }
    }
    __syncthreads();
    for (int e = tid; e < group * DH; e += 256) {
        const int h = e / DH, ch = e % DH;
        const float mx = fmaxf(fmaxf(mg.m[0][h], mg.m[1][h]), fmaxf(mg.m[2][h], mg.m[3][h]));
        float ov = 0.f, lv = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (mg.m[k][h] == -INFINITY && mg.l[k][h] == 0.f) continue;  // a wave without keys
            const float f = exp2_hw(mg.m[k][h] - mx);
            ov += f * mg.o[k][h][ch];
            lv += f * mg.l[k][h];
        }
        if (nsplit == 1) {
            sparse_store<DH>(a, r, g * group + h, ch, ov, lv);
        } else {
            float* rec = a.work + ((int64_t(r) * a.Hq + g * group + h) * nsplit + split) * (DH + 4);
            rec[4 + ch] = ov;
            if (ch == 0) rec[0] = mx, rec[1] = lv;
        }
    }
}

// a workgroup per (row, query head), a lane per channel: the ranges' results
template <int DH>
__global__ __launch_bounds__(DH) void attn_sparse_combine_kernel(SparseAttnArgs a, int nsplit) {
    const int r = blockIdx.x / a.Hq, h = blockIdx.x % a.Hq, ch = threadIdx.x;
    int seq;
    if (row_position(a.c, r, &seq) < 0) return;
    const float* rec = a.work + (int64_t(r) * a.Hq + h) * nsplit * (DH + 4);
    float mx = -INFINITY;
    for (int s = 0; s < nsplit; ++s) mx = fmaxf(mx, rec[s * (DH + 4)]);
    float o = 0.f, l = 0.f;
    for (int s = 0; s < nsplit; ++s) {
        const float m = rec[s * (DH + 4)], ls = rec[s * (DH + 4) + 1];
        if (m == -INFINITY && ls == 0.f) continue;
        const float f = exp2_hw(m - mx);
        l += f * ls;
        o += f * rec[s * (DH + 4) + 4 + ch];
    }
    sparse_store<DH>(a, r, h, ch, o, l);
}

// Ranges of a row's list: about four workgroups per CU over all rows and heads,
// whole pages, at least 32 key slots for each wave, at most 2048 list entries
// (16 KB of shared memory).
void sparse_plan(int64_t rows, int64_t Hkv, int64_t ps, int64_t top, int* per, int* nsplit) {
    const int64_t want = std::max<int64_t>(1, 1024 / (rows * Hkv));
    const int64_t most = std::max<int64_t>(1, top * ps / 128);
    const int64_t n = std::max(std::min(std::min(want, most), top), (top + 2047) / 2048);
    *per = int((top + n - 1) / n);
    *nsplit = int((top + *per - 1) / *per);
}

}  // namespace

void launch_attn_select(const SelectArgs& a, hipStream_t s) {
    const unsigned heads = unsigned(a.c.rows * a.c.Hkv);
    if (a.c.max_pages > a.top) {
        const dim3 grid(heads, unsigned((a.c.max_pages + 255) / 256));
        if (a.c.Dh == 256)
            hipLaunchKernelGGL(page_scores_kernel<256>, grid, dim3(256), 0, s, a);
        else
            hipLaunchKernelGGL(page_scores_kernel<128>, grid, dim3(256), 0, s, a);
    }
    hipLaunchKernelGGL(page_select_kernel, dim3(heads), dim3(64), 0, s, a);
}

int64_t attn_sparse_work_bytes(int64_t rows, int64_t Hq, int64_t Hkv, int64_t Dh, int64_t page_size, int64_t top) {
    int per, nsplit;
    sparse_plan(rows, Hkv, page_size, top, &per, &nsplit);
    return nsplit == 1 ? 0 : rows * Hq * nsplit * (Dh + 4) * 4;
}

void launch_attn_sparse(const SparseAttnArgs& a, hipStream_t s) {
    int per, nsplit;
    sparse_plan(a.c.rows, a.c.Hkv, a.c.page_size, a.top, &per, &nsplit);
    const dim3 grid(unsigned(int64_t(a.c.rows) * a.c.Hkv * nsplit));
    const size_t smem = size_t(per) * sizeof(ListEntry);
    if (a.c.Dh == 256)
        hipLaunchKernelGGL((attn_sparse_kernel<256, false, 1>), grid, dim3(256), smem, s, a, per, nsplit);
    else if (!a.c.q8)
        hipLaunchKernelGGL((attn_sparse_kernel<128, false, 1>), grid, dim3(256), smem, s, a, per, nsplit);
    else if (a.Hq / a.c.Hkv <= 4)
        hipLaunchKernelGGL((attn_sparse_kernel<128, true, 1>), grid, dim3(256), smem, s, a, per, nsplit);
    else
        hipLaunchKernelGGL((attn_sparse_kernel<128, true, 2>), grid, dim3(256), smem, s, a, per, nsplit);
    if (nsplit == 1) return;
    const dim3 heads(unsigned(a.c.rows * a.Hq));
    if (a.c.Dh == 256)
        hipLaunchKernelGGL(attn_sparse_combine_kernel<256>, heads, dim3(256), 0, s, a, nsplit);
    else
        hipLaunchKernelGGL(attn_sparse_combine_kernel<128>, heads, dim3(128), 0, s, a, nsplit);
}

}  // namespace hero
