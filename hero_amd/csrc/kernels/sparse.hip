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
// a wave per (row, query head), lane l channels l + 64 m
template <int DH, bool Q8>
__global__ __launch_bounds__(64) void attn_sparse_kernel(SparseAttnArgs a) {
    constexpr int M = DH / 64;
    const PagedRows& c = a.c;
    const int l = threadIdx.x, r = blockIdx.x / a.Hq, h = blockIdx.x % a.Hq, g = h / (a.Hq / c.Hkv);
    int seq;
    const int pos = row_position(c, r, &seq);
    if (pos < 0) return;
    float q[M], o[M];
    for (int m = 0; m < M; ++m) q[m] = a.q_rot[(int64_t(r) * a.Hq + h) * DH + l + 64 * m], o[m] = 0.f;
    float mx = -INFINITY, sum = 0.f;
    const int32_t* list = a.selected + (int64_t(r) * c.Hkv + g) * a.top;
    auto load = [&](int64_t page, int64_t row, int m) {
        const int j = l + 64 * m;
        if constexpr (Q8) {
            const uint8_t* qp = q8_page<DH>(c, page);
            return half_bits_to_f32(reinterpret_cast<const uint16_t*>(qp + q8_scales_at<DH>(c))[row * (DH / 32) + j / 32]) * float(int8_t(qp[row * DH + j]));
        } else {
            return float(f16_page<DH>(c, page)[row * DH + j]);
        }
    };
    for (int i = 0; i < a.top; ++i) {
        const int lp = list[i];
        if (lp < 0 || lp > pos / c.page_size) continue;
        const int64_t page = pool_page(c, seq, lp);
        if (page < 0) continue;
        const int n = min(c.page_size, pos + 1 - lp * c.page_size);
        for (int t = 0; t < n; ++t) {
            float s = 0.f;
            for (int m = 0; m < M; ++m) s += q[m] * load(page, page_row_index(c, 0, g, t), m);
            for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off);
            s *= a.score_scale;
            const float m2 = fmaxf(mx, s), f = exp_f32(mx - m2), p = exp_f32(s - m2);
            mx = m2;
            sum = sum * f + p;
            for (int m = 0; m < M; ++m) o[m] = o[m] * f + p * load(page, page_row_index(c, 1, g, t), m);
        }
    }
    const int64_t width = int64_t(a.Hq) * DH;
    for (int m = 0; m < M; ++m) {
        const int j = l + 64 * m;
        const float gate = a.proj[int64_t(r) * a.proj_stride + int64_t(h) * 2 * DH + DH + j];
        const float out = sum > 0.f ? (o[m] / sum) * sigmoid_f32(gate) : sum != sum ? sum : 0.f;
        const int64_t idx = int64_t(r) * width + int64_t(h) * DH + j;
        if (a.out_f32) a.out_f32[idx] = out;
        if (a.act_out) {
            float amax = fabsf(out);
            for (int off = 16; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor(amax, off));
            const float d = amax / 127.f, id = d != 0.f ? 1.f / d : 0.f;
            int8_t* qs = static_cast<int8_t*>(a.act_out);
            qs[idx] = int8_t(int(roundf(out * id)));
            if ((l & 31) == 0) reinterpret_cast<float*>(qs + int64_t(c.rows) * width)[idx >> 5] = half_bits_to_f32(fp32_to_fp16_ref(d));
        }
    }
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

int64_t attn_sparse_work_bytes(int64_t, int64_t, int64_t, int64_t, int64_t, int64_t) { return 0; }

void launch_attn_sparse(const SparseAttnArgs& a, hipStream_t s) {
    const dim3 grid(unsigned(a.c.rows * a.Hq));
    if (a.c.Dh == 256)
        hipLaunchKernelGGL((attn_sparse_kernel<256, false>), grid, dim3(64), 0, s, a);
    else if (a.c.q8)
        hipLaunchKernelGGL((attn_sparse_kernel<128, true>), grid, dim3(64), 0, s, a);
    else
        hipLaunchKernelGGL((attn_sparse_kernel<128, false>), grid, dim3(64), 0, s, a);
}

}  // namespace hero
