// kvcache.hip -- rows of many sequences into the paged K/V cache and back:
// append (query / key norms and rotation, fp16 or Q8_0 quantization, page
// summaries) and read.
//
// Append equals what hero_attn_decode_paged stores for the same token, bit for
// bit: q and k are normalised with the reference's sequential sum of squares
// (nm/src/components.hpp:176-181) and rotated by the same table products
// (nm/src/attention.hpp:76-91), K and V are rounded to fp16 or pass the
// reference's activation quantizer (nm/src/quant_i8.hpp:70-80).
//
// A workgroup of the K/V part owns one K/V head of one run of rows: consecutive
// rows of one sequence in one page. It alone therefore sees every key of the
// page that this call writes, and reads the page's earlier keys back from the
// pool, so the summary needs no second launch, no atomics and nothing kept
// from earlier calls. The chain of a row's squares is as long as the row (one
// dependent add per channel); lanes of one wave run the chains of up to 64
// rows side by side.
#include "hero/device.hpp"
#include "hero/kernels.hpp"
#include "hero/paged.hpp"

namespace hero {

namespace {

constexpr int kApRows = 64;  // rows per pass of the K/V part
constexpr int kApQ = 32;     // (row, query head) items per workgroup of the q part

// x rounded to fp32 by whatever formed it, then to fp16 (the compiler may not
// round a product to fp16 at once)
__device__ __forceinline__ uint16_t f16_bits(float x) {
    asm("" : "+v"(x));
    const _Float16 h = _Float16(x);
    uint16_t b;
    __builtin_memcpy(&b, &h, 2);
    return b;
}

// quantize_row_q8_0 of a 32-value block held one value per lane by 32 lanes
__device__ __forceinline__ int q8_code(float x, uint16_t* dh) {
    float amax = fabsf(x);
    for (int off = 16; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor(amax, off, 32));
    const float d = amax / 127.f;
    const float id = d != 0.f ? 1.f / d : 0.f;
    *dh = fp32_to_fp16_ref(d);
    return int(int8_t(int(roundf(x * id))));
}

// 1 / rms of a row of DH values in shared memory, squares added in order
template <int DH>
__device__ __forceinline__ float row_scale(const float* row, float eps) {
    float ss = 0.f;
    const float4* r4 = reinterpret_cast<const float4*>(row);
#pragma unroll 8
    for (int i = 0; i < DH / 4; ++i) {
        const float4 v = r4[i];
        ss += v.x * v.x;
        ss += v.y * v.y;
        ss += v.z * v.z;
        ss += v.w * v.w;
    }
    return 1.f / sqrtf(ss / float(DH) + eps);
}

// norm and rotation of a row held by 32 lanes, lane l channels l + 32 m
template <int DH>
__device__ __forceinline__ void norm_rotate(const float* row, const float* gamma, float scale, const float* cs, int l, float (&y)[DH / 32]) {
    float n[DH / 32];
#pragma unroll
    for (int m = 0; m < DH / 32; ++m) n[m] = gamma[l + 32 * m] * row[l + 32 * m] * scale;
#pragma unroll
    for (int m = 0; m < DH / 64; ++m) {
        const float2 t = reinterpret_cast<const float2*>(cs)[l + 32 * m];
        const float xx = n[m], yy = n[m + DH / 64];
        y[m] = xx * t.x - yy * t.y;
        y[m + DH / 64] = yy * t.x + xx * t.y;
    }
}

template <int DH, bool Q8>
__global__ __launch_bounds__(256) void kv_append_kernel(KvAppendArgs a, int kv_blocks) {
    constexpr int M = DH / 32, kStride = DH + 4;
    constexpr int kBuf = kApRows * kStride > 16 * DH ? kApRows * kStride : 16 * DH;
    const PagedRows& c = a.c;
    const int tid = threadIdx.x, hw = tid >> 5, l = tid & 31;
    __shared__ __align__(16) float buf[kBuf];
    __shared__ float scale[kApRows];
    if (int(blockIdx.x) >= kv_blocks) {  // queries
        const int64_t items = int64_t(c.rows) * a.Hq, i0 = int64_t(blockIdx.x - kv_blocks) * kApQ;
        const int n = int(min(int64_t(kApQ), items - i0));
        for (int e = tid; e < n * DH; e += 256) {
            const int64_t it = i0 + e / DH;
            buf[(e / DH) * kStride + e % DH] = a.proj[it / a.Hq * a.proj_stride + it % a.Hq * 2 * DH + e % DH];
        }
        __syncthreads();
        if (tid < n) scale[tid] = row_scale<DH>(buf + tid * kStride, a.eps);
        __syncthreads();
        for (int i = hw; i < n; i += 8) {
            const int64_t it = i0 + i;
            int seq;
            const int pos = row_position(c, int(it / a.Hq), &seq);
            if (pos < 0 || pos >= a.rope_positions) continue;
            float y[M];
            norm_rotate<DH>(buf + i * kStride, a.q_gamma, scale[i], a.rope_cs + int64_t(pos) * DH, l, y);
#pragma unroll
            for (int m = 0; m < M; ++m) a.q_rot[it * DH + l + 32 * m] = y[m];
        }
        return;
    }
    const int r0 = blockIdx.x / c.Hkv, g = blockIdx.x % c.Hkv, ps = c.page_size;
    int seq, prev_seq;
    const int pos = row_position(c, r0, &seq);
    if (pos < 0 || pos >= a.rope_positions) return;
    const int slot0 = pos % ps;
    if (r0 > 0 && slot0 > 0) {  // inside the run of an earlier row
        const int prev = row_position(c, r0 - 1, &prev_seq);
        if (prev == pos - 1 && prev_seq == seq) return;
    }
    const int64_t page = pool_page(c, seq, pos / ps);
    if (page < 0) return;
    // the run: rows r0 + i at pos + i in this page
    __shared__ int run;
    if (tid == 0) run = min(ps - slot0, c.rows - r0);
    __syncthreads();
    if (tid > 0 && tid < ps - slot0 && r0 + tid < c.rows) {
        int s2;
        const int p2 = row_position(c, r0 + tid, &s2);
        if (p2 != pos + tid || s2 != seq || p2 >= a.rope_positions) atomicMin(&run, tid);
    }
    __syncthreads();
    const int n = run;

    float hi[M], lo[M];
#pragma unroll
    for (int m = 0; m < M; ++m) hi[m] = -INFINITY, lo[m] = INFINITY;
    auto bound = [&](int m, float x) {
        hi[m] = fmaxf(hi[m], x);
        lo[m] = fminf(lo[m], x);
    };
    uint16_t* const fpage = const_cast<uint16_t*>(reinterpret_cast<const uint16_t*>(f16_page<DH>(c, page)));
    uint8_t* const qpage = q8_page<DH>(c, page);
    uint16_t* const qscales = reinterpret_cast<uint16_t*>(qpage + q8_scales_at<DH>(c));
    for (int t = hw; t < slot0; t += 8) {  // keys of earlier calls
        const int64_t row = page_row_index(c, 0, g, t);
#pragma unroll
        for (int m = 0; m < M; ++m) {
            if constexpr (Q8)
                bound(m, half_bits_to_f32(qscales[row * M + m]) * float(int8_t(qpage[row * DH + l + 32 * m])));
            else
                bound(m, half_bits_to_f32(fpage[row * DH + l + 32 * m]));
        }
    }
    for (int c0 = 0; c0 < n; c0 += kApRows) {
        const int nr = min(kApRows, n - c0);
        __syncthreads();
        for (int e = tid; e < nr * DH; e += 256)
            buf[(e / DH) * kStride + e % DH] = a.proj[int64_t(r0 + c0 + e / DH) * a.proj_stride + a.k_off + int64_t(g) * DH + e % DH];
        __syncthreads();
        if (tid < nr) scale[tid] = row_scale<DH>(buf + tid * kStride, a.eps);
        __syncthreads();
        for (int i = hw; i < nr; i += 8) {
            const int t = slot0 + c0 + i;
            const float* v = a.proj + int64_t(r0 + c0 + i) * a.proj_stride + a.v_off + int64_t(g) * DH;
            const int64_t krow = page_row_index(c, 0, g, t), vrow = page_row_index(c, 1, g, t);
            float y[M];
            norm_rotate<DH>(buf + i * kStride, a.k_gamma, scale[i], a.rope_cs + int64_t(pos + c0 + i) * DH, l, y);
#pragma unroll
            for (int m = 0; m < M; ++m) {
                const float vm = v[l + 32 * m];
                if constexpr (Q8) {
                    uint16_t dk, dv;
                    const int qk = q8_code(y[m], &dk), qv = q8_code(vm, &dv);
                    qpage[krow * DH + l + 32 * m] = uint8_t(qk);
                    qpage[vrow * DH + l + 32 * m] = uint8_t(qv);
                    if (l == 0) qscales[krow * M + m] = dk, qscales[vrow * M + m] = dv;
                    bound(m, half_bits_to_f32(dk) * float(qk));
                } else {
                    const uint16_t kb = f16_bits(y[m]);
                    fpage[krow * DH + l + 32 * m] = kb;
                    fpage[vrow * DH + l + 32 * m] = f16_bits(vm);
                    bound(m, half_bits_to_f32(kb));
                }
            }
        }
    }
    // the eight half-waves' bounds, then the codes: lane j < DH channel j
    __syncthreads();
#pragma unroll
    for (int m = 0; m < M; ++m) buf[hw * 2 * DH + l + 32 * m] = hi[m], buf[hw * 2 * DH + DH + l + 32 * m] = lo[m];
    __syncthreads();
    float mx = -INFINITY, mn = INFINITY;
    if (tid < DH)
        for (int w = 0; w < 8; ++w) mx = fmaxf(mx, buf[w * 2 * DH + tid]), mn = fminf(mn, buf[w * 2 * DH + DH + tid]);
    float amax = tid < DH ? fmaxf(fabsf(mx), fabsf(mn)) : 0.f;
    for (int off = 32; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor(amax, off));
    if ((tid & 63) == 0) scale[tid >> 6] = amax;
    __syncthreads();
    amax = fmaxf(fmaxf(scale[0], scale[1]), fmaxf(scale[2], scale[3]));
    const float d = amax / 127.f, id = d != 0.f ? 1.f / d : 0.f;
    uint8_t* sum = c.summaries + page * kv_summary_page_bytes(c.Hkv, DH);
    if (tid < DH) {
        sum[int64_t(g) * 2 * DH + tid] = uint8_t(int8_t(int(roundf(mx * id))));
        sum[int64_t(g) * 2 * DH + DH + tid] = uint8_t(int8_t(int(roundf(-mn * id))));
    }
    if (tid == 0) reinterpret_cast<float*>(sum + int64_t(c.Hkv) * 2 * DH)[g] = round11(d);
}

// eight channels a lane: a row's K (or V, or bounds) of all heads is one
// contiguous run of the output
template <int DH, bool Q8, typename T>
__global__ __launch_bounds__(256) void kv_read_kernel(KvReadArgs a) {
    const PagedRows& c = a.c;
    const int r = blockIdx.x, kw8 = c.Hkv * DH / 8;
    int seq;
    const int pos = row_position(c, r, &seq);
    if (pos < 0) return;
    const int64_t page = pool_page(c, seq, pos / c.page_size);
    if (page < 0) return;
    const int t = pos % c.page_size;
    for (int e = blockIdx.y * 256 + threadIdx.x; e < 4 * kw8; e += 256 * gridDim.y) {
        const int what = e / kw8, ch = e % kw8 * 8, g = ch / DH, j = ch % DH;
        T* out = static_cast<T*>(a.out[what]);
        if (!out) continue;
        float x[8];
        if (what >= 2) {
            const uint8_t* sum = c.summaries + page * kv_summary_page_bytes(c.Hkv, DH);
            const int2 q = *reinterpret_cast<const int2*>(sum + int64_t(g) * 2 * DH + (what - 2) * DH + j);
            const float d = reinterpret_cast<const float*>(sum + int64_t(c.Hkv) * 2 * DH)[g] * (what == 2 ? 1.f : -1.f);
#pragma unroll
            for (int u = 0; u < 8; ++u) x[u] = d * float(int8_t((u < 4 ? q.x : q.y) >> (8 * (u & 3))));
        } else {
            const int64_t row = page_row_index(c, what, g, t);
            if constexpr (Q8) {
                const uint8_t* qp = q8_page<DH>(c, page);
                const int2 q = *reinterpret_cast<const int2*>(qp + row * DH + j);
                const float d = half_bits_to_f32(reinterpret_cast<const uint16_t*>(qp + q8_scales_at<DH>(c))[row * (DH / 32) + j / 32]);
#pragma unroll
                for (int u = 0; u < 8; ++u) x[u] = d * float(int8_t((u < 4 ? q.x : q.y) >> (8 * (u & 3))));
            } else {
                typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
                const h8_t h = *reinterpret_cast<const h8_t*>(f16_page<DH>(c, page) + row * DH + j);
#pragma unroll
                for (int u = 0; u < 8; ++u) x[u] = float(h[u]);
            }
        }
        T y[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) y[u] = T(x[u]);
        __builtin_memcpy(__builtin_assume_aligned(out + int64_t(r) * c.Hkv * DH + ch, 16), y, sizeof(y));
    }
}

}  // namespace

void launch_kv_append(const KvAppendArgs& a, hipStream_t s) {
    const int64_t kv = int64_t(a.c.rows) * a.c.Hkv, q = (int64_t(a.c.rows) * a.Hq + kApQ - 1) / kApQ;
    const dim3 grid(unsigned(kv + q));
    if (a.c.Dh == 256)
        hipLaunchKernelGGL((kv_append_kernel<256, false>), grid, dim3(256), 0, s, a, int(kv));
    else if (a.c.q8)
        hipLaunchKernelGGL((kv_append_kernel<128, true>), grid, dim3(256), 0, s, a, int(kv));
    else
        hipLaunchKernelGGL((kv_append_kernel<128, false>), grid, dim3(256), 0, s, a, int(kv));
}

namespace {
template <int DH, bool Q8>
void kv_read_typed(const KvReadArgs& a, hipStream_t s) {
    const dim3 grid(unsigned(a.c.rows));
    if (a.f16)
        hipLaunchKernelGGL((kv_read_kernel<DH, Q8, _Float16>), grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((kv_read_kernel<DH, Q8, float>), grid, dim3(256), 0, s, a);
}
}  // namespace

void launch_kv_read(const KvReadArgs& a, hipStream_t s) {
    if (a.c.Dh == 256)
        kv_read_typed<256, false>(a, s);
    else if (a.c.q8)
        kv_read_typed<128, true>(a, s);
    else
        kv_read_typed<128, false>(a, s);
}

}  // namespace hero
