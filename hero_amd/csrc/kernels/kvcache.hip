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
// dependent add per channel); lanes of one wave run the chains of up to 32
// rows side by side. Everything else is 32 lanes per row, four neighbouring
// channels each, so that a row is read and written in whole words.
//
// Bound: for single tokens the dependent reads (position, page id, row), the chain
// (0.4 us for 128 channels, twice that for 256) and the exchange of the bounds: 4.6
// us for one row of 32 + 8 heads of 128, 5.6 us for 16 + 4 heads of 256, 6.4 us for
// sixteen rows into Q8_0 pages that hold 32 keys on average. For chunks the same
// latencies and HBM: 1000 rows (41 MB) 15.5 us into Q8_0 pages, 14.6 into fp16 ones
// (256-wide heads 15.5), 8.6 us at a large copy's 4.76 TB/s. Reading back 8192 Q8_0 rows as fp32 (85 MB): 18.3 us,
// 4.6 TB/s, as a copy.
#include "hero/device.hpp"
#include "hero/kernels.hpp"
#include "hero/paged.hpp"

namespace hero {

namespace {

// chunks: workgroups per K/V head, set for eight of them (two workgroups per CU).
// Fewer heads make fewer workgroups: 1000 rows of one K/V head take 8.0 us (pages
// of 16: 8.7), of two 8.9, of four 10.3, of eight 14.6
constexpr int kApSpread = 61;

// x rounded to fp32 by whatever formed it, then to fp16 (the compiler may not
// round a product to fp16 at once)
__device__ __forceinline__ uint16_t f16_bits(float x) {
    asm("" : "+v"(x));
    const _Float16 h = _Float16(x);
    uint16_t b;
    __builtin_memcpy(&b, &h, 2);
    return b;
}

__device__ __forceinline__ float4 load4(const float* p) {  // at any float's address
    float4 v;
    __builtin_memcpy(&v, p, 16);
    return v;
}

// quantize_row_q8_0 of a 32-value block held four values per lane by 8 lanes:
// the four codes packed; *dh the block's fp16 step
__device__ __forceinline__ uint32_t q8_codes(const float (&x)[4], uint16_t* dh) {
    float amax = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
    auto with = [](float v, int bits) { return fmaxf(v, __int_as_float(bits)); };
    amax = with(amax, __builtin_amdgcn_update_dpp(0, __float_as_int(amax), 0xB1, 0xF, 0xF, false));   // quad_perm [1,0,3,2]
    amax = with(amax, __builtin_amdgcn_update_dpp(0, __float_as_int(amax), 0x4E, 0xF, 0xF, false));   // quad_perm [2,3,0,1]
    amax = with(amax, __builtin_amdgcn_update_dpp(0, __float_as_int(amax), 0x141, 0xF, 0xF, false));  // row_half_mirror
    const float d = amax / 127.f;
    const float id = d != 0.f ? 1.f / d : 0.f;
    *dh = fp32_to_fp16_ref(d);
    uint32_t w = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) w |= uint32_t(round_code(x[k] * id) & 0xFF) << (8 * k);
    return w;
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

// A head's weights and rotation for lane l of 32: channels 4 l + 128 m + k and
// their partners, half a head away (the same lane's for 256 channels)
template <int DH>
struct HeadLane {
    float g[2][4];  // of the lane's channels, and of their partners (DH 128) or channels + 128 (DH 256)
    __device__ __forceinline__ HeadLane(const float* gamma, int l) {
        const int a = 4 * l, b = DH == 128 ? (4 * l + 64) & 127 : 4 * l + 128;
#pragma unroll
        for (int k = 0; k < 4; ++k) g[0][k] = gamma[a + k], g[1][k] = gamma[b + k];
    }
    // norm and rotation: the lane's own values x, its partners' in the row in
    // shared memory, cs the (cos, sin) of its four planes
    __device__ __forceinline__ void rotate(const float4 (&x)[DH / 128], const float* row, float scale, const float4 (&cs)[2], int l, float (&y)[DH / 128][4]) const {
        const float4 xa = x[0], xb = DH == 128 ? *reinterpret_cast<const float4*>(row + ((4 * l + 64) & 127)) : x[DH / 128 - 1];
        const float na[4] = {g[0][0] * xa.x * scale, g[0][1] * xa.y * scale, g[0][2] * xa.z * scale, g[0][3] * xa.w * scale};
        const float nb[4] = {g[1][0] * xb.x * scale, g[1][1] * xb.y * scale, g[1][2] * xb.z * scale, g[1][3] * xb.w * scale};
        const float co[4] = {cs[0].x, cs[0].z, cs[1].x, cs[1].z}, si[4] = {cs[0].y, cs[0].w, cs[1].y, cs[1].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if constexpr (DH == 128) {  // (lo, hi) = (own, partner) for the lower half's lanes, else the other way
                y[0][k] = l < 16 ? na[k] * co[k] - nb[k] * si[k] : na[k] * co[k] + nb[k] * si[k];
            } else {
                y[0][k] = na[k] * co[k] - nb[k] * si[k];
                y[DH / 128 - 1][k] = nb[k] * co[k] + na[k] * si[k];
            }
        }
    }
};
template <int DH>
__device__ __forceinline__ void load_cs(const float* rope_cs, int pos, int l, float4 (&cs)[2]) {
    const float* p = rope_cs + int64_t(pos) * DH + 2 * (4 * l % (DH / 2));
    cs[0] = load4(p);
    cs[1] = load4(p + 4);
}

// One K/V head of the run that starts in row r0, by the whole workgroup.
template <int DH, bool Q8, int NT, int T>
__device__ __forceinline__ void append_run(const KvAppendArgs& a, int g, int r0, const HeadLane<DH>& lane, float* buf, float* scale, int* run) {
    constexpr int V = DH / 128, kStride = DH + 4, HW = NT / 32, kRows = HW * T;
    const PagedRows& c = a.c;
    const int tid = threadIdx.x, hw = tid >> 5, l = tid & 31, ps = c.page_size;
    int seq;
    const int pos = row_position(c, r0, &seq), slot0 = pos % ps, room = min(ps - slot0, c.rows - r0);
    const int64_t page = pool_page(c, seq, pos / ps);
    if (page < 0) return;
    float hi[V][4], lo[V][4];
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
        for (int k = 0; k < 4; ++k) hi[v][k] = -INFINITY, lo[v][k] = INFINITY;
    auto bound = [&](int v, int k, float x) {
        hi[v][k] = fmaxf(hi[v][k], x);
        lo[v][k] = fminf(lo[v][k], x);
    };
    uint16_t* const fpage = const_cast<uint16_t*>(reinterpret_cast<const uint16_t*>(f16_page<DH>(c, page)));
    uint8_t* const qpage = q8_page<DH>(c, page);
    uint16_t* const qscales = reinterpret_cast<uint16_t*>(qpage + q8_scales_at<DH>(c));
    // the run: rows r0 + i at pos + i in this page
    int n = 1;
    if (NT > 256 || c.row_seq) {
        __syncthreads();
        if (tid == 0) *run = room;
        __syncthreads();
        if (tid > 0 && tid < room) {
            int s2;
            const int p2 = row_position(c, r0 + tid, &s2);
            if (p2 != pos + tid || s2 != seq || p2 >= a.rope_positions) atomicMin(run, tid);
        }
        __syncthreads();
        n = *run;
    }
    for (int c0 = 0; c0 < n; c0 += kRows) {
        const int nr = min(kRows, n - c0);
        const float* rows = a.proj + int64_t(r0 + c0) * a.proj_stride + int64_t(g) * DH + 4 * l;
        float4 kx[T][V], vx[T][V], cs[T][2];
#pragma unroll
        for (int j = 0; j < T; ++j) {
            const int i = min(hw + HW * j, nr - 1);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                kx[j][v] = load4(rows + int64_t(i) * a.proj_stride + a.k_off + 128 * v);
                vx[j][v] = load4(rows + int64_t(i) * a.proj_stride + a.v_off + 128 * v);
            }
            load_cs<DH>(a.rope_cs, pos + c0 + i, l, cs[j]);
        }
        if (c0 == 0) {  // keys of earlier calls
            for (int t = hw; t < slot0; t += HW) {
                const int64_t row = page_row_index(c, 0, g, t);
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    if constexpr (Q8) {
                        const uint32_t q = *reinterpret_cast<const uint32_t*>(qpage + row * DH + 4 * l);
                        const float d = half_bits_to_f32(qscales[row * 4 + l / 8]);
#pragma unroll
                        for (int k = 0; k < 4; ++k) bound(v, k, d * float(int8_t(q >> (8 * k))));
                    } else {
                        const ushort4 h = *reinterpret_cast<const ushort4*>(fpage + row * DH + 128 * v + 4 * l);
                        bound(v, 0, half_bits_to_f32(h.x)), bound(v, 1, half_bits_to_f32(h.y)), bound(v, 2, half_bits_to_f32(h.z)), bound(v, 3, half_bits_to_f32(h.w));
                    }
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < T; ++j)
#pragma unroll
            for (int v = 0; v < V; ++v) *reinterpret_cast<float4*>(buf + (hw + HW * j) * kStride + 128 * v + 4 * l) = kx[j][v];
        __syncthreads();
        if (tid < nr) scale[tid] = row_scale<DH>(buf + tid * kStride, a.eps);
        __syncthreads();
#pragma unroll
        for (int j = 0; j < T; ++j) {
            const int i = hw + HW * j, t = slot0 + c0 + i;
            if (i >= nr) continue;
            const int64_t krow = page_row_index(c, 0, g, t), vrow = page_row_index(c, 1, g, t);
            float y[V][4];
            lane.rotate(kx[j], buf + i * kStride, scale[i], cs[j], l, y);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float x[4] = {vx[j][v].x, vx[j][v].y, vx[j][v].z, vx[j][v].w};
                if constexpr (Q8) {
                    uint16_t dk, dv;
                    const uint32_t qk = q8_codes(y[v], &dk), qv = q8_codes(x, &dv);
                    *reinterpret_cast<uint32_t*>(qpage + krow * DH + 4 * l) = qk;
                    *reinterpret_cast<uint32_t*>(qpage + vrow * DH + 4 * l) = qv;
                    if (l % 8 == 0) qscales[krow * 4 + l / 8] = dk, qscales[vrow * 4 + l / 8] = dv;
#pragma unroll
                    for (int k = 0; k < 4; ++k) bound(v, k, half_bits_to_f32(dk) * float(int8_t(qk >> (8 * k))));
                } else {
                    const ushort4 kb = make_ushort4(f16_bits(y[v][0]), f16_bits(y[v][1]), f16_bits(y[v][2]), f16_bits(y[v][3]));
                    *reinterpret_cast<ushort4*>(fpage + krow * DH + 128 * v + 4 * l) = kb;
                    *reinterpret_cast<ushort4*>(fpage + vrow * DH + 128 * v + 4 * l) = make_ushort4(f16_bits(x[0]), f16_bits(x[1]), f16_bits(x[2]), f16_bits(x[3]));
                    bound(v, 0, half_bits_to_f32(kb.x)), bound(v, 1, half_bits_to_f32(kb.y)), bound(v, 2, half_bits_to_f32(kb.z)), bound(v, 3, half_bits_to_f32(kb.w));
                }
            }
        }
    }
    // the half-waves' bounds, then the codes: lane j < DH channel j
    __syncthreads();
#pragma unroll
    for (int v = 0; v < V; ++v) {
        *reinterpret_cast<float4*>(buf + hw * 2 * DH + 128 * v + 4 * l) = make_float4(hi[v][0], hi[v][1], hi[v][2], hi[v][3]);
        *reinterpret_cast<float4*>(buf + hw * 2 * DH + DH + 128 * v + 4 * l) = make_float4(lo[v][0], lo[v][1], lo[v][2], lo[v][3]);
    }
    __syncthreads();
    float mx = -INFINITY, mn = INFINITY;
    if (tid < DH) {
#pragma unroll 8
        for (int w = 0; w < HW; ++w) mx = fmaxf(mx, buf[w * 2 * DH + tid]), mn = fminf(mn, buf[w * 2 * DH + DH + tid]);
        float amax = fmaxf(fabsf(mx), fabsf(mn));
        for (int off = 32; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor(amax, off));
        if ((tid & 63) == 0) scale[tid >> 6] = amax;
    }
    __syncthreads();
    if (tid < DH) {
        float amax = scale[0];
#pragma unroll
        for (int w = 1; w < DH / 64; ++w) amax = fmaxf(amax, scale[w]);
        const float d = amax / 127.f, id = d != 0.f ? 1.f / d : 0.f;
        uint8_t* sum = c.summaries + page * kv_summary_page_bytes(c.Hkv, DH);
        sum[int64_t(g) * 2 * DH + tid] = uint8_t(round_code(mx * id));
        sum[int64_t(g) * 2 * DH + DH + tid] = uint8_t(round_code(-mn * id));
        if (tid == 0) reinterpret_cast<float*>(sum + int64_t(c.Hkv) * 2 * DH)[g] = round11(d);
    }
}

// NT lanes, T rows (or (row, query head) items) for each of their half-waves a
// pass, everything a pass reads in flight before the chains run. Rows that come
// one per sequence: 256 lanes, T = 1. Chunks: 512 lanes, T = 2: half a page of
// 64 positions a pass (T = 4, a whole one, is 6% slower: fewer waves fit). A workgroup of the K/V part works off the runs that
// start in rows b, b + spread, ...: neighbouring rows of different sequences
// go to different workgroups, and so do the pages of one chunk, whose starts
// are a page size apart, as `spread` is odd; there are few of them, as most find no
// start (one per row and head cost 50 us of launching alone at 1000 rows).
template <int DH, bool Q8, int NT, int T>
__global__ __launch_bounds__(NT, NT / 128) void kv_append_kernel(KvAppendArgs a, int spread) {
    constexpr int V = DH / 128, kStride = DH + 4, HW = NT / 32, kRows = HW * T;
    constexpr int kBuf = kRows * kStride > HW * 2 * DH ? kRows * kStride : HW * 2 * DH;
    const PagedRows& c = a.c;
    const int tid = threadIdx.x, hw = tid >> 5, l = tid & 31;
    __shared__ __align__(16) float buf[kBuf];
    __shared__ float scale[kRows];
    __shared__ int run;
    const int kv_blocks = spread * c.Hkv;
    if (int(blockIdx.x) >= kv_blocks) {  // queries
        const int64_t items = int64_t(c.rows) * a.Hq, i0 = int64_t(blockIdx.x - kv_blocks) * kRows;
        const int n = int(min(int64_t(kRows), items - i0));
        const HeadLane<DH> lane(a.q_gamma, l);
        float4 x[T][V], cs[T][2];
        int pos[T];
#pragma unroll
        for (int j = 0; j < T; ++j) {
            const int64_t it = i0 + min(hw + HW * j, n - 1);
            int seq;
            pos[j] = row_position(c, int(it / a.Hq), &seq);
            if (pos[j] >= a.rope_positions || hw + HW * j >= n) pos[j] = -1;
            load_cs<DH>(a.rope_cs, max(pos[j], 0), l, cs[j]);
            const float* q = a.proj + it / a.Hq * a.proj_stride + it % a.Hq * 2 * DH + 4 * l;
#pragma unroll
            for (int v = 0; v < V; ++v) x[j][v] = load4(q + 128 * v);
        }
#pragma unroll
        for (int j = 0; j < T; ++j)
#pragma unroll
            for (int v = 0; v < V; ++v) *reinterpret_cast<float4*>(buf + (hw + HW * j) * kStride + 128 * v + 4 * l) = x[j][v];
        __syncthreads();
        if (tid < n) scale[tid] = row_scale<DH>(buf + tid * kStride, a.eps);
        __syncthreads();
#pragma unroll
        for (int j = 0; j < T; ++j) {
            if (pos[j] < 0) continue;
            float y[V][4];
            lane.rotate(x[j], buf + (hw + HW * j) * kStride, scale[hw + HW * j], cs[j], l, y);
#pragma unroll
            for (int v = 0; v < V; ++v)
                *reinterpret_cast<float4*>(a.q_rot + (i0 + hw + HW * j) * DH + 128 * v + 4 * l) = make_float4(y[v][0], y[v][1], y[v][2], y[v][3]);
        }
        return;
    }
    const int g = blockIdx.x % c.Hkv, b = blockIdx.x / c.Hkv, ps = c.page_size;
    const HeadLane<DH> lane(a.k_gamma, l);
    for (int64_t first = b; first < c.rows; first += 64 * int64_t(spread)) {
        // which of the next 64 rows start a run: a lane each
        bool starts = false;
        if (const int64_t r = first + int64_t(tid & 63) * spread; r < c.rows) {
            int s, before;
            const int p = row_position(c, int(r), &s);
            starts = p >= 0 && p < a.rope_positions && !(r > 0 && p % ps > 0 && row_position(c, int(r) - 1, &before) == p - 1 && before == s);
        }
        for (uint64_t left = __ballot(starts); left; left &= left - 1)
            append_run<DH, Q8, NT, T>(a, g, int(first + (__ffsll((unsigned long long)left) - 1) * int64_t(spread)), lane, buf, scale, &run);
    }
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
    for (int e = threadIdx.x; e < 4 * kw8; e += 256) {
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

namespace {
template <int DH, bool Q8, int NT, int T>
void kv_append_sized(const KvAppendArgs& a, int spread, hipStream_t s) {
    const int64_t per = NT / 32 * T, q = (int64_t(a.c.rows) * a.Hq + per - 1) / per;
    hipLaunchKernelGGL((kv_append_kernel<DH, Q8, NT, T>), dim3(unsigned(int64_t(spread) * a.c.Hkv + q)), dim3(NT), 0, s, a, spread);
}
template <int DH, bool Q8>
void kv_append_typed(const KvAppendArgs& a, hipStream_t s) {
    if (!a.c.row_seq || a.c.rows == 1)  // runs of one row
        kv_append_sized<DH, Q8, 256, 1>(a, a.c.rows, s);
    else
        kv_append_sized<DH, Q8, 512, 2>(a, std::min(a.c.rows, kApSpread), s);
}
}  // namespace

void launch_kv_append(const KvAppendArgs& a, hipStream_t s) {
    if (a.c.Dh == 256)
        kv_append_typed<256, false>(a, s);
    else if (a.c.q8)
        kv_append_typed<128, true>(a, s);
    else
        kv_append_typed<128, false>(a, s);
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
