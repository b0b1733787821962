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
// Scores are int8 matrix products of 16 pages x 16 columns x 64 bytes: the
// columns are the query heads of a K/V head (GP, the group rounded up to a
// power of two) times RT rows, which share the pages' reads where they belong
// to one sequence. Lane 16 g + c brings 16 bytes of page c and the same bytes of
// column c's codes, and gets the sums of pages 4 g .. 4 g + 3 for column c. The
// codes are formed once per workgroup, a wave per head.
//
// Bound: one token over 500 pages (1 MB of summaries): latency, 8.4 us in one
// launch -- three dependent reads, some 600 instructions that run once, and five
// to seven rounds of the search. Sixteen tokens over 2047 pages each (67 MB): 18
// to 20 us for the scores, 3.5 TB/s of records that lie 256 bytes at a time in no
// order (sixty-four tokens: 3.7 TB/s), and 8 us for the choice; 14.4 us at a
// copy's rate. 500 rows of a chunk over 251 to 258 pages: 18 us, vector
// instructions (the exact scores take 64-bit products and maxima, about 45
// instructions for four pages and rows). Heads of 256 channels, 16 over 4: 10.7, 28
// and 16.5 us for the three.
typedef int v4i_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float max_over_rows(float x) {  // over the four g of a column
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}

// order-preserving key of a score; 0 is kept for pages that cannot be taken
__device__ __forceinline__ uint64_t score_key(double s) {
    if (s != s) return 1;
    const int64_t b = __double_as_longlong(s + 0.0);  // -0 counts as 0
    return b < 0 ? ~uint64_t(b) : uint64_t(b) | (uint64_t(1) << 63);
}

template <int CTRL>
__device__ __forceinline__ double max_with(double v) {  // with a lane of the same 16
    const int2 x = __builtin_bit_cast(int2, v);
    const int2 y = make_int2(__builtin_amdgcn_update_dpp(0, x.x, CTRL, 0xF, 0xF, false), __builtin_amdgcn_update_dpp(0, x.y, CTRL, 0xF, 0xF, false));
    return fmax(v, __builtin_bit_cast(double, y));
}

// maximum over the wave (in scalar registers)
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
    x = max(x, uint32_t(__builtin_amdgcn_update_dpp(0, int(x), 0xB1, 0xF, 0xF, false)));   // quad_perm [1,0,3,2]
    x = max(x, uint32_t(__builtin_amdgcn_update_dpp(0, int(x), 0x4E, 0xF, 0xF, false)));   // quad_perm [2,3,0,1]
    x = max(x, uint32_t(__builtin_amdgcn_update_dpp(0, int(x), 0x141, 0xF, 0xF, false)));  // row_half_mirror
    x = max(x, uint32_t(__builtin_amdgcn_update_dpp(0, int(x), 0x140, 0xF, 0xF, false)));  // row_mirror
    return max(max(uint32_t(__builtin_amdgcn_readlane(int(x), 0)), uint32_t(__builtin_amdgcn_readlane(int(x), 16))),
               max(uint32_t(__builtin_amdgcn_readlane(int(x), 32)), uint32_t(__builtin_amdgcn_readlane(int(x), 48))));
}

// The codes of RT rows' query heads, by the whole workgroup (a wave per head):
// positive parts, then negative, as the pages' [max | -min] go. A head below 2^-80,
// whose step or the step's reciprocal may leave fp32's normal range, is scaled by
// 2^64 first, which changes no code, and its step back in 64 bits.
template <int DH, int GP, int RT>
struct QueryCodes {
    alignas(16) uint8_t q[RT * GP][2 * DH];
    double step[RT * GP];
};
template <int DH, int GP, int RT>
__device__ __forceinline__ void form_codes(const SelectArgs& a, int g, int r0, QueryCodes<DH, GP, RT>& qc) {
    const int lane = threadIdx.x & 63, group = a.Hq / a.c.Hkv;
#pragma unroll 1
    for (int h = threadIdx.x >> 6; h < RT * GP; h += blockDim.x >> 6) {
        const float* x = a.q_rot + (int64_t(min(r0 + h / GP, a.c.rows - 1)) * a.Hq + g * group + min(h % GP, group - 1)) * DH;
        float v[DH / 64];
        uint32_t most = 0;  // of the magnitudes' bits
#pragma unroll
        for (int m = 0; m < DH / 64; ++m) v[m] = x[lane + 64 * m];
#pragma unroll
        for (int m = 0; m < DH / 64; ++m) most = max(most, __float_as_uint(v[m]) & 0x7fffffffu);
        const float amax = __uint_as_float(wave_max(most));
        const bool small = amax < 0x1p-80f;
        const float up = small ? 0x1p64f : 1.f, d = amax * up / 127.f, id = d != 0.f ? 1.f / d : 0.f;
#pragma unroll
        for (int m = 0; m < DH / 64; ++m) {
            const int code = round_code(v[m] * up * id);
            qc.q[h][lane + 64 * m] = uint8_t(max(code, 0));
            qc.q[h][DH + lane + 64 * m] = uint8_t(max(-code, 0));
        }
        if (lane == 0) qc.step[h] = double(round11(d)) * (small ? 0x1p-64 : 1.);
    }
}

// The scores of pages 64 k .., k = first, first + stride, ..., for rows r0 .. r0
// + RT - 1 and K/V head g, by one wave; store(row, page, key) for every page the
// row sees, of the rows that see more than `top`. Contains the workgroup's
// barrier between forming the codes and using them.
template <int DH, int GP, int RT, class Store>
__device__ __forceinline__ void score_pages(const SelectArgs& a, int g, int r0, int first, int stride, QueryCodes<DH, GP, RT>& qc, char* tile, Store store) {
    constexpr int KS = DH / 32;                           // 64-byte steps of [max | -min]
    constexpr int ROW = 2 * DH, CH = ROW / 16;            // a page's bounds, and its 16-byte chunks
    constexpr int TT = DH == 128 && RT == 1 ? 4 : 2;      // tiles of 16 pages in flight (four of several rows spill)
    constexpr int CG = RT > 1 ? 1 : GP == 8 ? 2 : TT;     // a lone row's repeated columns finish this many tiles at once
    const PagedRows& c = a.c;
    const int lane = threadIdx.x & 63, g4 = lane >> 4, c16 = lane & 15, sub = c16 % GP, rt = RT > 1 ? c16 / GP : 0, cg = c16 / GP % CG;
    const int r = r0 + min(rt, RT - 1);
    int seq = -1, pos = -1;
    if (r < c.rows) pos = row_position(c, r, &seq);
    const int sees = pos < 0 ? 0 : pos / c.page_size + 1;
    bool todo = rt < RT && sees > a.top && c16 < GP * CG * RT;
    int64_t id0 = -1;  // the first pages, before the codes are formed
    if (RT == 1 && 64 * first + lane < sees && sees > a.top) id0 = pool_page(c, seq, 64 * first + lane);
    form_codes<DH, GP, RT>(a, g, r0, qc);
    __syncthreads();
    if (!__any(todo)) return;

    const int col = RT > 1 ? min(c16, RT * GP - 1) : sub;
    v4i_t q[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) q[s] = *reinterpret_cast<const v4i_t*>(&qc.q[col][64 * s + 16 * g4]);
    const double step = qc.step[col];
    const int64_t page_bytes = kv_summary_page_bytes(c.Hkv, DH);
    const uint8_t* const steps_at = c.summaries + int64_t(c.Hkv) * 2 * DH + 4 * g;
    const uint8_t* const codes_at = c.summaries + int64_t(g) * 2 * DH;
    int put = lane / CH * ROW + (lane % CH ^ lane / CH) * 16, get = c16 * ROW + (g4 ^ c16) * 16;
    // The lanes exchange rows through the tile, whose stores and reads the hardware
    // keeps in order. The compiler does too, as long as a lane's read may be of
    // what the lane itself stored: it is not to know either place. (wave_exchange
    // would hold the global reads as well: 2% of one token's time, 7% of a chunk's
    // over heads of 256 channels.)
    asm volatile("" : "+v"(put), "+v"(get));
    while (const uint64_t left = __ballot(todo)) {  // the rows of one sequence at a time
        const int s0 = RT == 1 ? __builtin_amdgcn_readfirstlane(seq) : __shfl(seq, __ffsll((unsigned long long)left) - 1);
        const bool mine = todo && seq == s0;
        int most = mine ? sees : 0;
        if constexpr (RT > 1)
            for (int off = 8; off > 0; off >>= 1) most = max(most, __shfl_xor(most, off));
        most = __builtin_amdgcn_readfirstlane(most);
        todo = todo && !mine;
        auto page_of = [&](int k) { return 64 * k + lane < most ? pool_page(c, s0, 64 * k + lane) : int64_t(-1); };
        int64_t next = RT == 1 ? id0 : page_of(first);
#pragma unroll 1
        for (int k = first; 64 * k < most; k += stride) {
            const int64_t id = next;
            next = page_of(k + stride);
            const int id_l = id < 0 ? 0 : int(id);  // page 0 for none: read, then ranked last
            const float step_l = id < 0 ? __uint_as_float(0x7fc00000u) : *reinterpret_cast<const float*>(steps_at + id * page_bytes);
#pragma unroll 1
            for (int t0 = 0; t0 < 4; t0 += TT) {
                if (64 * k + 16 * t0 >= most) break;
                // whole records are read (KS loads a tile, 1024 bytes each) and pass
                // through the wave's tile, chunk k of record r at k ^ r: the product
                // wants 16 lanes on 16 records, which a load does as 64 requests
                v4i_t b[TT][KS], sum[TT];
#pragma unroll
                for (int t = 0; t < TT; ++t)
#pragma unroll
                    for (int n = 0; n < KS; ++n) {
                        const int from = 16 * (t0 + t) + (64 * n + lane) / CH;
                        b[t][n] = *reinterpret_cast<const v4i_t*>(codes_at + int64_t(uint32_t(__shfl(id_l, from))) * page_bytes + lane % CH * 16);
                    }
#pragma unroll
                for (int t = 0; t < TT; ++t) {
#pragma unroll
                    for (int n = 0; n < KS; ++n) *reinterpret_cast<v4i_t*>(tile + 1024 * n + (put ^ (64 / CH * n % 16 * 16))) = b[t][n];
                    sum[t] = v4i_t{0, 0, 0, 0};
#pragma unroll
                    for (int s = 0; s < KS; ++s) sum[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(*reinterpret_cast<const v4i_t*>(tile + (get ^ 64 * s)), q[s], sum[t], 0, 0, 0);
                }
#pragma unroll
                for (int t = 0; t < TT; t += CG)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        int x = sum[t][i];
#pragma unroll
                        for (int u = 1; u < CG; ++u) x = cg == u ? sum[t + u][i] : x;
                        double s = double(x) * step;
                        if constexpr (GP >= 2) s = max_with<0xB1>(s);   // quad_perm [1,0,3,2]
                        if constexpr (GP >= 4) s = max_with<0x4E>(s);   // quad_perm [2,3,0,1]
                        if constexpr (GP >= 8) s = max_with<0x141>(s);  // row_half_mirror
                        const int at_page = 16 * (t0 + t + cg) + 4 * g4 + i;
                        s *= double(__shfl(step_l, at_page));
                        if (mine && (GP >= 4 ? sub == i : (i & (GP - 1)) == sub) && 64 * k + at_page < sees) store(rt, 64 * k + at_page, score_key(s));
                    }
            }
        }
    }
}

// NT lanes choose the pages of one (row, K/V head) that sees `sees` > top pages:
// the first and last ones, and of the others the best by key, lane t holding
// pages t, t + NT, ... (at most KPL). The smallest key that is taken is found
// two bits at a time, in the upper 32 bits from the first bit in which the keys
// differ; most searches end there, as soon as exactly the wanted number of keys
// lies at or above. Otherwise the lower 32 bits of those equal so far decide,
// then the order of the pages. All of it is latency, of the counts and of
// fetching the instructions, which run once or a few times: one search serves
// both halves.
struct SelectShared {
    alignas(16) int count[3][4];  // of the waves together: this count's, the last one's, the next one's (zero)
    uint32_t ends[2];
    int place[16 * 16];
};
template <int NT, int KPL>
__device__ __forceinline__ void choose_pages(const uint64_t* keys, int sees, int top, int sink, int recent, int32_t* out, SelectShared* sh) {
    constexpr int NW = NT / 64;
    const int t = NT == 64 ? threadIdx.x & 63 : threadIdx.x, w = t >> 6, lane = t & 63;
    int need = top - sink - recent;
    uint32_t cur[KPL], lo[KPL];
    uint32_t in = 0, open = 0;  // bit i: page NT i + t is taken; may be taken
#pragma unroll
    for (int i = 0; i < KPL; ++i) {
        const int p = NT * i + t;
        const bool may = p >= sink && p < sees - recent;
        const uint64_t k = keys[min(p, sees - 1)];
        cur[i] = may ? uint32_t(k >> 32) : 0;
        lo[i] = uint32_t(k);
        open |= may ? 1u << i : 0u;
        in |= p < sees && !may ? 1u << i : 0u;
    }
    int turn = 0;
    auto over_waves = [&](int (&n)[3]) {  // sums of the waves' counts
        if constexpr (NW > 1) {
            if (lane < 3) atomicAdd(&sh->count[turn][lane], lane == 0 ? n[0] : lane == 1 ? n[1] : n[2]);
            __syncthreads();
            const int4 x = *reinterpret_cast<const int4*>(sh->count[turn]);
            turn = turn == 2 ? 0 : turn + 1;
            // the counters after the next ones were last read before this barrier
            if (t < 4) sh->count[turn == 2 ? 0 : turn + 1][t] = 0;
            n[0] = __builtin_amdgcn_readfirstlane(x.x), n[1] = __builtin_amdgcn_readfirstlane(x.y), n[2] = __builtin_amdgcn_readfirstlane(x.z);
        }
    };
    uint32_t most = 0, least = 0;  // of the upper halves (least: inverted)
#pragma unroll
    for (int i = 0; i < KPL; ++i)
        most = max(most, cur[i]), least = max(least, open >> i & 1 ? ~cur[i] : 0u);
    uint32_t both[2] = {wave_max(most), wave_max(least)};
    if constexpr (NW > 1) {
        if (t < 12) sh->count[t / 4][t % 4] = 0;
        if (t < 2) sh->ends[t] = 0;
        __syncthreads();
        if (lane < 2) atomicMax(&sh->ends[lane], lane ? both[1] : both[0]);
        __syncthreads();
        both[0] = __builtin_amdgcn_readfirstlane(sh->ends[0]), both[1] = __builtin_amdgcn_readfirstlane(sh->ends[1]);
    }
    const uint32_t differ = both[0] ^ ~both[1];
    int bits = differ ? (33 - __builtin_clz(differ)) & ~1 : 0;  // an even number
    uint32_t th = bits == 32 ? 0 : both[0] >> bits << bits;
#pragma unroll 1
    for (int half = 0; half < 2 && need > 0; ++half) {
        bool exact = false;
#pragma unroll 1
        while (bits > 0 && !exact) {  // the largest th with at least `need` keys at or above
            bits -= 2;
            int n[3] = {0, 0, 0};
#pragma unroll
            for (int i = 0; i < KPL; ++i)
#pragma unroll
                for (int v = 0; v < 3; ++v) n[v] += __popcll(__ballot(cur[i] >= (th | uint32_t(v + 1) << bits)));
            over_waves(n);
            const int v = n[2] >= need ? 3 : n[1] >= need ? 2 : n[0] >= need ? 1 : 0;
            th |= uint32_t(v) << bits;
            exact = (v == 3 ? n[2] : v == 2 ? n[1] : v == 1 ? n[0] : 0) == need;
        }
        int above[3] = {0, 0, 0};
#pragma unroll
        for (int i = 0; i < KPL; ++i) {
            const bool up = (open >> i & 1) && (cur[i] > th || (exact && cur[i] == th));
            above[0] += __popcll(__ballot(up));
            const bool still = (open >> i & 1) && !up && cur[i] == th;
            in |= up ? 1u << i : 0u;
            open = (open & ~(1u << i)) | (still ? 1u << i : 0u);
            cur[i] = still ? lo[i] : 0;
        }
        over_waves(above);
        need -= above[0];
        bits = 32;
        th = 0;
    }
    // ascending pages are (i, wave, lane): each chosen page's place, and before it
    // that of the equal keys, of which the first `need` are taken
#pragma unroll 1
    for (int last = need > 0 ? 0 : 1; last < 2; ++last) {
        const uint32_t set = last ? in : open;
        if constexpr (NW > 1) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < KPL; ++i) {
                const int n = __popcll(__ballot(set >> i & 1));
                if (lane == 0) sh->place[i * NW + w] = n;
            }
            __syncthreads();
            if (w == 0) {  // exclusive sums of KPL * NW counts, four a lane
                int v[4], s = 0;
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = 4 * lane + k < KPL * NW ? sh->place[4 * lane + k] : 0;
#pragma unroll
                for (int k = 0; k < 4; ++k) s += v[k];
                int x = s;
                for (int off = 1; off < 64; off <<= 1) {
                    const int y = __shfl_up(x, off);
                    if (lane >= off) x += y;
                }
                x -= s;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if (4 * lane + k < KPL * NW) sh->place[4 * lane + k] = x;
                    x += v[k];
                }
            }
            __syncthreads();
        }
        int at = 0;
#pragma unroll
        for (int i = 0; i < KPL; ++i) {
            const uint64_t m = __ballot(set >> i & 1);
            if constexpr (NW > 1) at = sh->place[i * NW + w];
            const int place = at + __popcll(m & ((uint64_t(1) << lane) - 1));
            if (set >> i & 1) {
                if (last)
                    out[place] = NT * i + t;
                else if (place < need)
                    in |= 1u << i;
            }
            at += __popcll(m);
        }
    }
}

// fewer pages than the list holds: all of them, -1 behind
__device__ __forceinline__ void list_all(int32_t* out, int sees, int top, int t, int nt) {
    for (int i = t; i < top; i += nt) out[i] = i < sees ? i : -1;
}

__device__ __forceinline__ int row_sees(const PagedRows& c, int r) {
    int seq;
    const int pos = row_position(c, r, &seq);
    return pos < 0 ? 0 : pos / c.page_size + 1;
}

// The waves of a workgroup score up to 512 (a lone row) or 1024 pages for RT rows
// into shared memory, then a wave per row chooses: its counts need no barrier.
// Longer lists of a lone row are faster over many workgroups in two launches:
// 1000 pages 11 to 12 against 15 us, 4000 pages 15 against 40 us (one sequence;
// the same times for sixteen). The table's width decides, as the host does not know
// the positions: the 501 pages that take 8.4 us in a table of their own take 11.7 in
// one of 4096. Tiles whose rows belong to several sequences score them one after
// another: sixteen tokens over 501 pages take 41.8 us with row_seq, 12.1 without.
template <int RT>
constexpr int kSelThreads = RT == 1 ? 512 : 256;
template <int DH, int GP, int RT>
__global__ __launch_bounds__(kSelThreads<RT>, 4) void select_pages_kernel(SelectArgs a) {
    const PagedRows& c = a.c;
    const int w = threadIdx.x >> 6, g = blockIdx.x % c.Hkv, r0 = blockIdx.x / c.Hkv * RT;
    extern __shared__ __align__(16) uint64_t sel_keys[];  // [RT][max_pages]
    __shared__ QueryCodes<DH, GP, RT> qc;
    __shared__ __align__(16) char tiles[kSelThreads<RT> / 64][32 * DH];
    score_pages<DH, GP, RT>(a, g, r0, w, kSelThreads<RT> / 64, qc, tiles[w], [&](int rt, int page, uint64_t k) { sel_keys[rt * c.max_pages + page] = k; });
    __syncthreads();
    const int r = r0 + w;
    if (w >= RT || r >= c.rows) return;
    int32_t* out = a.selected + (int64_t(r) * c.Hkv + g) * a.top;
    const uint64_t* keys = sel_keys + w * c.max_pages;
    const int sees = row_sees(c, r);
    if (sees <= a.top)
        list_all(out, sees, a.top, threadIdx.x & 63, 64);
    else if (RT > 1 && sees <= 320)  // five keys a lane instead of eight: 500 rows over 250 pages 17.8 us instead of 19.0, over 100 pages 13.5 instead of 15.0
        choose_pages<64, 5>(keys, sees, a.top, a.sink, a.recent, out, nullptr);
    else if (RT == 1 || sees <= 512)
        choose_pages<64, 8>(keys, sees, a.top, a.sink, a.recent, out, nullptr);
    else if constexpr (RT > 1)
        choose_pages<64, 16>(keys, sees, a.top, a.sink, a.recent, out, nullptr);
}

// More pages: scores to the workspace, a wave per 64 pages at a time ...
template <int DH, int GP, int RT>
__global__ __launch_bounds__(256, 4) void page_scores_kernel(SelectArgs a) {
    const PagedRows& c = a.c;
    const int w = threadIdx.x >> 6, g = blockIdx.x % c.Hkv, r0 = blockIdx.x / c.Hkv * RT;
    __shared__ QueryCodes<DH, GP, RT> qc;
    __shared__ __align__(16) char tiles[4][32 * DH];
    score_pages<DH, GP, RT>(a, g, r0, blockIdx.y * 4 + w, gridDim.y * 4, qc, tiles[w],
                            [&](int rt, int page, uint64_t k) { a.keys[(int64_t(r0 + rt) * c.Hkv + g) * c.max_pages + page] = k; });
}
// ... then a workgroup per (row, K/V head) chooses among up to KPL NT pages
template <int NT, int KPL>
__global__ __launch_bounds__(NT) void choose_pages_kernel(SelectArgs a) {
    const PagedRows& c = a.c;
    const int r = blockIdx.x / c.Hkv, g = blockIdx.x % c.Hkv;
    int32_t* out = a.selected + (int64_t(r) * c.Hkv + g) * a.top;
    __shared__ SelectShared sh;
    const int sees = row_sees(c, r);
    if (sees <= a.top)
        list_all(out, sees, a.top, threadIdx.x, NT);
    else
        choose_pages<NT, KPL>(a.keys + (int64_t(r) * c.Hkv + g) * c.max_pages, sees, a.top, a.sink, a.recent, out, &sh);
}

// any number of pages: the same search with the keys read again for every bit
__global__ __launch_bounds__(1024) void choose_pages_long_kernel(SelectArgs a) {
    const PagedRows& c = a.c;
    const int t = threadIdx.x, lane = t & 63, w = t >> 6, r = blockIdx.x / c.Hkv, g = blockIdx.x % c.Hkv;
    int32_t* out = a.selected + (int64_t(r) * c.Hkv + g) * a.top;
    const int sees = row_sees(c, r);
    if (sees <= a.top) {
        list_all(out, sees, a.top, t, 1024);
        return;
    }
    __shared__ int part[16];
    const uint64_t* keys = a.keys + (int64_t(r) * c.Hkv + g) * c.max_pages;
    auto key = [&](int i) { return i >= sees ? 0 : i < a.sink || i >= sees - a.recent ? ~uint64_t(0) : keys[i]; };
    auto total = [&](int n) {  // of the waves' counts
        __syncthreads();
        if (lane == 0) part[w] = n;
        __syncthreads();
        n = 0;
        for (int k = 0; k < 16; ++k) n += part[k];
        return n;
    };
    uint64_t th = 0;  // the largest with at least top keys at or above
    for (int bit = 63; bit >= 0; --bit) {
        const uint64_t u = th | (uint64_t(1) << bit);
        int n = 0;
        for (int i = t; i - t < sees; i += 1024) n += __popcll(__ballot(key(i) >= u));
        if (total(n) >= a.top) th = u;
    }
    int n = 0;
    for (int i = t; i - t < sees; i += 1024) n += __popcll(__ballot(key(i) > th));
    int equal = a.top - total(n), at = 0;
    const uint64_t below = (uint64_t(1) << lane) - 1;
    if (w != 0) return;
    for (int i = lane; i - lane < sees && at < a.top; i += 64) {
        const uint64_t k = key(i), eq = __ballot(k == th);
        const bool take = k > th || (k == th && __popcll(eq & below) < equal);
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
// Both products run on the matrix cores, and no lane exchanges anything between
// them (lane = 16 g + c below):
//   scores   S^T[key][column] = K Q^T, 16 keys x 16 columns x 32 channels. Lane
//            (g, c) brings 16 bytes of key c, and gets the scores of keys 4 g ..
//            4 g + 3 for column c. A load whose neighbouring lanes read
//            different rows takes several times as long as one of whole rows, so
//            the keys are read as whole rows and pass through a tile of shared
//            memory that is the wave's own.
//   values   O^T[channel][column] += V^T P^T, 16 channels x 16 columns x 32
//            keys. The order of the 32 keys is free as long as both operands
//            agree, so a lane's eight scores (keys 4 g .. 4 g + 3 of both
//            halves) are its operand, and lane (g, c) loads those keys'
//            channels 8 c .. 8 c + 7: whole rows per load, transposed in the
//            lane's registers. Product e covers channels 8 c + e, and a lane
//            ends with 32 consecutive channels of its column's head.
// The matrix cores multiply fp16; queries and weights are fp32. Each is split
// into two fp16 terms (22 bits). A head's query is scaled by a power of two to
// at most 1 first, and a weight is 2^13 2^(s - m) with m at most 2 below
// the running maximum, so that neither term leaves fp16's range: terms are
// dropped below 2^-38 of the largest. (The factor comes after the exponential:
// s - m + 13 would be rounded to 2^-21, s - m near the maximum hardly at all.)
// Against 64 bits lists of 3, 64 and 2048 keys of random fp16 pages are off by
// 1.0e-7, 1.9e-7 and 2.4e-7 (2-norm), a plain fp32 evaluation by 0.9e-7, 1.6e-7 and
// 3.3e-7. The up to eight heads of a group (or of
// several rows) times two terms are the 16 columns: head h in columns h and h +
// 8, added where both are done.
// fp16 pages: keys and values are exact.
// Q8_0 pages: codes are exact in fp16. A key block's product is scaled by the
// block's step afterwards. A value block's step goes into the weights: column
// (block, head) holds weights times that block's steps, for four heads at a
// time, and of its result the 32 channels of that block count. The steps'
// power of two is kept apart per column (`ve`), as theirs range as widely as
// fp16 does.
//
// Bound: few tokens, latency (one token over 2048 keys 6.3 us, and 3.9 for
// merging the ranges); batches of tokens, HBM: sixteen over 2048 Q8_0 keys each
// (71 MB) 19 us, eight over 48 pages of 256-wide heads (101 MB) 22 us, sixteen
// over 32 fp16 pages (134 MB) 30 us, 3.7 to 4.6 TB/s of a copy's 4.76, and the
// merge 4 us. Chunks, what L2 gives and the vector instructions around the
// products: 500 rows over 16 pages each read 1.5 GB through L2 for 92 MB of
// distinct bytes, 88 to 89 us a call among others (98 alone under the profiler; eight
// heads per K/V head 109, 256-wide heads 85). Q8_0 pages, vector instructions: 140
// us, eight heads per K/V head 228.
typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
typedef float f4_t __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kPShift = 13;      // a weight's terms are of 2^13 2^(s - m); its part in the total is 2^(s - m)
constexpr float kPOne = 8192.f;  // 2^kPShift
constexpr float kPSlack = 2.f;   // m may lag the maximum by this: weights stay below 2^15

__device__ __forceinline__ float column_other(float x) {  // the value of column c ^ 8
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x128, 0xF, 0xF, false));  // row_ror:8
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

// A workgroup's pages, in shared memory: the pool page, how many of its keys each
// row sees (0: none, or not selected), and the most of them.
template <int R>
struct ListEntry {
    int32_t page;
    uint16_t most, keys[R];
};

template <int DH, int SLOTS>
struct SparseMerge {  // the four waves' results; a slot per (row, head)
    float m[4][SLOTS], l[4][SLOTS], o[4][SLOTS][DH];
};

// The pages of R rows' lists, each once with the rows' key counts: a page that
// several rows of one sequence select is read once for all of them. `top`
// entries a row, at most 512 together; a page's second place in one list stays an entry
// of its own. Entries in the order of row 0's list, then what row 1 adds, ...;
// returns their number.
struct UnionScratch {
    int32_t lp[512], page[512], count[512], sums[2][4];
    uint16_t keys[512][4];
};
template <int R>
__device__ __forceinline__ int build_union(const SparseAttnArgs& a, int g, int r0, const int (&seq)[R], const int (&pos)[R], ListEntry<R>* list, UnionScratch& u) {
    const PagedRows& c = a.c;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, top = a.top, ps = c.page_size, n = R * top;
    for (int x = tid; x < n; x += 256) {
        const int j = x / top;
        int lp = -1, count = 0, page = 0;
#pragma unroll
        for (int k = 0; k < R; ++k)
            if (k == j && pos[k] >= 0) {
                lp = a.selected[(int64_t(r0 + k) * c.Hkv + g) * top + x - j * top];
                if (lp >= 0 && lp <= pos[k] / ps) {
                    const int64_t id = pool_page(c, seq[k], lp);
                    if (id >= 0) page = int32_t(id), count = min(ps, pos[k] + 1 - lp * ps);
                }
            }
        u.lp[x] = count ? lp : -1;
        u.page[x] = page;
        u.count[x] = count;
#pragma unroll
        for (int k = 0; k < R; ++k) u.keys[x][k] = 0;
    }
    __syncthreads();
    bool own[2] = {false, false};
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int x = tid + 256 * k;
        if (x >= n || u.lp[x] < 0) continue;
        const int j = x / top, lp = u.lp[x];
        int owner = x;
        bool again = false;
#pragma unroll 8
        for (int y = j * top; y < x; ++y) again |= u.lp[y] == lp;
        if (!again) {
            int s = 0;
#pragma unroll
            for (int q = 0; q < R; ++q) s = q == j ? seq[q] : s;
#pragma unroll
            for (int q = R - 2; q >= 0; --q) {  // the earliest row's first place wins
                if (q >= j || seq[q] != s) continue;
#pragma unroll 8
                for (int y = (q + 1) * top - 1; y >= q * top; --y) owner = u.lp[y] == lp ? y : owner;
            }
        }
        own[k] = owner == x;
        u.keys[owner][j] = uint16_t(u.count[x]);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int s = __popcll(__ballot(own[k]));
        if (lane == 0) u.sums[k][w] = s;
    }
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        int at = total;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            at += q < w ? u.sums[k][q] : 0;
            total += u.sums[k][q];
        }
        const uint64_t m = __ballot(own[k]);
        at += __popcll(m & ((uint64_t(1) << lane) - 1));
        if (own[k]) {
            const int x = tid + 256 * k;
            ListEntry<R> e;
            e.page = u.page[x];
            e.most = 0;
#pragma unroll
            for (int q = 0; q < R; ++q) {
                e.keys[q] = u.keys[x][q];
                e.most = max(e.most, e.keys[q]);
            }
            list[at] = e;
        }
    }
    return total;
}

template <int DH>
__device__ __forceinline__ void sparse_store(const SparseAttnArgs& a, int r, int h, int ch, float o, float l, float gate) {
    const int64_t width = int64_t(a.Hq) * DH, idx = int64_t(r) * width + int64_t(h) * DH + ch;
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

// A (row, query head) over the keys of a workgroup's list that the row (its k-th)
// sees, in plain fp32 by one wave: a lane per key for the scores, a lane per
// channel, of 64 from `ch0` on, for the sum. A key of score -inf has weight 0;
// where every key does, m is -inf and `any` true.
template <int DH, bool Q8, int R>
__device__ __forceinline__ void attend_plain(const SparseAttnArgs& a, int r, int k, int g, int h, int ch0, const ListEntry<R>* list, int ne, float& m, float& l, float& o,
                                             bool& any) {
    const PagedRows& c = a.c;
    const int lane = threadIdx.x & 63;
    const float* const q = a.q_rot + (int64_t(r) * a.Hq + h) * DH;
    const float scale = a.score_scale * kLog2e;
    m = -INFINITY, l = o = 0.f, any = false;
#pragma unroll 1
    for (int e = 0; e < ne; ++e) {
        const int64_t page = list[e].page;
        const int n = list[e].keys[k];
        const _Float16* const fpage = f16_page<DH>(c, page);
        const uint8_t* const qpage = q8_page<DH>(c, page);
        const _Float16* const steps = reinterpret_cast<const _Float16*>(qpage + q8_scales_at<DH>(c));
        any |= n > 0;
#pragma unroll 1
        for (int t0 = 0; t0 < n; t0 += 64) {
            const bool mine = t0 + lane < n;
            const int64_t krow = page_row_index(c, 0, g, mine ? t0 + lane : t0);
            float s = 0.f;
#pragma unroll 1
            for (int ch = 0; ch < DH; ch += 8) {
                float x[8];
                if constexpr (Q8) {
                    const int2 w = *reinterpret_cast<const int2*>(qpage + krow * DH + ch);
                    const float d = float(steps[krow * (DH / 32) + ch / 32]);
#pragma unroll
                    for (int u = 0; u < 8; ++u) x[u] = d * float(int8_t((u < 4 ? w.x : w.y) >> (8 * (u & 3))));
                } else {
                    const h8_t w = *reinterpret_cast<const h8_t*>(fpage + krow * DH + ch);
#pragma unroll
                    for (int u = 0; u < 8; ++u) x[u] = float(w[u]);
                }
#pragma unroll
                for (int u = 0; u < 8; ++u) s += q[ch + u] * x[u];
            }
            s = mine ? s * scale : -INFINITY;
            float m2 = s;
            for (int off = 32; off > 0; off >>= 1) m2 = fmaxf(m2, __shfl_xor(m2, off));
            m2 = fmaxf(m, m2);
            const float p = mine ? exp2_hw(s - (m2 == -INFINITY ? 0.f : m2)) : 0.f, f = m == -INFINITY ? 1.f : exp2_hw(m - m2);
            m = m2;
            float sum = p;
            for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
            l = l * f + sum;
            o *= f;
            const int last = min(64, n - t0);
#pragma unroll 1
            for (int j0 = 0; j0 < last; j0 += 8) {
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int64_t at = page_row_index(c, 1, g, t0 + min(j0 + j, last - 1)) * DH + ch0 + lane;
                    if constexpr (Q8)
                        v[j] = float(steps[at / 32]) * float(int8_t(qpage[at]));
                    else
                        v[j] = float(fpage[at]);
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) o += __shfl(p, j0 + j) * (j0 + j < last ? v[j] : 0.f);
            }
        }
    }
}

// R rows by GP heads each, in GQ sets of 16 columns. fp16 pages: one set, R GP <= 8
// of GP a power of two, times two terms; R > 1: the rows of a chunk, which mostly
// select the same pages. Q8_0 pages: one row, a set for every four heads.
//
// Infinities and NaNs: the two terms of a query or weight may differ in sign, or
// one be 0, so that an infinite key or value turns a score or sum to NaN which
// the definition has infinite; and a row's columns, of weight 0 for the pages of
// other rows, get 0 times whatever those hold. All of it leaves a result that is
// not finite. What leaves none is marked: a column all of whose keys score -inf
// (NaN by the definition), and with Q8_0 any score of -inf (a block's infinite
// step times the sum of its products, where products may be infinite of both
// signs). A wave among whose 64 results (channels of one row and head) some are
// not finite forms them again in plain fp32, over the row's own keys: sixteen Q8_0
// sequences 219 us instead of 38 if every page holds such keys and values, 500
// fp16 rows 1.8 ms instead of 0.11 (one call, waited for).
template <int DH, bool Q8, int GQ, int R, int GP>
__global__ __launch_bounds__(256) void attn_sparse_kernel(SparseAttnArgs a, int per, int nsplit) {
    constexpr int KB = DH / 32, VH = DH / 128;  // 32-channel blocks, 128-channel halves
    static_assert(Q8 ? R == 1 && GP == 4 * GQ : GQ == 1 && R * GP <= 8);
    constexpr int SLOTS = Q8 ? 4 * GQ : 8;
    const PagedRows& c = a.c;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, g4 = lane >> 4, c16 = lane & 15;
    // K/V head fastest: with eight of them each XCD's L2 holds one head's pages
    const int tiles = R > 1 ? (c.rows + R - 1) / R : c.rows;
    const int g = blockIdx.x % c.Hkv, r0 = int(blockIdx.x / c.Hkv % tiles) * R, split = blockIdx.x / c.Hkv / tiles;
    const int group = a.Hq / c.Hkv, ps = c.page_size;
    int seq[R], pos[R];
    bool some = false;
#pragma unroll
    for (int k = 0; k < R; ++k) {
        pos[k] = seq[k] = -1;
        if (R == 1 || r0 + k < c.rows) pos[k] = row_position(c, r0 + k, &seq[k]);
        some |= pos[k] >= 0;
    }
    if (!some) return;
    // the row and head of a column of set x
    const int col_row = R == 1 ? 0 : min((c16 & 7) / GP, R - 1);
    auto head_of = [&](int x) { return Q8 ? 4 * x + (c16 & 3) : c16 & (GP - 1); };
    auto used = [&](int x) {  // columns that stand for a row and head
        bool live = head_of(x) < group && (Q8 || (c16 & 7) / GP < R);
#pragma unroll
        for (int k = 0; k < R; ++k) live = live && (col_row != k || pos[k] >= 0);
        return live;
    };
    extern __shared__ __align__(16) char list_mem[];
    ListEntry<R>* const list = reinterpret_cast<ListEntry<R>*>(list_mem);
    // the waves' key tiles (32 keys each); before, what the list is built in, and
    // behind, the waves' results
    constexpr int ROW = Q8 ? DH : 2 * DH, TILE = 32 * ROW, CH = ROW / 16;
    using Merge = SparseMerge<DH, SLOTS>;
    __shared__ __align__(16) char shared_mem[sizeof(Merge) > 4 * TILE ? sizeof(Merge) : 4 * TILE];
    Merge& mg = *reinterpret_cast<Merge*>(shared_mem);
    char* const tile = shared_mem + w * TILE;
    // Chunk k (16 bytes) of a tile's row is kept at k ^ row % 16 (Q8_0: row / 2 % 8),
    // so that neither the stores (whole rows) nor the reads (one chunk of 16 rows)
    // meet in a bank. Load n of a unit's keys is rows 64 n / CH ..: its place, and
    // that of the 64-byte step k of row c16, differ from lane constants by the
    // exclusive or of a constant (formed at each use: kept, they cost ten registers)
    int put = (lane / CH) * ROW + ((lane % CH) ^ (Q8 ? lane / CH >> 1 & 7 : lane / CH)) * 16;
    int get = c16 * ROW + (Q8 ? ((g4 >> 1) ^ (c16 >> 1 & 7)) * 16 + (g4 & 1) * 8 : (g4 ^ c16) * 16);
    auto put_at = [&](int n) { return 1024 * n + (put ^ ((64 / CH * n % 16 >> (Q8 ? 1 : 0)) * 16)); };
    auto get_at = [&](int hf, int k) { return 16 * hf * ROW + (get ^ (Q8 ? 32 * k : 64 * k)); };
    // the columns' query terms: the first in columns 0 .. 7, the second in 8 .. 15
    // (of the same heads). A wave forms its share of the 32-channel blocks for all
    // four.
    constexpr int PER = KB / 4;
    __shared__ h8_t terms[GQ][KB][64];
    __shared__ float biggest[GQ][4][16];
    float qv[GQ][PER][8];  // on the way while the list is built
#pragma unroll
    for (int x = 0; x < GQ; ++x) {
        const float* q_row = a.q_rot + (int64_t(min(r0 + col_row, c.rows - 1)) * a.Hq + g * group + min(head_of(x), group - 1)) * DH;
#pragma unroll
        for (int y = 0; y < PER; ++y) {
            const float4* p = reinterpret_cast<const float4*>(q_row + 32 * (PER * w + y) + 8 * g4);
            const float4 lo = p[0], hi = p[1];
            qv[x][y][0] = lo.x, qv[x][y][1] = lo.y, qv[x][y][2] = lo.z, qv[x][y][3] = lo.w;
            qv[x][y][4] = hi.x, qv[x][y][5] = hi.y, qv[x][y][6] = hi.z, qv[x][y][7] = hi.w;
        }
    }
    int ne;
    if constexpr (R > 1) {
        static_assert(sizeof(UnionScratch) <= sizeof(shared_mem));
        ne = __builtin_amdgcn_readfirstlane(build_union<R>(a, g, r0, seq, pos, list, *reinterpret_cast<UnionScratch*>(shared_mem)));
    } else {
        const int e0 = split * per;
        ne = min(per, a.top - e0);
        for (int i = tid; i < ne; i += 256) {
            const int lp = a.selected[(int64_t(r0) * c.Hkv + g) * a.top + e0 + i];
            ListEntry<R> e{0, 0, {0}};
            if (lp >= 0 && lp <= pos[0] / ps) {
                const int64_t page = pool_page(c, seq[0], lp);
                if (page >= 0) e.page = int32_t(page), e.most = e.keys[0] = uint16_t(min(ps, pos[0] + 1 - lp * ps));
            }
            list[i] = e;
        }
    }

#pragma unroll
    for (int x = 0; x < GQ; ++x) {
        float amax = 0.f;
#pragma unroll
        for (int y = 0; y < PER; ++y)
#pragma unroll
            for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(qv[x][y][j]));
        amax = max_over_rows(amax);
        if (g4 == 0) biggest[x][w][c16] = amax;
    }
    __syncthreads();
    float qscale[GQ];
#pragma unroll
    for (int x = 0; x < GQ; ++x) {
        const bool have = used(x);
        const float amax = fmaxf(fmaxf(biggest[x][0][c16], biggest[x][1][c16]), fmaxf(biggest[x][2][c16], biggest[x][3][c16]));
        const int e = __builtin_amdgcn_frexp_expf(amax);  // amax <= 2^e
        qscale[x] = ldexpf(a.score_scale * kLog2e, e);
#pragma unroll
        for (int y = 0; y < PER; ++y) {
            h8_t f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                _Float16 hi, lo;
                split_f16(have ? ldexpf(qv[x][y][j], -e) : 0.f, hi, lo);
                f[j] = c16 < 8 ? hi : lo;
            }
            terms[x][PER * w + y][lane] = f;
        }
    }
    __syncthreads();
    h8_t qf[GQ][KB];
#pragma unroll
    for (int x = 0; x < GQ; ++x)
#pragma unroll
        for (int y = 0; y < KB; ++y) qf[x][y] = terms[x][y][lane];

    const int hp = ps / 16, halves = ne * hp, step_e = 8 / hp, step_b = 8 % hp;
    const int wu = __builtin_amdgcn_readfirstlane(w);
    const int64_t page_stride = Q8 ? 2 * int64_t(c.Hkv) * ps * (DH + DH / 16) : 4 * int64_t(c.Hkv) * ps * DH;
    const int64_t krow0 = int64_t(g) * ps, vrow0 = (int64_t(c.Hkv) + g) * ps;
    const char* const pool = reinterpret_cast<const char*>(c.pages);
    const float is_lo = c16 < 8 ? 0.f : 1.f;
    float m[GQ], l[GQ], low[GQ];  // low: Q8_0, the smallest score, or 0
    int saw[GQ];                  // whether the column has seen a key
    f4_t o[GQ][8 * VH];
#pragma unroll
    for (int x = 0; x < GQ; ++x) {
        m[x] = -INFINITY;
        l[x] = low[x] = 0.f;
        saw[x] = 0;
#pragma unroll
        for (int e = 0; e < 8 * VH; ++e) o[x][e] = f4_t{0.f, 0.f, 0.f, 0.f};
    }
    int ve = -200;  // Q8_0: the column's accumulators are in units of 2^ve

    // the wave's units: halves 2 (w + 4 n) and the one behind, as entry and 16-key
    // block; `next` finds the following one that holds keys
    int entry[2], block[2], at = wu;
#pragma unroll
    for (int s = 0; s < 2; ++s) entry[s] = (2 * wu + s) / hp, block[s] = (2 * wu + s) % hp;
    int next_page[2], next_off[2], next_nv[2], next_mine[GQ][2];
    auto next = [&] {
        while (2 * at < halves) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const ListEntry<R>& le = list[min(entry[s], ne - 1)];
                next_off[s] = 16 * block[s];
                next_page[s] = __builtin_amdgcn_readfirstlane(le.page);
                const bool real = 2 * at + s < halves;
                next_nv[s] = real ? __builtin_amdgcn_readfirstlane(max(0, min(16, int(le.most) - next_off[s]))) : 0;
#pragma unroll
                for (int x = 0; x < GQ; ++x) {
                    next_mine[x][s] = next_nv[s];
                    if constexpr (R > 1) next_mine[x][s] = min(next_nv[s], max(0, int(le.keys[col_row]) - next_off[s]));
                }
                entry[s] += step_e;
                block[s] += step_b;
                if (block[s] >= hp) block[s] -= hp, ++entry[s];
            }
            at += 4;
            if (next_nv[0] + next_nv[1] == 0) continue;
            if (next_nv[0] == 0) next_page[0] = next_page[1], next_off[0] = next_off[1];  // an entry of none names no page: read what is there, use nothing
            if (next_nv[1] == 0) next_page[1] = next_page[0], next_off[1] = next_off[0];
            return true;
        }
        return false;
    };
    // the keys through the wave's tile: read as whole rows, lane by lane on (16
    // lanes on 16 rows, as the product wants them, are 64 requests a load: 118 us
    // of 146 for 500 rows' loads alone), 16 bytes each; of one row's fp16 heads of
    // 128 channels a unit ahead, else there are not the registers
    constexpr int LOADS = 2 * CH / 4;  // of 1024 bytes, half of them a half
    constexpr bool AHEAD = DH == 128 && R == 1 && !Q8;
    v4i_t staged[LOADS];
    auto stage = [&](const int (&page)[2], const int (&off)[2]) {
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            const __amdgpu_buffer_rsrc_t b = buffer_of(pool + page[hf] * page_stride + (krow0 + off[hf]) * ROW, 16 * ROW);
#pragma unroll
            for (int k = 0; k < LOADS / 2; ++k) staged[hf * (LOADS / 2) + k] = __builtin_amdgcn_raw_buffer_load_b128(b, 16 * lane + 1024 * k, 0, 0);
        }
    };
    bool more = next();
    if (AHEAD && more) stage(next_page, next_off);
    while (more) {
        int page[2], off[2], nv[2], mine[GQ][2];  // keys of the half that any row, the set's column sees
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            page[s] = next_page[s], off[s] = next_off[s], nv[s] = next_nv[s];
#pragma unroll
            for (int x = 0; x < GQ; ++x) mine[x][s] = next_mine[x][s], saw[x] |= mine[x][s];
        }
        const bool full = nv[0] + nv[1] == 32;
        auto weights_base = [&](int x, const f4_t (&s)[2], const int (&sees)[2], auto rescale) {
            float top = -INFINITY;
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                const float of = fmaxf(fmaxf(s[hf][0], s[hf][1]), fmaxf(s[hf][2], s[hf][3]));
                top = fmaxf(top, R > 1 && sees[hf] == 0 ? -INFINITY : of);
            }
            if (__any(top > m[x] + kPSlack)) {
                const float m2 = fmaxf(m[x], max_over_rows(top)), f = m2 == -INFINITY ? 1.f : exp2_hw(m[x] - m2);
                m[x] = m2;
                l[x] *= f;
                rescale(f);
            }
            return fmaxf(m[x], -3e38f);  // a column that has seen no key: 2^-inf, not NaN
        };

        if (!AHEAD) stage(page, off);
        asm volatile("" : "+v"(put), "+v"(get));  // see put_at
        __builtin_amdgcn_sched_barrier(0);  // a unit's loads are all in flight before the first is waited for
        if constexpr (!Q8) {
            h8_t vf[VH][8];
            // 256 channels: the values take the keys' registers once those are in the
            // tile, so that two workgroups fit a compute unit
            constexpr bool LATE = DH == 256;
#pragma unroll
            for (int turn = 0; turn < 2; ++turn) {
                if (turn == (LATE ? 1 : 0)) {
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        const __amdgpu_buffer_rsrc_t b = buffer_of(pool + page[hf] * page_stride + (vrow0 + off[hf]) * ROW, 16 * ROW);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int v = 0; v < VH; ++v)
                                vf[v][4 * hf + i] = __builtin_bit_cast(h8_t, __builtin_amdgcn_raw_buffer_load_b128(b, 8 * DH * g4 + 16 * c16 + 2 * DH * i + 256 * v, 0, 0));
                    }
                    __builtin_amdgcn_sched_barrier(0);
                } else {
#pragma unroll
                    for (int k = 0; k < LOADS; ++k) *reinterpret_cast<v4i_t*>(tile + put_at(k)) = staged[k];
                    wave_exchange();
                    __builtin_amdgcn_sched_barrier(0);
                    if (AHEAD) {
                        more = next();
                        if (more) stage(next_page, next_off);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            f4_t acc[GQ][2];
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
#pragma unroll
                for (int x = 0; x < GQ; ++x) acc[x][hf] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < KB; ++k) {
                    const h8_t kf = *reinterpret_cast<const h8_t*>(tile + get_at(hf, k));
#pragma unroll
                    for (int x = 0; x < GQ; ++x) acc[x][hf] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[x][k], acc[x][hf], 0, 0, 0);
                }
            }
            h8_t pf[GQ];
#pragma unroll
            for (int x = 0; x < GQ; ++x) {
                f4_t s[2];
#pragma unroll
                for (int hf = 0; hf < 2; ++hf)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[hf][i] = (acc[x][hf][i] + column_other(acc[x][hf][i])) * qscale[x];
                // halves that a column sees in part are masked key by key, halves
                // that it does not see as a whole
                const bool partly = R == 1 ? !full : __any((mine[x][0] & 15) + (mine[x][1] & 15));
                if (partly) {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (4 * g4 + (i & 3) >= mine[x][i >> 2]) s[i >> 2][i & 3] = -INFINITY;
                }
                const float base = weights_base(x, s, mine[x], [&](float f) {
#pragma unroll
                    for (int e = 0; e < 8 * VH; ++e) o[x][e] *= f;
                });
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    const float less = R > 1 && mine[x][hf] == 0 ? INFINITY : base;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float p = exp2_hw(s[hf][i] - less);
                        l[x] += p;
                        p *= kPOne;
                        asm("" : "+v"(p));  // as in split_f16
                        // the column's term: fp16(p), or of the rest (is_lo 1)
                        const float rest = __builtin_fmaf(-float(_Float16(p)), is_lo, p);
                        pf[x][4 * hf + i] = _Float16(rest);
                    }
                }
            }
            if (!full) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (4 * g4 + (i & 3) >= nv[i >> 2]) {
#pragma unroll
                        for (int v = 0; v < VH; ++v) vf[v][i] = h8_t{};
                    }
            }
#pragma unroll
            for (int v = 0; v < VH; ++v)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    h8_t y;
#pragma unroll
                    for (int i = 0; i < 8; ++i) y[i] = vf[v][i][e];
#pragma unroll
                    for (int x = 0; x < GQ; ++x) o[x][8 * v + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y, pf[x], o[x][8 * v + e], 0, 0, 0);
                }
        } else {
            uint2 vq[8];
            v4i_t kd[2][2], vd[2][2];
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                const char *pg = pool + page[hf] * page_stride, *steps = pg + q8_scales_at<DH>(c);
                const __amdgpu_buffer_rsrc_t vb = buffer_of(pg + (vrow0 + off[hf]) * ROW, 16 * ROW);
                const __amdgpu_buffer_rsrc_t kd_b = buffer_of(steps + (krow0 + off[hf]) * (2 * KB), 32 * KB), vd_b = buffer_of(steps + (vrow0 + off[hf]) * (2 * KB), 32 * KB);
#pragma unroll
                for (int n = 0; n < 2; ++n) kd[hf][n] = __builtin_amdgcn_raw_buffer_load_b128(kd_b, 8 * KB * g4 + 16 * n, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; ++i) vq[4 * hf + i] = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(vb, 4 * DH * g4 + 8 * c16 + DH * i, 0, 0));
#pragma unroll
                for (int n = 0; n < 2; ++n) vd[hf][n] = __builtin_amdgcn_raw_buffer_load_b128(vd_b, 8 * KB * g4 + 16 * n, 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int k = 0; k < LOADS; ++k) *reinterpret_cast<v4i_t*>(tile + put_at(k)) = staged[k];
            wave_exchange();
            __builtin_amdgcn_sched_barrier(0);
            // scores: a block's product, then the key's step of that block
            f4_t s[GQ][2];
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                h8_t steps[2] = {__builtin_bit_cast(h8_t, kd[hf][0]), __builtin_bit_cast(h8_t, kd[hf][1])};  // [key][block]
#pragma unroll
                for (int x = 0; x < GQ; ++x) s[x][hf] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < KB; ++k) {
                    const h8_t kf = codes8_to_half(*reinterpret_cast<const uint2*>(tile + get_at(hf, k)));
#pragma unroll
                    for (int x = 0; x < GQ; ++x) {
                        f4_t acc = {0.f, 0.f, 0.f, 0.f};
                        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[x][k], acc, 0, 0, 0);
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[x][hf][i] = __builtin_fmaf(float(steps[i >> 1][4 * (i & 1) + k]), acc[i], s[x][hf][i]);
                    }
                }
#pragma unroll
                for (int x = 0; x < GQ; ++x)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const bool sees = 4 * g4 + i < mine[x][hf];
                        const float sum = (s[x][hf][i] + column_other(s[x][hf][i])) * qscale[x];
                        low[x] = fminf(low[x], sees ? sum : 0.f);
                        s[x][hf][i] = sees ? sum : -INFINITY;
                    }
            }
            // the column's value steps, 2^(13 - ve) times, 0 past the keys
            float d[8], dmax = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const v4i_t two = vd[i >> 2][(i & 3) >> 1];
                const uint64_t four = (i & 1) ? uint64_t(uint32_t(two.w)) << 32 | uint32_t(two.z) : uint64_t(uint32_t(two.y)) << 32 | uint32_t(two.x);
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
            for (int i = 0; i < 8; ++i) d[i] = ldexpf(d[i], kPShift - ve);
            h8_t ph[GQ], pl[GQ];
#pragma unroll
            for (int x = 0; x < GQ; ++x) {
                const float base = weights_base(x, s[x], mine[x], [&](float f) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) o[x][e] *= f;
                });
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
        if (!AHEAD) more = next();
        wave_exchange();  // the tile's reads, before the next unit's stores
    }

    // merge: a lane holds channels 128 v + 32 g4 + 8 i + e of its column's head
    __syncthreads();
#pragma unroll
    for (int x = 0; x < GQ; ++x) {
        const bool marked = (Q8 && low[x] == -INFINITY) || (saw[x] && m[x] == -INFINITY);
        const float sum = kPOne * sum_over_rows(marked ? NAN : l[x]);
        const int slot = Q8 ? 4 * x + (c16 & 3) : c16 & 7;
#pragma unroll
        for (int n = 0; n < 8 * VH; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (Q8)
                    o[x][n][i] = ldexpf(o[x][n][i], ve);
                else
                    o[x][n][i] += column_other(o[x][n][i]);
            }
        if (used(x) && (Q8 ? (c16 >> 2) == g4 : c16 < 8)) {
            if (Q8 || g4 == 0) mg.m[w][slot] = m[x], mg.l[w][slot] = sum;
#pragma unroll
            for (int v = 0; v < VH; ++v)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float4* to = reinterpret_cast<float4*>(&mg.o[w][slot][128 * v + 32 * g4 + 8 * i]);
                    to[0] = make_float4(o[x][8 * v][i], o[x][8 * v + 1][i], o[x][8 * v + 2][i], o[x][8 * v + 3][i]);
                    to[1] = make_float4(o[x][8 * v + 4][i], o[x][8 * v + 5][i], o[x][8 * v + 6][i], o[x][8 * v + 7][i]);
                }
        }
    }
    __syncthreads();
    // up to NI results a lane, all their gates on the way at once
    constexpr int NI = (R * (R == 1 ? 8 : GP) * DH + 255) / 256;
    const int to = R * group * DH;
    auto record = [&](int h) { return a.work + ((int64_t(r0) * a.Hq + g * group + h) * nsplit + split) * (DH + 4); };
    auto live = [&](int k) {
        bool yes = R == 1;
#pragma unroll
        for (int q = 0; q < R && R > 1; ++q) yes = yes || (q == k && pos[q] >= 0);
        return yes;
    };
    // the maximum of the four waves' parts of a result, their shares and total
    auto parts = [&](int slot, float (&f)[4], float& lv) {
        float mw[4], lw[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) mw[q] = mg.m[q][slot], lw[q] = mg.l[q][slot];
        const float mx = fmaxf(fmaxf(mw[0], mw[1]), fmaxf(mw[2], mw[3]));
        lv = 0.f;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            f[q] = mw[q] == -INFINITY && lw[q] == 0.f ? 0.f : exp2_hw(mw[q] - mx);  // a wave without keys: 0
            lv = __builtin_fmaf(f[q], lw[q], lv);
        }
        return mx;
    };
    auto slot_of = [&](int k, int h) { return k * GP + h; };
    float gate[NI];
    if (nsplit == 1) {
#pragma unroll
        for (int n = 0; n < NI; ++n) {
            const int e = min(tid + 256 * n, to - 1), k = R == 1 ? 0 : e / (group * DH);
            gate[n] = a.proj[int64_t(min(r0 + k, c.rows - 1)) * a.proj_stride + (g * group + e / DH - k * group) * 2 * DH + DH + e % DH];
        }
    }
    uint32_t again = 0;  // bit n: the wave's results n are not all finite
#pragma unroll
    for (int n = 0; n < NI; ++n) {
        const int e = tid + 256 * n;
        if (e >= to) break;
        const int k = R == 1 ? 0 : e / (group * DH), h = e / DH - k * group, ch = e % DH;
        if (!live(k)) continue;
        const int slot = slot_of(k, h);
        float f[4], lv, ov = 0.f;
        const float mx = parts(slot, f, lv);
#pragma unroll
        for (int q = 0; q < 4; ++q) ov = __builtin_fmaf(f[q], mg.o[q][slot][ch], ov);
        again |= __any(__builtin_fmaf(ov, 0.f, lv * 0.f) != 0.f) ? 1u << n : 0u;
        if (nsplit == 1) {
            sparse_store<DH>(a, r0 + k, g * group + h, ch, ov, lv, gate[n]);
        } else {
            float* rec = record(h);
            rec[4 + ch] = ov;
            if (ch == 0) rec[0] = mx, rec[1] = lv;
        }
    }
    // a wave's 64 results are channels of one (row, head)
#pragma unroll 1
    for (int n = 0; again >> n; ++n) {
        if (!(again >> n & 1)) continue;
        const int e = 64 * wu + 256 * n, k = R == 1 ? 0 : e / (group * DH), h = e / DH - k * group, ch0 = e % DH, ch = ch0 + lane;
        float m1, l1, o1, f[4], lv;
        bool any;
        attend_plain<DH, Q8, R>(a, r0 + k, k, g, g * group + h, ch0, list, ne, m1, l1, o1, any);
        if (nsplit == 1) {
            const float of = a.proj[int64_t(r0 + k) * a.proj_stride + int64_t(g * group + h) * 2 * DH + DH + ch];
            sparse_store<DH>(a, r0 + k, g * group + h, ch, o1, any && m1 == -INFINITY ? NAN : l1, of);
        } else {
            float* rec = record(h);
            const float mx = parts(slot_of(k, h), f, lv);
            if (lv * 0.f == 0.f) {  // the values alone: beside the total that is there
                rec[4 + ch] = kPOne * exp2_hw(m1 - mx) * o1;
            } else {  // a total of 1 beside m = -inf: keys, but none with a weight
                rec[4 + ch] = kPOne * o1;
                if (ch == 0) rec[0] = m1, rec[1] = any && m1 == -INFINITY ? 1.f : kPOne * l1;
            }
        }
    }
}

// a workgroup per (row, query head), a lane per channel: the ranges' results,
// their maxima and sums read once by a lane each
template <int DH>
__global__ __launch_bounds__(DH) void attn_sparse_combine_kernel(SparseAttnArgs a, int nsplit) {
    constexpr int kRec = DH + 4, kPass = 16;
    const int r = blockIdx.x / a.Hq, h = blockIdx.x % a.Hq, t = threadIdx.x;
    int seq;
    if (row_position(a.c, r, &seq) < 0) return;
    extern __shared__ float share[];  // [nsplit], a multiple of kPass: a range's share of the result, 0 behind
    __shared__ float part[2][DH / 64];
    const float* rec = a.work + (int64_t(r) * a.Hq + h) * nsplit * kRec;
    const int padded = (nsplit + kPass - 1) / kPass * kPass;
    auto over_waves = [&](float v, int k, auto f) {
        for (int off = 32; off > 0; off >>= 1) v = f(v, __shfl_xor(v, off));
        if ((t & 63) == 0) part[k][t >> 6] = v;
        __syncthreads();
        v = part[k][0];
#pragma unroll
        for (int w = 1; w < DH / 64; ++w) v = f(v, part[k][w]);
        return v;
    };
    const float gate = a.proj[int64_t(r) * a.proj_stride + int64_t(h) * 2 * DH + DH + t];
    float mx = -INFINITY;
    for (int s = t; s < nsplit; s += DH) mx = fmaxf(mx, rec[int64_t(s) * kRec]);
    mx = over_waves(mx, 0, [](float x, float y) { return fmaxf(x, y); });
    float l = 0.f;
    for (int s = t; s < padded; s += DH) {
        float f = 0.f;
        if (s < nsplit) {
            const float m = rec[int64_t(s) * kRec], ls = rec[int64_t(s) * kRec + 1];
            if (m != -INFINITY || ls != 0.f) f = exp2_hw(m - mx), l += f * ls;  // a range without keys has neither
        }
        share[s] = f;
    }
    l = over_waves(l, 1, [](float x, float y) { return x + y; });
    float o = 0.f;
    for (int s = 0; s < nsplit; s += kPass) {
        float v[kPass];
#pragma unroll
        for (int k = 0; k < kPass; ++k) v[k] = rec[int64_t(min(s + k, nsplit - 1)) * kRec + 4 + t];
#pragma unroll
        for (int k = 0; k < kPass; ++k) o += share[s + k] * v[k];
    }
    sparse_store<DH>(a, r, h, t, o, l, gate);
}

// Ranges of a row's list: about two workgroups per CU over all rows and heads (as many
// as fit; with four the sixteen Q8_0 sequences take 28 us instead of 24),
// whole pages, at least 32 key slots for each wave, at most 2048 list entries
// (16 KB of shared memory).
void sparse_plan(int64_t rows, int64_t Hkv, int64_t ps, int64_t top, int* per, int* nsplit) {
    const int64_t want = std::max<int64_t>(1, 512 / (rows * Hkv));
    const int64_t most = std::max<int64_t>(1, top * ps / 128);
    const int64_t n = std::max(std::min(std::min(want, most), top), (top + 2047) / 2048);
    *per = int((top + n - 1) / n);
    *nsplit = int((top + *per - 1) / *per);
}

}  // namespace

namespace {
template <int DH, int GP, int RT>
void select_rows(const SelectArgs& a, hipStream_t s) {
    const PagedRows& c = a.c;
    const unsigned tiles = unsigned((c.rows + RT - 1) / RT * c.Hkv), heads = unsigned(c.rows * c.Hkv);
    if (c.max_pages <= (RT == 1 ? 512 : 1024)) {
        hipLaunchKernelGGL((select_pages_kernel<DH, GP, RT>), dim3(tiles), dim3(kSelThreads<RT>), size_t(RT) * c.max_pages * 8, s, a);
        return;
    }
    // a workgroup's four waves take 64 pages each at a time; about four workgroups per CU
    const unsigned most = unsigned((c.max_pages + 255) / 256), ranges = std::min(most, std::max(1u, 1024 / tiles));
    hipLaunchKernelGGL((page_scores_kernel<DH, GP, RT>), dim3(tiles, ranges), dim3(256), 0, s, a);
    if (c.max_pages <= 2048)
        hipLaunchKernelGGL((choose_pages_kernel<256, 8>), dim3(heads), dim3(256), 0, s, a);
    else if (c.max_pages <= 4096)
        hipLaunchKernelGGL((choose_pages_kernel<512, 8>), dim3(heads), dim3(512), 0, s, a);
    else if (c.max_pages <= 16384)
        hipLaunchKernelGGL((choose_pages_kernel<1024, 16>), dim3(heads), dim3(1024), 0, s, a);
    else
        hipLaunchKernelGGL(choose_pages_long_kernel, dim3(heads), dim3(1024), 0, s, a);
}

// rows without row_seq belong to sequences of their own and share no page;
// others are taken in tiles
template <int DH, int GP>
void select_group(const SelectArgs& a, hipStream_t s) {
    constexpr int RT = GP == 8 ? 2 : 4;
    if (a.c.row_seq && a.c.rows > 1)
        select_rows<DH, GP, RT>(a, s);
    else
        select_rows<DH, GP, 1>(a, s);
}

template <int DH>
void select_heads(const SelectArgs& a, hipStream_t s) {
    switch (a.Hq / a.c.Hkv) {
        case 1: select_group<DH, 1>(a, s); break;
        case 2: select_group<DH, 2>(a, s); break;
        case 3:
        case 4: select_group<DH, 4>(a, s); break;
        default: select_group<DH, 8>(a, s); break;
    }
}
}  // namespace

void launch_attn_select(const SelectArgs& a, hipStream_t s) {
    if (a.c.Dh == 256)
        select_heads<256>(a, s);
    else
        select_heads<128>(a, s);
}

// Room for any call of up to `rows` rows: rows * Hkv * ranges is at most 512 where
// the plan takes several ranges to fill the chip, twice rows * Hkv where it
// does for the list's length.
int64_t attn_sparse_work_bytes(int64_t rows, int64_t Hq, int64_t Hkv, int64_t Dh, int64_t page_size, int64_t top) {
    const int64_t most = std::min(top, std::max<int64_t>(1, top * page_size / 128));
    const int64_t parts = std::max(most > 1 ? std::min<int64_t>(512, rows * Hkv * most) : 0, top > 2048 ? 2 * rows * Hkv : 0);
    return parts * (Hq / Hkv) * (Dh + 4) * 4;
}

namespace {
template <int DH, bool Q8, int GQ, int R, int GP>
void sparse_rows(const SparseAttnArgs& a, int per, int nsplit, hipStream_t s) {
    const int64_t tiles = (a.c.rows + R - 1) / R;
    hipLaunchKernelGGL((attn_sparse_kernel<DH, Q8, GQ, R, GP>), dim3(unsigned(tiles * a.c.Hkv * nsplit)), dim3(256), size_t(R > 1 ? R * a.top : per) * sizeof(ListEntry<R>),
                       s, a, per, nsplit);
}

// Chunks with enough rows to fill the chip take several rows a workgroup, so
// that a page which neighbouring rows select is read once for them: lists of 16
// pages of 32 query heads break even at 128 rows (34 us; 64 rows 29 against 20 us
// alone), lists of 128 pages take 137 against 180 us there and 433 against 600 us
// at 500 rows. 512 list entries a workgroup are what its scratch holds. Groups of
// more than four heads fill the columns by themselves, and Q8_0 pages, whose
// values and weights cost more instructions than their reads time, gain nothing.
bool sparse_shares(const SparseAttnArgs& a) {
    const int group = a.Hq / a.c.Hkv;
    return a.c.row_seq && !a.c.q8 && group <= 4 && a.top <= (group <= 2 ? 128 : 256) && int64_t(a.c.rows) * a.c.Hkv >= 1024;
}
}  // namespace

void launch_attn_sparse(const SparseAttnArgs& a, hipStream_t s) {
    int per, nsplit;
    sparse_plan(a.c.rows, a.c.Hkv, a.c.page_size, a.top, &per, &nsplit);
    const int group = a.Hq / a.c.Hkv;
    if (sparse_shares(a)) {
        if (a.c.Dh == 256)
            group <= 2 ? sparse_rows<256, false, 1, 4, 2>(a, per, 1, s) : sparse_rows<256, false, 1, 2, 4>(a, per, 1, s);
        else
            group <= 2 ? sparse_rows<128, false, 1, 4, 2>(a, per, 1, s) : sparse_rows<128, false, 1, 2, 4>(a, per, 1, s);
        return;
    }
    if (a.c.Dh == 256)
        sparse_rows<256, false, 1, 1, 8>(a, per, nsplit, s);
    else if (!a.c.q8)
        sparse_rows<128, false, 1, 1, 8>(a, per, nsplit, s);
    else if (group <= 4)
        sparse_rows<128, true, 1, 1, 4>(a, per, nsplit, s);
    else
        sparse_rows<128, true, 2, 1, 8>(a, per, nsplit, s);
    if (nsplit == 1) return;
    const dim3 heads(unsigned(a.c.rows * a.Hq));
    if (a.c.Dh == 256)
        hipLaunchKernelGGL(attn_sparse_combine_kernel<256>, heads, dim3(256), size_t(nsplit + 15) / 16 * 64, s, a, nsplit);
    else
        hipLaunchKernelGGL(attn_sparse_combine_kernel<128>, heads, dim3(128), size_t(nsplit + 15) / 16 * 64, s, a, nsplit);
}

}  // namespace hero
