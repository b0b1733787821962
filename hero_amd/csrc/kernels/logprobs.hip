// logprobs.hip -- log probabilities of given tokens, the entropy of their
// distributions and the most likely alternatives, in one pass over the logits.
//
// With z = x / temp and M the largest logit of a row, c of them and R = sum of
// exp(z - M / temp) over all others,
//   log sum exp(z) = M / temp + log c + log1p(R / c)
//   entropy        = log c + log1p(R / c) - sum (z - M / temp) exp(z - M / temp) / (c + R).
// Keeping the largest out of R leaves the small differences that a nearly certain
// token's log probability and entropy consist of; in a sum 1 + R they would drown.
//
// A row is cut into ranges, one for each wave: the running M, c, R and the entropy's sum T, and
// for the alternatives nothing but the largest of every 64 logits. A second launch, a workgroup per row, joins the
// ranges, takes the n-th largest of 256 groups of these maxima for a bar that n logits reach at least, and
// reads the few blocks again whose largest reaches it. (Sorted lists that each wave keeps along the
// way: one row of 151936 with twenty alternatives 16.2 us instead of 11.3, 1000 rows 219 instead of 116.)
//
// What bounds it: many rows, the memory: 1000 rows of 151936 at 5.7 TB/s in 107 us, and 9 us for the joins. Few rows, the
// two launches: of one row's 11.3 us the first takes 4.1 (3.6 with one logit per lane), the second 6, each round
// to memory and back about 1 us of it. Where fewer logits than alternatives are above -inf, the bar is -inf and
// the second launch reads the row again: one row of 151936 with ten such logits and twenty alternatives 75 us, 1000 rows 339.
#include "hero/device.hpp"
#include "hero/kernels.hpp"

#include <type_traits>

namespace hero {

namespace {

constexpr float kLog2eF = 1.4426950408889634f, kLn2F = 0.6931471805599453f, kLowestF = -3.402823466e38f;
constexpr int kBatch = 16;  // logits a lane takes at a time

struct RangeSum {  // what a range leaves behind
    float m, c, r, t;
};

// larger logit, larger value; -0 as 0; NaN below everything
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);
    return x == x ? (u & 0x80000000u ? ~u : u | 0x80000000u) : 0u;
}
__device__ __forceinline__ float logit_of(uint32_t order) {
    return order == 0u ? __uint_as_float(0x7FC00000u) : __uint_as_float(order & 0x80000000u ? order & 0x7FFFFFFFu : ~order);
}

// Differences of logits over temp. From temp 1 on those of their halves, and twice the quotient: what a difference loses by
// that is below 2^-149, and two logits may be further apart than fp32 reaches where the quotient is not. Below, a
// difference that does not fit has no quotient that does.
struct Scale {
    float part, back, temp, k2;  // 1 or 1/2, its reciprocal; 1 / part / temp in units of log2
    __device__ __forceinline__ explicit Scale(float t) : part(t >= 1.f ? 0.5f : 1.f), back(t >= 1.f ? 2.f : 1.f), temp(t), k2(kLog2eF * back / t) {}
    __device__ __forceinline__ float log2_of(float x, float m_part) const { return __builtin_fmaf(x, part, -m_part) * k2; }  // (m_part: m times part)
    __device__ __forceinline__ float of(float x, float m) const { return __builtin_fmaf(x, part, -(m * part)) / temp * back; }
};

// the larger of two running maxima takes the other's sums over
__device__ __forceinline__ void join(RangeSum& a, const RangeSum& b, const Scale& scale) {
    const float m = fmaxf(a.m, b.m), m_part = m * scale.part;
    // (m - m: 0, also for equal infinities)
    const float da = a.m == m ? 0.f : scale.log2_of(a.m, m_part), db = b.m == m ? 0.f : scale.log2_of(b.m, m_part);
    const float fa = __builtin_amdgcn_exp2f(da), fb = __builtin_amdgcn_exp2f(db);
    const float sa = a.m == m ? a.r : (a.r + a.c) * fa, sb = b.m == m ? b.r : (b.r + b.c) * fb;
    const float ta = a.m == m ? a.t : fa * a.t + fmaxf(da, -200.f) * sa, tb = b.m == m ? b.t : fb * b.t + fmaxf(db, -200.f) * sb;
    a.c = (a.m == m ? a.c : 0.f) + (b.m == m ? b.c : 0.f);
    a.m = m;
    a.r = sa + sb;
    a.t = ta + tb;
}

// over the wave's lanes, in every lane
template <class F>
__device__ __forceinline__ float over_lanes(float v, F f) {
    auto with = [](float x, auto ctrl) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value, 0xF, 0xF, true)); };
    v = f(v, with(v, std::integral_constant<int, 0xB1>{}));   // quad_perm [1,0,3,2]
    v = f(v, with(v, std::integral_constant<int, 0x4E>{}));   // quad_perm [2,3,0,1]
    v = f(v, with(v, std::integral_constant<int, 0x141>{}));  // row_half_mirror
    v = f(v, with(v, std::integral_constant<int, 0x140>{}));  // row_mirror
    auto at = [&](int lane) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane)); };
    return f(f(at(0), at(16)), f(at(32), at(48)));
}
__device__ __forceinline__ void join_lanes(RangeSum& s, const Scale& scale) {
    const RangeSum all{over_lanes(s.m, [](float x, float y) { return fmaxf(x, y); }), 0.f, 0.f, 0.f};
    join(s, all, scale);
    auto sum = [](float x, float y) { return x + y; };
    s = {all.m, over_lanes(s.c, sum), over_lanes(s.r, sum), over_lanes(s.t, sum)};
}

// Of every 64 kBatch logits sixteen blocks, one of each four lanes: sixteen neighbours of every 256.
constexpr int kBlocks = 16, kKept = 64;  // blocks of a batch; batches whose blocks' maxima a wave keeps before it stores them
__device__ __forceinline__ int block_id(int block, int k, int i) { return block / kBlocks * 64 * kBatch + 256 * k + 16 * (block % kBlocks) + i; }
struct LogprobsWork {
    RangeSum* sums;      // [m][ranges]
    uint32_t* maxima;    // [m][blocks], as order_of
};

// A wave per range: whole batches of 64 kBatch logits, one ahead. Lane l brings logits 4 l .. 4 l + 3 of each
// 256; the row's last four stand in for ones past its end, and count once.
template <bool TOP>
__global__ __launch_bounds__(256) void logprobs_range_kernel(LogprobsArgs a, LogprobsWork w, int ranges, int per, int blocks) {
    constexpr int kStep = 64 * kBatch;
    const int lane = threadIdx.x & 63;
    const int64_t item = int64_t(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (item >= a.m * ranges) return;
    const int64_t row = item / ranges;
    const int first = int(item % ranges) * per * kStep, last = int(min(a.v, int64_t(first) + int64_t(per) * kStep)), v_end = int(a.v);
    const float* x = a.logits + row * a.stride;
    const Scale scale(a.temp);
    RangeSum s{kLowestF, 0.f, 0.f, 0.f};
    float m_part = kLowestF * scale.part;
    float ahead[kBatch];
    // Stores would hold up the wait for the loads behind them: 1000 rows of 151936 take 103 us without the maxima, 118 with a store for each
    // batch or each four.
    __shared__ uint32_t kept[TOP ? 4 : 1][TOP ? kKept * kBlocks : 4];
    uint32_t* maxima = kept[TOP ? threadIdx.x >> 6 : 0];
    auto store = [&](int batch, int n) {  // n batches, from the range's batch on
        uint32_t* to = w.maxima + row * blocks + (first / kStep + batch) * kBlocks;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        for (int i = 4 * lane; i < n * kBlocks; i += 256) __builtin_memcpy(to + i, maxima + i, 16);
    };
#pragma unroll 1
    for (int at = first - kStep; at < last; at += kStep) {
        float v[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) v[j] = ahead[j];
        if (const int next = at + kStep; next < last) {
            if (v_end >= 4) {
#pragma unroll
                for (int k = 0; k < kBatch / 4; ++k) __builtin_memcpy(ahead + 4 * k, x + min(next + 4 * lane + 256 * k, v_end - 4), 16);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) ahead[j] = x[min(j, v_end - 1)];
            }
        }
        if (at < first) {  // the first batch is on its way
            if (a.targets && (a.targets[row] < 0 || a.targets[row] >= a.v)) return;
            continue;
        }
        const float missing = TOP ? __uint_as_float(0x7FC00000u) : -INFINITY;  // (NaN: below -inf among the maxima)
        bool partial = false;
        if (at + kStep > last) {
            partial = true;
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {
                const int from = at + 4 * lane + 256 * (j / 4), i = v_end >= 4 ? min(from, v_end - 4) + j % 4 : j < 4 ? from + j : last;
                if (i < from || i >= last) v[j] = missing;
            }
        }
        float best = v[0];
#pragma unroll
        for (int j = 1; j < kBatch; ++j) best = fmaxf(best, v[j]);
        if constexpr (TOP) {
            auto with = [](float x, auto ctrl) { return fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value, 0xF, 0xF, true))); };
            const float four = with(with(best, std::integral_constant<int, 0xB1>{}), std::integral_constant<int, 0x4E>{});
            const int batch = (at - first) / kStep;
            maxima[batch % kKept * kBlocks + lane / 4] = order_of(four);
            if (batch % kKept == kKept - 1) store(batch - (kKept - 1), kKept);
            if (partial) {
#pragma unroll
                for (int j = 0; j < kBatch; ++j) {
                    const int from = at + 4 * lane + 256 * (j / 4), i = v_end >= 4 ? min(from, v_end - 4) + j % 4 : j < 4 ? from + j : last;
                    if (i < from || i >= last) v[j] = -INFINITY;
                }
            }
        }
        if (__ballot(best > s.m)) {  // one maximum for the wave: one of 64 would change in most batches
            const RangeSum next{over_lanes(best, [](float x, float y) { return fmaxf(x, y); }), 0.f, 0.f, 0.f};
            join(s, next, scale);
            m_part = s.m * scale.part;
        }
        // a batch's own sums first: a row of 262144 adds 256 of them and not 4096 terms, whose roundings go the same way where the
        // terms are equal (5e-5 of the sum, so 4e-6)
        float r = 0.f, t = 0.f;
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const float d = scale.log2_of(v[j], m_part);
            const bool top = v[j] == s.m;
            const float e = top ? 0.f : __builtin_amdgcn_exp2f(d);
            s.c += top ? 1.f : 0.f;
            r += e;
            t += e * fmaxf(d, -200.f);
        }
        s.r += r;
        s.t += t;
    }
    if constexpr (TOP) {
        const int batches = (last - first + kStep - 1) / kStep;
        store(batches - batches % kKept, batches % kKept);
    }
    join_lanes(s, scale);
    if (lane == 0) w.sums[item] = s;
}

// A workgroup per row. The last wave joins the sums; the others look for the alternatives.
constexpr int kJoinThreads = 512, kGathered = 4096, kListed = 256;
__global__ __launch_bounds__(kJoinThreads) void logprobs_join_kernel(LogprobsArgs a, LogprobsWork w, int ranges, int blocks) {
    const int64_t row = int64_t(blockIdx.y) * gridDim.x + blockIdx.x;
    if (row >= a.m) return;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, v_end = int(a.v);
    const int target = a.targets ? a.targets[row] : 0;
    if (target < 0 || target >= a.v) return;
    __shared__ uint64_t gathered[kGathered];
    __shared__ uint32_t groups[kJoinThreads], listed[kListed], bar, count, keys;
    __shared__ float of_row[2];  // the largest logit and the logarithm of the sum
    const float* x = a.logits + row * a.stride;
    const float own = a.logprob ? x[target] : 0.f;
    const Scale scale(a.temp);
    const uint32_t* maxima = w.maxima + row * blocks;
    const bool last = wave == kJoinThreads / 64 - 1;
    auto maximum = [&](int i) { return i < blocks ? maxima[i] : 0u; };
    uint32_t held[8];
    if (a.top) {
#pragma unroll
        for (int j = 0; j < 8; ++j) held[j] = maximum(t + j * kJoinThreads);
        uint32_t most = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) most = max(most, held[j]);
        for (int i = t + 8 * kJoinThreads; i < blocks; i += kJoinThreads) most = max(most, maxima[i]);
        groups[t] = most;
    }
    if (t == 0) count = 0, keys = 0;
    __syncthreads();
    if (last) {
        RangeSum s{kLowestF, 0.f, 0.f, 0.f};
        for (int i = lane; i < ranges; i += 64) join(s, w.sums[row * ranges + i], scale);
        join_lanes(s, scale);
        if (s.m == INFINITY) s.r = __uint_as_float(0x7FC00000u);
        const float log_sum = logf(s.c) + log1pf(s.r / s.c);
        if (lane == 0) {
            of_row[0] = s.m, of_row[1] = log_sum;
            if (a.logprob) a.logprob[row] = scale.of(own, s.m) - log_sum;
            if (a.entropy) a.entropy[row] = log_sum - kLn2F * s.t / (s.c + s.r);
        }
    }
    if (a.top == 0) return;
    // The smallest of the largest of 256 groups' maxima, top of them and those that share 20 bits with the last
    // (0 where fewer hold anything).
    if (wave == 0) {
        uint32_t of[4], found = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) of[j] = max(groups[lane + 64 * j], groups[lane + 64 * j + 256]);
#pragma unroll
        for (int bit = 31; bit >= 12; --bit) {
            int n = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) n += __popcll(__ballot(of[j] >= (found | 1u << bit)));
            if (n >= a.top) found |= 1u << bit;
        }
        uint32_t least = ~0u;
#pragma unroll
        for (int j = 0; j < 4; ++j) least = min(least, of[j] >= found ? of[j] : ~0u);
        for (int off = 32; off > 0; off >>= 1) least = min(least, uint32_t(__shfl_xor(int(least), off)));
        if (lane == 0) bar = least;
    }
    __syncthreads();
    auto list = [&](uint32_t m, int i) {
        if (i < blocks && m >= bar)
            if (const uint32_t at = atomicAdd(&count, 1u); at < kListed) listed[at] = i;
    };
#pragma unroll
    for (int j = 0; j < 8; ++j) list(held[j], t + j * kJoinThreads);
    for (int i = t + 8 * kJoinThreads; i < blocks; i += kJoinThreads) list(maxima[i], i);
    __syncthreads();
    // Blocks that reach the bar, each by sixteen lanes: their logits that do. (The order of the keys differs from run to
    // run, their places do not: no two are equal.) Where too many tie at the bar, only those above it; where
    // these are too many, those above the exact bar, which are fewer than top.
    const bool few = count <= kListed;
    const int candidates = few ? int(count) : blocks;
    auto each = [&](auto f) {
        for (int i = t / 16; i < candidates; i += kJoinThreads / 16) {
            const int block = few ? int(listed[i]) : i;
            if (maxima[block] < bar) continue;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (const int id = block_id(block, j, t & 15); id < v_end) f(order_of(x[id]), id);
        }
    };
    bool above = !few;
#pragma unroll 1
    for (bool exact = false;;) {
        each([&](uint32_t order, int id) {
            if (order >= bar && !(above && order == bar))
                if (const uint32_t at = atomicAdd(&keys, 1u); at < kGathered) gathered[at] = uint64_t(order) << 32 | (0xFFFFFFFFu - uint32_t(id));
        });
        __syncthreads();
        if (keys <= kGathered || exact) break;
        uint32_t known = 0, left = a.top;  // the bar's upper bytes; how many of the logits that share them it is
        if (above) {
            exact = true;
#pragma unroll 1
            for (int shift = 24; shift >= 0; shift -= 8) {
                __syncthreads();
                if (t < 256) groups[t] = 0;
                __syncthreads();
                each([&](uint32_t order, int) {
                    if (order >= bar && uint64_t(order) >> (shift + 8) == uint64_t(known) >> (shift + 8)) atomicAdd(&groups[order >> shift & 255], 1u);
                });
                __syncthreads();
                int byte = 255;
                for (; byte > 0 && groups[byte] < left; --byte) left -= groups[byte];
                known |= uint32_t(byte) << shift;
            }
        }
        above = true;
        __syncthreads();
        if (t == 0) {
            keys = 0;
            if (exact) bar = known;
        }
        __syncthreads();
    }
    if (above && keys < uint32_t(a.top)) {
        // the lowest ids among the equal ones
        __syncthreads();
        if (wave == 0) {
            uint32_t have = keys;
            for (int i = 0; i < blocks && have < uint32_t(a.top); i += 64) {
                const uint64_t reach = __ballot(i + lane < blocks && maxima[min(i + lane, blocks - 1)] >= bar);
                for (int j = 0; j < 64; ++j) {  // 64 ids of a batch, in their order
                    const int id = (i / kBlocks * kBatch + j) * 64 + lane;
                    if ((reach >> (j / kBatch * kBlocks) & ((1u << kBlocks) - 1)) == 0 || have >= uint32_t(a.top)) continue;
                    const uint64_t equal = __ballot(id < v_end && order_of(x[min(id, v_end - 1)]) == bar);
                    const uint32_t at = have + __builtin_amdgcn_mbcnt_hi(uint32_t(equal >> 32), __builtin_amdgcn_mbcnt_lo(uint32_t(equal), 0));
                    if ((equal >> lane & 1) && at < uint32_t(a.top)) gathered[at] = uint64_t(bar) << 32 | (0xFFFFFFFFu - uint32_t(id));
                    have += __popcll(equal);
                }
            }
            if (lane == 0) keys = min(have, uint32_t(a.top));
        }
        __syncthreads();
    }
    const int found = int(keys);
    for (int i = t; i < found; i += kJoinThreads) {
        const uint64_t k = gathered[i];
        int place = 0;
#pragma unroll 4
        for (int j = 0; j < found; ++j) place += gathered[j] > k;
        if (place >= a.top) continue;
        a.top_ids[row * a.top + place] = int32_t(0xFFFFFFFFu - uint32_t(k));
        a.top_logprobs[row * a.top + place] = scale.of(logit_of(uint32_t(k >> 32)), of_row[0]) - of_row[1];
    }
}

// Ranges of a row: about 2048 waves over all rows, at least one batch each (4096 and 8192 waves: 16 rows of 262144 and 1000
// rows of 151936 take 2 to 6 % longer).
constexpr int64_t kWaves = 2048;
void logprobs_plan(int64_t m, int64_t v, int* ranges, int* per) {
    const int64_t batches = (v + 64 * kBatch - 1) / (64 * kBatch), want = std::max<int64_t>(1, std::min(batches, kWaves / m));
    *per = int((batches + want - 1) / want);
    *ranges = int((batches + *per - 1) / *per);
}

}  // namespace

namespace {
int64_t blocks_of(int64_t v) { return (v + 64 * kBatch - 1) / (64 * kBatch) * kBlocks; }
}  // namespace

int64_t logprobs_work_bytes(int64_t m, int64_t v, int top) {
    // m ranges(m) is at most kWaves or m
    const int64_t batches = (v + 64 * kBatch - 1) / (64 * kBatch), parts = std::max(m, std::min(kWaves, m * batches));
    return parts * int64_t(sizeof(RangeSum)) + (top ? m * blocks_of(v) * 4 : 0);
}

void launch_logprobs(const LogprobsArgs& a, hipStream_t s) {
    int ranges, per;
    logprobs_plan(a.m, a.v, &ranges, &per);
    const int blocks = int(blocks_of(a.v));
    LogprobsWork w;
    w.sums = static_cast<RangeSum*>(a.work);
    w.maxima = reinterpret_cast<uint32_t*>(w.sums + a.m * ranges);
    const dim3 grid(unsigned((a.m * ranges + 3) / 4));
    if (a.top)
        hipLaunchKernelGGL(logprobs_range_kernel<true>, grid, dim3(256), 0, s, a, w, ranges, per, blocks);
    else
        hipLaunchKernelGGL(logprobs_range_kernel<false>, grid, dim3(256), 0, s, a, w, ranges, per, blocks);
    const unsigned wide = unsigned(std::min<int64_t>(a.m, 1 << 16));  // (a dimension has less than 2^32 threads)
    hipLaunchKernelGGL(logprobs_join_kernel, dim3(wide, unsigned((a.m + wide - 1) / wide)), dim3(kJoinThreads), 0, s, a, w, ranges, blocks);
}

}  // namespace hero
