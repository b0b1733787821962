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
// A row is cut into ranges, one for each wave: the running M, c, R and the
// entropy's sum T lane by lane, and the range's best keys as a sorted list, one a lane. A
// key is the logit in an order-preserving form, then the id's complement, so
// that equal logits rank by ascending id and no two keys are equal. A second launch, a wave
// per row, joins the ranges.
#include "hero/device.hpp"
#include "hero/kernels.hpp"

namespace hero {

namespace {

constexpr float kLog2eF = 1.4426950408889634f, kLn2F = 0.6931471805599453f, kLowestF = -3.402823466e38f;
constexpr int kBatch = 16;  // logits a lane takes at a time

struct RangeSum {  // what a range leaves behind, before its keys
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
__device__ __forceinline__ uint64_t key_of(float x, uint32_t id) { return uint64_t(order_of(x)) << 32 | (0xFFFFFFFFu - id); }

__device__ __forceinline__ uint64_t lane_key(uint64_t v, int lane) {
    return uint64_t(uint32_t(__builtin_amdgcn_readlane(int(v >> 32), lane))) << 32 | uint32_t(__builtin_amdgcn_readlane(int(v), lane));
}
__device__ __forceinline__ uint64_t lane_before(uint64_t v) {  // the value of lane - 1 (wave_shr:1)
    return uint64_t(uint32_t(__builtin_amdgcn_update_dpp(0, int(v >> 32), 0x138, 0xF, 0xF, false))) << 32 |
           uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x138, 0xF, 0xF, false));
}

// The best keys so far, descending, one a lane; `least` the top-th of them (0: not that many yet)
struct TopList {
    uint64_t mine = 0, least = 0;
    // up to kBatch keys a lane (0: none)
    __device__ __forceinline__ void add(const uint64_t (&key)[kBatch], int top, int lane) {
        uint64_t best = key[0];
#pragma unroll
        for (int j = 1; j < kBatch; ++j) best = key[j] > best ? key[j] : best;
        uint64_t bar = least;
        if (__popcll(__ballot(best > bar)) > top) {
            // more lanes with a better key than there are places: the top-th largest of the
            // lanes' best, to 24 bits, is a bar that the keys to take all reach
            uint32_t at = 0;
            const uint32_t hi = uint32_t(best >> 32);
#pragma unroll
            for (int bit = 31; bit >= 8; --bit)
                if (__popcll(__ballot(hi >= (at | 1u << bit))) >= top) at |= 1u << bit;
            const uint64_t from = uint64_t(at) << 32;
            if (from > bar) bar = from - 1;
        }
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            for (uint64_t hits = __ballot(key[j] > bar); hits; hits &= hits - 1) {
                const uint64_t k = lane_key(key[j], __ffsll((unsigned long long)hits) - 1);
                if (k <= least) continue;
                const int place = __popcll(__ballot(mine > k));
                const uint64_t before = lane_before(mine);
                mine = lane < place ? mine : lane == place ? k : before;
                least = lane_key(mine, top - 1);
            }
        }
    }
};

// the larger of two running maxima takes the other's sums over
__device__ __forceinline__ void join(RangeSum& a, const RangeSum& b, float k2) {
    const float m = fmaxf(a.m, b.m);
    // (m - m: 0, also for equal infinities)
    const float da = a.m == m ? 0.f : (a.m - m) * k2, db = b.m == m ? 0.f : (b.m - m) * k2;
    const float fa = __builtin_amdgcn_exp2f(da), fb = __builtin_amdgcn_exp2f(db);
    const float sa = a.m == m ? a.r : (a.r + a.c) * fa, sb = b.m == m ? b.r : (b.r + b.c) * fb;
    const float ta = a.m == m ? a.t : fa * a.t + fmaxf(da, -200.f) * sa, tb = b.m == m ? b.t : fb * b.t + fmaxf(db, -200.f) * sb;
    a.c = (a.m == m ? a.c : 0.f) + (b.m == m ? b.c : 0.f);
    a.m = m;
    a.r = sa + sb;
    a.t = ta + tb;
}

struct LogprobsWork {
    RangeSum* sums;   // [m][ranges]
    uint64_t* keys;   // [m][ranges][top]
};

// a wave per range: whole batches of 64 kBatch logits
template <bool TOP>
__global__ __launch_bounds__(256) void logprobs_range_kernel(LogprobsArgs a, LogprobsWork w, int ranges, int per) {
    const int lane = threadIdx.x & 63;
    const int64_t item = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (item >= a.m * ranges) return;
    const int64_t row = item / ranges;
    if (a.targets && (a.targets[row] < 0 || a.targets[row] >= a.v)) return;
    const int64_t first = (item % ranges) * per * int64_t(64 * kBatch), last = min(a.v, first + int64_t(per) * 64 * kBatch);
    const float* x = a.logits + row * a.stride;
    const float k2 = kLog2eF / a.temp;
    RangeSum s{kLowestF, 0.f, 0.f, 0.f};
    TopList list;
    for (int64_t at = first; at < last; at += 64 * kBatch) {
        float v[kBatch];
        const int64_t mine = at + 4 * lane;
        if (at + 64 * kBatch <= last) {
#pragma unroll
            for (int k = 0; k < kBatch / 4; ++k) __builtin_memcpy(v + 4 * k, x + mine + 256 * k, 16);
        } else {
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {
                const int64_t i = mine + 256 * (j / 4) + j % 4;
                v[j] = x[min(i, a.v - 1)];
                if (i >= last) v[j] = -INFINITY;
            }
        }
        float best = v[0];
#pragma unroll
        for (int j = 1; j < kBatch; ++j) best = fmaxf(best, v[j]);
        if (best > s.m) {
            RangeSum next{best, 0.f, 0.f, 0.f};
            join(s, next, k2);
        }
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const float d = (v[j] - s.m) * k2;
            const bool top = v[j] == s.m;
            const float e = top ? 0.f : __builtin_amdgcn_exp2f(d);
            s.c += top ? 1.f : 0.f;
            s.r += e;
            s.t += e * fmaxf(d, -200.f);
        }
        if constexpr (TOP) {
            if (list.least == 0 || __ballot(best >= logit_of(uint32_t(list.least >> 32)))) {
                uint64_t key[kBatch];
#pragma unroll
                for (int j = 0; j < kBatch; ++j) {
                    const int64_t i = mine + 256 * (j / 4) + j % 4;
                    key[j] = i < last ? key_of(v[j], uint32_t(i)) : 0;
                }
                list.add(key, a.top, lane);
            }
        }
    }
    for (int off = 32; off > 0; off >>= 1) {
        const RangeSum o{__shfl_xor(s.m, off), __shfl_xor(s.c, off), __shfl_xor(s.r, off), __shfl_xor(s.t, off)};
        join(s, o, k2);
    }
    if (lane == 0) w.sums[item] = s;
    if (TOP && lane < a.top) w.keys[item * a.top + lane] = list.mine;
}

// a wave per row
__global__ __launch_bounds__(64) void logprobs_join_kernel(LogprobsArgs a, LogprobsWork w, int ranges) {
    const int64_t row = blockIdx.x;
    const int lane = threadIdx.x;
    const int target = a.targets ? a.targets[row] : 0;
    if (target < 0 || target >= a.v) return;
    const float* x = a.logits + row * a.stride;
    const float own = a.logprob ? x[target] : 0.f, k2 = kLog2eF / a.temp;
    RangeSum s{kLowestF, 0.f, 0.f, 0.f};
    for (int i = lane; i < ranges; i += 64) join(s, w.sums[row * ranges + i], k2);
    for (int off = 32; off > 0; off >>= 1) {
        const RangeSum o{__shfl_xor(s.m, off), __shfl_xor(s.c, off), __shfl_xor(s.r, off), __shfl_xor(s.t, off)};
        join(s, o, k2);
    }
    if (s.m == INFINITY) s.r = __uint_as_float(0x7FC00000u);
    const float log_sum = logf(s.c) + log1pf(s.r / s.c);
    if (lane == 0) {
        if (a.logprob) a.logprob[row] = (own - s.m) / a.temp - log_sum;
        if (a.entropy) a.entropy[row] = log_sum - kLn2F * s.t / (s.c + s.r);
    }
    if (a.top == 0) return;
    TopList list;
    const int n = ranges * a.top;
    for (int at = 0; at < n; at += 64 * kBatch) {
        uint64_t key[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const int i = at + 64 * j + lane;
            key[j] = i < n ? w.keys[row * n + i] : 0;
        }
        list.add(key, a.top, lane);
    }
    if (lane < a.top) {
        a.top_ids[row * a.top + lane] = int32_t(0xFFFFFFFFu - uint32_t(list.mine));
        a.top_logprobs[row * a.top + lane] = (logit_of(uint32_t(list.mine >> 32)) - s.m) / a.temp - log_sum;
    }
}

// Ranges of a row: about 2048 waves over all rows, at least one batch each.
void logprobs_plan(int64_t m, int64_t v, int* ranges, int* per) {
    const int64_t batches = (v + 64 * kBatch - 1) / (64 * kBatch), want = std::max<int64_t>(1, std::min(batches, 4096 / m));
    *per = int((batches + want - 1) / want);
    *ranges = int((batches + *per - 1) / *per);
}

}  // namespace

int64_t logprobs_work_bytes(int64_t m, int64_t v, int top) {
    // m ranges(m) is at most 4096 or m
    const int64_t batches = (v + 64 * kBatch - 1) / (64 * kBatch), parts = std::max(m, std::min<int64_t>(4096, m * batches));
    return parts * int64_t(sizeof(RangeSum) + 8 * top);
}

void launch_logprobs(const LogprobsArgs& a, hipStream_t s) {
    int ranges, per;
    logprobs_plan(a.m, a.v, &ranges, &per);
    LogprobsWork w;
    w.sums = static_cast<RangeSum*>(a.work);
    w.keys = reinterpret_cast<uint64_t*>(w.sums + a.m * ranges);
    const dim3 grid(unsigned((a.m * ranges + 3) / 4));
    if (a.top)
        hipLaunchKernelGGL(logprobs_range_kernel<true>, grid, dim3(256), 0, s, a, w, ranges, per);
    else
        hipLaunchKernelGGL(logprobs_range_kernel<false>, grid, dim3(256), 0, s, a, w, ranges, per);
    hipLaunchKernelGGL(logprobs_join_kernel, dim3(unsigned(a.m)), dim3(64), 0, s, a, w, ranges);
}

}  // namespace hero
