// A router's logits to expert numbers and scores: what the routed layers take.
//
// A warp a row, lane l holding the experts l, l + 32, .. in registers. The choice is topk rounds of "the largest key, the lowest number
// among equals": keys are the picks' bit patterns made to order as whole numbers, so a round is one or three warp reductions and
// a look through one lane's values. Without bias or groups the pick is the logit itself (both scorings rise with it); with them it is
// score + bias in 64 bits, where two sums that differ in the last bits of 32 must still order as their exact values do. Bound by
// the logits' bytes on long prompts (4 bytes an expert and row), by latency on decode rows.
#include "t3_fp8.cuh"
#include "t3_fp8.h"
#include "t3_internal.h"

namespace t3 {
namespace {

constexpr uint32_t kWarps = 4;
constexpr uint32_t kFull = 0xFFFFFFFFu;

// Keys of one warp-wide order: 0 taken, 1 removed (a logit at or below its type's lowest number), then the numbers, NaN last
__device__ __forceinline__ uint32_t key_of(float v) {
    if (isnan(v)) return 0xFFFFFFFFu;
    if (v == 0.0f) v = 0.0f;  // -0 and 0 are equal
    const uint32_t b = __float_as_uint(v);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t key_of(double v) {
    if (isnan(v)) return ~0ull;
    if (v == 0.0) v = 0.0;
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    return b >> 63 ? ~b : b | 0x8000000000000000ull;
}
__device__ __forceinline__ uint32_t warp_max(uint32_t k) { return __reduce_max_sync(kFull, k); }
__device__ __forceinline__ uint64_t warp_max(uint64_t k) {
    const uint32_t hi = __reduce_max_sync(kFull, (uint32_t)(k >> 32));
    return (uint64_t)hi << 32 | __reduce_max_sync(kFull, (uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
}

__device__ __forceinline__ bool removed(float v, int dt) {
    return v <= (dt == kF16 ? -65504.0f : dt == kBf16 ? __uint_as_float(0xFF7F0000u) : __uint_as_float(0xFF7FFFFFu));
}

// PER: experts a lane; WIDE: picks of 64 bits (bias or groups)
template <uint32_t PER, bool WIDE>
__global__ void __launch_bounds__(kWarps * 32u) route_rows(const RouteArgs a) {
    using Key = typename std::conditional<WIDE, uint64_t, uint32_t>::type;
    extern __shared__ double picks[];  // WIDE, groups: [warps][experts]
    pdl_trigger();
    pdl_wait();
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const size_t row = (size_t)blockIdx.x * kWarps + warp;
    if (row >= a.rows) return;
    const size_t at = row * a.experts;

    float v[PER];
    uint32_t out = 0;  // a bit for each removed expert of the lane
    float top = -INFINITY;
    bool any = false;
#pragma unroll
    for (uint32_t j = 0; j < PER; ++j) {
        const uint32_t e = lane + 32u * j;
        v[j] = e < a.experts ? load_act(a.logits, a.dt, at + e) : -INFINITY;
        if (removed(v[j], a.dt)) out |= 1u << j;
        else any = true, top = fmaxf(top, v[j]);
    }
    static_assert(PER <= 32u, "a bit an expert");
    any = __any_sync(kFull, any);
    for (uint32_t d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, d));
    float sum = 0.0f;
    if (a.scoring == 0) {  // softmax's denominator
#pragma unroll
        for (uint32_t j = 0; j < PER; ++j)
            if (!((out >> j) & 1u)) sum += expf(v[j] - top);
        for (uint32_t d = 16; d; d >>= 1) sum += __shfl_xor_sync(kFull, sum, d);
    }

    Key key[PER];
    if (WIDE) {
        double total = 0.0;
        double pick[PER];
#pragma unroll
        for (uint32_t j = 0; j < PER; ++j) {
            pick[j] = 0.0;
            if ((out >> j) & 1u) continue;
            pick[j] = a.scoring == 0 ? exp((double)v[j] - (double)top) : 1.0 / (1.0 + exp(-(double)v[j]));
            total += pick[j];
        }
        if (a.scoring == 0)
            for (uint32_t d = 16; d; d >>= 1) total += __shfl_xor_sync(kFull, total, d);
        uint32_t groups_in = kFull;
        const uint32_t wide = a.experts / a.groups;
#pragma unroll
        for (uint32_t j = 0; j < PER; ++j) {
            const uint32_t e = lane + 32u * j;
            if (a.scoring == 0) pick[j] /= total;
            if (a.bias && e < a.experts) pick[j] += (double)a.bias[e];
        }
        if (a.groups > 1u) {
            // a group's rank is by the sum of its two largest picks that are not removed; lane g adds up group g
            double* mine = picks + (size_t)warp * a.experts;
#pragma unroll
            for (uint32_t j = 0; j < PER; ++j)
                if (lane + 32u * j < a.experts) mine[lane + 32u * j] = (out >> j) & 1u ? -INFINITY : pick[j];
            __syncwarp();
            Key rank = 0;
            if (lane < a.groups) {
                double first = -INFINITY, second = -INFINITY;
                bool bad = false;
                for (uint32_t i = 0; i < wide; ++i) {
                    const double p = mine[lane * wide + i];
                    bad |= isnan(p);
                    if (p > first) second = first, first = p;
                    else if (p > second) second = p;
                }
                const double both = second == -INFINITY ? first : first + second;
                rank = bad ? (Key)key_of((double)NAN) : (Key)key_of(both);
            }
            uint32_t ahead = 0;
            for (uint32_t g = 0; g < a.groups; ++g) {
                const Key other = __shfl_sync(kFull, rank, g);
                ahead += other > rank || (other == rank && g < lane);
            }
            groups_in = __ballot_sync(kFull, lane < a.groups && ahead < a.group_topk);
        }
#pragma unroll
        for (uint32_t j = 0; j < PER; ++j) {
            const uint32_t e = lane + 32u * j;
            key[j] = (out >> j) & 1u ? (Key)1 : (Key)key_of(pick[j]);
            if (e >= a.experts || (a.groups > 1u && !((groups_in >> (e / wide)) & 1u))) key[j] = 0;
        }
    } else {
#pragma unroll
        for (uint32_t j = 0; j < PER; ++j) {
            key[j] = (out >> j) & 1u ? (Key)1 : (Key)key_of(v[j]);
            if (lane + 32u * j >= a.experts) key[j] = 0;
        }
    }

    // rounds: lane k ends with the k-th choice
    uint32_t chosen = 0;
    bool gone = false;  // it is a removed one
    for (uint32_t k = 0; k < a.topk; ++k) {
        Key best = key[0];
        uint32_t j0 = 0;
#pragma unroll
        for (uint32_t j = 1; j < PER; ++j)
            if (key[j] > best) best = key[j], j0 = j;
        const Key most = warp_max(best);
        const uint32_t e = __reduce_min_sync(kFull, best == most ? lane + 32u * j0 : kFull);
        if (lane == (e & 31u))
#pragma unroll
            for (uint32_t j = 0; j < PER; ++j)
                if (j == e >> 5) key[j] = 0;
        if (lane == k) chosen = e, gone = most == (Key)1;
    }
    float score = 0.0f;
    if (lane < a.topk && !gone) {
        const float l = load_act(a.logits, a.dt, at + chosen);
        const float e = expf(a.scoring == 0 ? l - top : -fabsf(l));  // the sigmoid by the exponential that cannot overflow
        score = a.scoring == 0 ? e / sum : (l < 0.0f ? e : 1.0f) / (1.0f + e);
    }
    if (!any) score = 0.0f;
    if (a.renormalise) {
        float all = score;
        for (uint32_t d = 16; d; d >>= 1) all += __shfl_xor_sync(kFull, all, d);
        score = all == 0.0f ? 0.0f : score / all;
    }
    if (lane < a.topk) {
        a.inds[row * a.topk + lane] = (int32_t)chosen;
        a.scores[row * a.topk + lane] = score * a.scale;
    }
}

}  // namespace

cudaError_t launch_route(const RouteArgs& a, bool overlap, cudaStream_t stream) {
    const bool wide = a.bias || a.groups > 1u;
    const uint32_t smem = wide && a.groups > 1u ? kWarps * a.experts * 8u : 0u;
    const dim3 grid((unsigned)((a.rows + kWarps - 1u) / kWarps));
    auto go = [&](auto kernel) { return launch_overlapped(kernel, grid, kWarps * 32u, smem, stream, overlap, 1, a); };
    if (wide) {
        if (a.experts <= 128u) return go(route_rows<4, true>);
        if (a.experts <= 256u) return go(route_rows<8, true>);
        if (a.experts <= 512u) return go(route_rows<16, true>);
        return go(route_rows<32, true>);
    }
    if (a.experts <= 128u) return go(route_rows<4, false>);
    if (a.experts <= 256u) return go(route_rows<8, false>);
    if (a.experts <= 512u) return go(route_rows<16, false>);
    return go(route_rows<32, false>);
}

}  // namespace t3
