// A router's logits to expert numbers and scores: what the routed layers take.
//
// A warp a row, lane l holding the experts l, l + 32, .. in registers. The choice is topk rounds of "the largest key, the lowest number
// among equals": keys are the picks' bit patterns made to order as whole numbers, so a round is two warp reductions and a look
// through each lane's values. Without bias or groups the pick is the logit itself (both scorings rise with it); with them it is score + bias,
// where two sums that differ in the last bits must still order as their exact values do: they are taken in 32 bits, and those that
// a choice hangs on and that are too near each other once more in 64. (All rows in 64 bits: 27.5 us at 8192 rows of 256 experts.) Long prompts: 1670
// instructions a row of 256 experts in 8 groups, 17.9 us at 8192 rows; a round is 69 of them, eight a third. While a multiprocessor has warps (31 of
// 64 on average) its schedulers issue in 62 % of the cycles and wait for a warp's last instruction in the others; the grid is 1.4 rounds of CTAs, so over the
// launch it is about half. Decode rows are bound by latency (4.8 us at one row of 512, ten rounds).
#include <cfloat>

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

// a type's lowest finite number: a logit at or below it removes its expert
__device__ __forceinline__ float lowest(int dt) { return dt == kF16 ? -65504.0f : __uint_as_float(dt == kBf16 ? 0xFF7F0000u : 0xFF7FFFFFu); }

__device__ __forceinline__ float number_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key); }
template <typename F>
__device__ __forceinline__ F warp_sum(F v) {
    for (uint32_t d = 16; d; d >>= 1) v += __shfl_xor_sync(kFull, v, d);
    return v;
}

// lanes that look through a group together: a power of two
__device__ __forceinline__ uint32_t group_lanes(uint32_t groups) { return groups <= 1u ? 32u : 1u << (31u - __clz(32u / groups)); }

// a sigmoid's pick in 64 bits: expert e's score and bias
__device__ __noinline__ double sigmoid_pick(float v, const float* bias, uint32_t e) {
    const double p = 1.0 / (1.0 + exp(-(double)v));
    return bias ? p + (double)bias[e] : p;
}

// Whether expert e of the row is removed: asked of its logit, since a pick of -inf is a live expert's too, whose bias is.
__device__ __noinline__ bool removed(const RouteArgs& a, size_t at, uint32_t e) { return load_act(a.logits, a.dt, at + e) <= lowest(a.dt); }

// The picks of one row in 64 bits and the choice among them, for the rows whose order 32 bits leave open and sigmoid_pick of a few experts does
// not settle: mine [experts] doubles of the warp's. Returns lane k's k-th choice, its highest bit set for a removed expert.
__device__ __noinline__ uint32_t choose_wide(const RouteArgs& a, size_t at, float top, double* mine, uint32_t lane) {
    double total = 0.0;
    uint32_t gone = 0;  // a bit for each 32 experts: this lane's is removed
#pragma unroll 1
    for (uint32_t e = lane; e < a.experts; e += 32u) {
        const float v = load_act(a.logits, a.dt, at + e);
        double p = -INFINITY;
        if (!(v <= lowest(a.dt))) p = a.scoring == 0 ? exp((double)v - (double)top) : sigmoid_pick(v, a.bias, e), total += p;
        else gone |= 1u << (e >> 5);
        mine[e] = p;
    }
    total = warp_sum(total);
#pragma unroll 1
    for (uint32_t e = lane; e < a.experts; e += 32u) {
        double p = mine[e];
        if (p != -INFINITY) {
            if (a.scoring == 0) mine[e] = p / total + (a.bias ? (double)a.bias[e] : 0.0);
        }
    }
    __syncwarp();
    uint32_t groups_in = kFull;
    const uint32_t wide = a.experts / a.groups;
    if (a.groups > 1u) {
        double first = -INFINITY, second = -INFINITY;
        bool bad = false;
        uint32_t live = 0;
        const uint32_t lanes = group_lanes(a.groups), g = lane / lanes;
        if (g < a.groups)
#pragma unroll 1
            for (uint32_t i = lane & (lanes - 1u); i < wide; i += lanes) {
                const double p = mine[g * wide + i];
                bad |= isnan(p);
                live += p != -INFINITY || !removed(a, at, g * wide + i);
                second = fmax(second, fmin(first, p));
                first = fmax(first, p);
            }
#pragma unroll 1
        for (uint32_t d = lanes >> 1; d; d >>= 1) {
            const double f = __shfl_xor_sync(kFull, first, d), s = __shfl_xor_sync(kFull, second, d);
            bad |= __shfl_xor_sync(kFull, (int)bad, d) != 0;
            live += __shfl_xor_sync(kFull, live, d);
            second = fmax(fmax(second, s), fmin(first, f));
            first = fmax(first, f);
        }
        // (a second of -inf is a live one where there are two, and the sum; a group without a live one is the last)
        const uint64_t mine_rank = bad ? ~0ull : live == 0u ? 0ull : key_of(live == 1u ? first : second == -INFINITY ? second : first + second);
        const uint64_t rank = __shfl_sync(kFull, mine_rank, lane * lanes & 31u);  // lane g: of group g
        uint32_t ahead = 0;
#pragma unroll 1
        for (uint32_t o = 0; o < a.groups; ++o) {
            const uint64_t other = __shfl_sync(kFull, rank, o);
            ahead += other > rank || (other == rank && o < lane);
        }
        groups_in = __ballot_sync(kFull, lane < a.groups && ahead < a.group_topk);
    }
    uint32_t chosen = 0, taken = 0;  // taken: a bit for each 32 experts, of this lane's
#pragma unroll 1
    for (uint32_t k = 0; k < a.topk; ++k) {
        uint64_t best = 0;
        uint32_t at_best = kFull;
#pragma unroll 1
        for (uint32_t e = lane; e < a.experts; e += 32u) {
            if (((taken >> (e >> 5)) & 1u) || !((groups_in >> (a.groups > 1u ? e / wide : 0u)) & 1u)) continue;
            const uint64_t key = (gone >> (e >> 5)) & 1u ? 1ull : key_of(mine[e]);
            if (key > best) best = key, at_best = e;
        }
        const uint64_t most = warp_max(best);
        const uint32_t e = __reduce_min_sync(kFull, best == most ? at_best : kFull);
        if (lane == (e & 31u)) taken |= 1u << (e >> 5);
        if (lane == k) chosen = e | (most == 1ull ? 0x80000000u : 0u);
    }
    return chosen;
}

// A lane's score times a number of the row's own, for scores that 32 bits hold with few bits or as 0: what divides them by their sum needs
// their ratios alone. The largest's exponential is 1.
__device__ __noinline__ float in_ratio(float logit, bool counts, int scoring) {
    const float most = number_of(warp_max(counts ? key_of(logit) : 0u));
    return counts ? expf(logit - most) / (scoring == 0 ? 1.0f : 1.0f + expf(logit)) : 0.0f;
}

// PER: experts a lane; WIDE: picks of score + bias
template <uint32_t PER, bool WIDE>
__global__ void __launch_bounds__(kWarps * 32u) route_rows(const __grid_constant__ RouteArgs a) {
    extern __shared__ double picks[];  // WIDE: [warps][experts + 32]
    pdl_wait();
    pdl_trigger();
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const size_t row = (size_t)blockIdx.x * kWarps + warp;
    if (row >= a.rows) return;
    const size_t at = row * a.experts;

    float v[PER];
    uint32_t out = 0;  // a bit for each removed expert of the lane
    float top = -INFINITY;
    if (a.dt == kF32) {
#pragma unroll
        for (uint32_t j = 0; j < PER; ++j) v[j] = lane + 32u * j < a.experts ? static_cast<const float*>(a.logits)[at + lane + 32u * j] : -INFINITY;
    } else {
#pragma unroll
        for (uint32_t j = 0; j < PER; ++j) {
            const uint16_t b = lane + 32u * j < a.experts ? static_cast<const uint16_t*>(a.logits)[at + lane + 32u * j] : (a.dt == kF16 ? 0xFC00u : 0xFF80u);
            v[j] = a.dt == kF16 ? __half2float(__ushort_as_half(b)) : __uint_as_float((uint32_t)b << 16);
        }
    }
    const float low = lowest(a.dt);
#pragma unroll
    for (uint32_t j = 0; j < PER; ++j) {
        if (v[j] <= low) out |= 1u << j;
        else top = fmaxf(top, v[j]);
    }
    static_assert(PER <= 32u, "a bit an expert");
    constexpr uint32_t kAll = PER == 32u ? kFull : (1u << (PER % 32u)) - 1u;
    const bool any = __any_sync(kFull, out != kAll);
    if (__any_sync(kFull, out != kAll)) {  // the largest of the live logits; with none but NaNs it stays -inf
        const uint32_t key = warp_max(key_of(top));
        top = key == kFull ? top : number_of(key);
    }
    float sum = 0.0f;
    if (a.scoring == 0) {  // softmax's denominator
#pragma unroll
        for (uint32_t j = 0; j < PER; ++j) {
            const float x = (out >> j) & 1u ? 0.0f : expf(v[j] - top);
            sum += x;
            if (WIDE) v[j] = x;  // (the picks need no more of the logit)
        }
        sum = warp_sum(sum);
    }

    uint32_t key[PER];
    bool lost = false;       // WIDE: the choice takes all of the row in 64 bits
    float slack = 0.0f;      // how far apart two picks are told apart for certain, ahead of their own rounding
    if (WIDE) {
        // Picks in 32 bits. What an order hangs on is looked at below: a score is off by at most 2^-21 (the sigmoid of the fast exponential and division),
        // or 45 steps of 2^-24 of the row's largest (softmax, whose sum is off by one for each addition), a sum with the bias by half a step
        // of its own. Rows with two that are nearer than that, one in a thousand, are settled in 64 bits.
        const float scale = a.scoring == 0 ? 1.0f / sum : 1.0f;  // of a softmax's terms; the largest is 1
        slack = scale * (a.scoring == 0 ? 0x1p-17f : 0x1.8p-20f);
        float* mine = reinterpret_cast<float*>(picks + (size_t)warp * (a.experts + 32u));
        const uint32_t wide = a.experts / a.groups, magic = ((1u << 20) + wide - 1u) / wide;  // e / wide = e magic >> 20, for e < 1024
        const uint32_t lanes = group_lanes(a.groups);
        bool odd = false;  // a live pick that is no number, or the lowest there is
#pragma unroll
        for (uint32_t j = 0; j < PER; ++j) {
            const uint32_t e = lane + 32u * j;
            float p = v[j] * scale;
            if (a.scoring != 0) {
                const float x = __expf(-fabsf(v[j]));
                p = __fdividef(v[j] < 0.0f ? x : 1.0f, 1.0f + x);
            }
            if (a.bias && e < a.experts) p += a.bias[e];
            const bool gone = (out >> j) & 1u;
            odd |= !gone && !(p > -INFINITY);
            key[j] = gone ? 1u : key_of(p);
            if (a.groups > 1u && e < a.experts) mine[e + ((e * magic) >> 20) * lanes] = gone ? -INFINITY : p;
            if (e >= a.experts) key[j] = 0;
        }
        odd = __any_sync(kFull, odd) != 0;
        lost = !any;
        if (odd) {
            bool nan = false;
#pragma unroll
            for (uint32_t j = 0; j < PER; ++j) nan |= key[j] == kFull;
            lost |= __any_sync(kFull, nan) != 0;
        }
        if (a.groups > 1u) {
            __syncwarp();
            // a group's rank is by the sum of its two largest picks that are not removed: of those in shared memory the removed ones are -inf, and the
            // live ones of -inf are looked for only where the row has one and a group is short of two others
            const uint32_t g = lane / lanes;
            float first = -INFINITY, second = -INFINITY;
            if (g < a.groups) {
                const float* p = mine + g * (wide + lanes);
#pragma unroll 4
                for (uint32_t i = lane & (lanes - 1u); i < wide; i += lanes) {
                    const float q = p[i];
                    second = fmaxf(second, fminf(first, q));
                    first = fmaxf(first, q);
                }
            }
#pragma unroll 1
            for (uint32_t d = lanes >> 1; d; d >>= 1) {
                const float f = __shfl_xor_sync(kFull, first, d), s = __shfl_xor_sync(kFull, second, d);
                second = fmaxf(fmaxf(second, s), fminf(first, f));
                first = fmaxf(first, f);
            }
            bool lowest_live = false;
            if (odd && __any_sync(kFull, g < a.groups && second == -INFINITY)) {
                if (g < a.groups)
#pragma unroll 1
                    for (uint32_t i = lane & (lanes - 1u); i < wide; i += lanes)
                        lowest_live |= mine[g * (wide + lanes) + i] == -INFINITY && !removed(a, at, g * wide + i);
#pragma unroll 1
                for (uint32_t d = lanes >> 1; d; d >>= 1) lowest_live |= __shfl_xor_sync(kFull, (int)lowest_live, d) != 0;
            }
            const float both = second == -INFINITY ? (lowest_live ? second : first) : first + second;
            const uint32_t rank = g < a.groups ? key_of(both) : 0u;
            uint32_t ahead = 0;
#pragma unroll 4
            for (uint32_t o = 0; o < a.groups; ++o) {
                const uint32_t other = __shfl_sync(kFull, rank, o * lanes);
                ahead += other > rank || (other == rank && o < g);
            }
            bool in = g < a.groups && ahead < a.group_topk;
            if (a.group_topk < a.groups) {
                const uint32_t least = __reduce_min_sync(kFull, in ? rank : kFull), next = __reduce_max_sync(kFull, in ? 0u : rank);
                const float l = number_of(least), n = number_of(next);
                // (a finite sum is clear of an infinite one; two of -inf are not: one may have no live expert, or be too large for 32 bits)
                if (!(l - n > 2.0f * slack + 0x1p-20f * (fminf(fabsf(l), FLT_MAX) + fminf(fabsf(n), FLT_MAX)))) {
                    // the groups' sums in 64 bits, of the two of each that are clear of its third; lane o's of group o
                    double sum64 = -INFINITY;
                    bool none = true;  // no live expert
                    bool settled = a.scoring != 0;
                    if (lane < a.groups) {
                        float one = -INFINITY, two = -INFINITY, three = -INFINITY;
                        uint32_t i1 = 0, i2 = 0;
                        const float* p = mine + lane * (wide + lanes);
#pragma unroll 1
                        for (uint32_t i = 0; i < wide; ++i) {
                            const float q = p[i];
                            if (q > one) three = two, two = one, i2 = i1, one = q, i1 = i;
                            else if (q > two) three = two, two = q, i2 = i;
                            else three = fmaxf(three, q);
                        }
                        settled &= two == -INFINITY || three == -INFINITY || two - three > slack + 0x1p-21f * (fabsf(two) + fabsf(three));
                        bool low = false;  // a live pick of -inf
                        if (odd && two == -INFINITY)
#pragma unroll 1
                            for (uint32_t i = 0; i < wide; ++i) low |= p[i] == -INFINITY && !removed(a, at, lane * wide + i);
                        none = one == -INFINITY && !low;
                        if (settled && one != -INFINITY && !low) {
                            sum64 = sigmoid_pick(load_act(a.logits, a.dt, at + lane * wide + i1), a.bias, lane * wide + i1);
                            if (two != -INFINITY) sum64 += sigmoid_pick(load_act(a.logits, a.dt, at + lane * wide + i2), a.bias, lane * wide + i2);
                        }
                    }
                    lost |= __any_sync(kFull, !settled) != 0;
                    const uint64_t mine64 = none ? 0ull : key_of(sum64);
                    uint32_t before = 0;
#pragma unroll 1
                    for (uint32_t o = 0; o < a.groups; ++o) {
                        const uint64_t other = __shfl_sync(kFull, mine64, o);
                        before += other > mine64 || (other == mine64 && o < lane);
                    }
                    in = __shfl_sync(kFull, before, g & 31u) < a.group_topk && g < a.groups;
                }
            }
            const uint32_t ins = __ballot_sync(kFull, in);
#pragma unroll
            for (uint32_t j = 0; j < PER; ++j)
                if (!((ins >> (((lane + 32u * j) * magic >> 20) * lanes & 31u)) & 1u)) key[j] = 0;
        }
    } else {
#pragma unroll
        for (uint32_t j = 0; j < PER; ++j) {
            key[j] = (out >> j) & 1u ? 1u : key_of(v[j]);
            if (lane + 32u * j >= a.experts) key[j] = 0;
        }
    }

    // Rounds: lane k ends with the k-th choice. WIDE goes on for as long as the next is too near the last to be told apart from it, so that the
    // lanes hold all that the choice may be among.
    uint32_t chosen = 0, its_key = 1, count = 0, last = 0, best = key[0];
#pragma unroll
    for (uint32_t j = 1; j < PER; ++j) best = max(best, key[j]);
    auto near = [&](uint32_t high, uint32_t low_key) {
        const float l = number_of(high), n = number_of(low_key);
        if (isinf(l) || isinf(n)) return false;  // a bias is: equal ones are equal in 64 bits too, and the lower number has been taken first
        return !(l - n > slack + 0x1p-21f * (fabsf(l) + fabsf(n)));
    };
#pragma unroll 1
    for (;; ++count) {
        if (!WIDE && count == a.topk) break;
        const uint32_t most = warp_max(best);
        if (WIDE && count >= a.topk) {
            if (most <= 1u || last <= 1u || !near(last, most)) break;
            if (count == 32u) {
                lost = true;
                break;
            }
        }
        uint32_t holders = __ballot_sync(kFull, best == most), e = 0;
        if ((holders & (holders - 1u)) != 0u) {  // equal keys in several lanes: the lowest expert's
            uint32_t first = kFull;
#pragma unroll
            for (uint32_t j = PER; j-- > 0u;)
                if (key[j] == most) first = lane + 32u * j;
            holders = 1u << (__reduce_min_sync(kFull, first) & 31u);
        }
        const uint32_t owner = __ffs(holders) - 1u;
        if (lane == owner) {
            uint32_t j0 = 0;
#pragma unroll
            for (uint32_t j = PER; j-- > 0u;)
                if (key[j] == most) j0 = j;
            best = 0;
#pragma unroll
            for (uint32_t j = 0; j < PER; ++j) {
                if (j == j0) key[j] = 0;
                best = max(best, key[j]);
            }
            e = lane + 32u * j0;
        }
        e = __shfl_sync(kFull, e, owner);
        if (lane == count) chosen = e, its_key = most;
        last = most;
    }
    bool gone = its_key == 1u;  // a removed one
    if (WIDE) {
        const uint32_t next = __shfl_down_sync(kFull, its_key, 1);
        if (__any_sync(kFull, lane + 1u < count && next > 1u && near(its_key, next))) {
            // the few in 64 bits, and in their order
            lost |= a.scoring == 0;
            if (!lost) {
                const double p = lane < count && !gone ? sigmoid_pick(load_act(a.logits, a.dt, at + chosen), a.bias, chosen) : 0.0;
                const uint64_t k64 = lane >= count ? 0ull : gone ? 1ull : key_of(p);
                uint32_t place = 0;
#pragma unroll 1
                for (uint32_t o = 0; o < count; ++o) {
                    const uint64_t other = __shfl_sync(kFull, k64, o);
                    const uint32_t its = __shfl_sync(kFull, chosen, o);
                    place += other > k64 || (other == k64 && its < chosen);
                }
                uint32_t* order = reinterpret_cast<uint32_t*>(picks + (size_t)warp * (a.experts + 32u));
                __syncwarp();
                if (lane < count) order[place] = chosen | (gone ? 0x80000000u : 0u);
                __syncwarp();
                chosen = order[lane < count ? lane : 0u];
                gone = chosen >> 31;
                chosen &= 0x7FFFFFFFu;
            }
        }
        if (lost) {
            __syncwarp();
            chosen = choose_wide(a, at, top, picks + (size_t)warp * (a.experts + 32u), lane);
            gone = chosen >> 31;
            chosen &= 0x7FFFFFFFu;
        }
    }
    float score = 0.0f, l = 0.0f;
    const bool counts = any && lane < a.topk && !gone;
    if (counts) {
        l = load_act(a.logits, a.dt, at + chosen);
        const float e = expf(a.scoring == 0 ? l - top : -fabsf(l));  // the sigmoid by the exponential that cannot overflow
        score = a.scoring == 0 ? e / sum : (l < 0.0f ? e : 1.0f) / (1.0f + e);
    }
    if (a.renormalise) {
        float all = warp_sum(score);
        if (all < 0x1p-16f) score = in_ratio(l, counts, a.scoring), all = warp_sum(score);
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
    const uint32_t smem = wide ? kWarps * (a.experts + 32u) * 8u : 0u;
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
