// Products with e4m3 weights that stream past few rows: the linear up to 128 rows a tile, and the routed layer's two launches.
//
//   y[n, o] = sum over 128-blocks k of  c[n, k, o / 128] * sum over the block of q[n, i] w[o, i],     c = x scale * w scale
//
// The product is taken transposed: a unit of work is a 128 x 128 block of the weight (the A operand, 128 outputs by 128 inputs,
// K-major as it lies in memory) against the same 128 inputs of the rows (B, 16 to 128 of them), so D [128 outputs x rows] lies in
// tensor memory with an output a lane, and the block's scale and a row's multiply its columns: the epilogue warps add c * D to f32
// sums in registers, since a scale changes every 128 inputs. Bound by the weight's bytes: a block is 16 KB, 700 cycles of a
// multiprocessor's share of memory, against 128 cycles of tensor core at 16 rows and some 60 instructions of epilogue.
//
// K is cut into slices, a CTA of a thread-block cluster each; the slices' sums meet in the cluster's shared memory, each CTA
// adding the columns n = rank, rank + split, .. in slice order, so the result does not depend on timing.
//
// Eight warps: 0-3 epilogue (32 outputs each), 4 TMA, 5 tcgen05.mma, 6 the columns' scales, 7 helps quantising. With QUANT the
// CTAs quantise the rows themselves (their own slice of them) while the first weights are on their way.
//
// The routed layer (rows <= 32): gate|up's unit of work for an expert is the same block against ALL rows of the call, whichever of them the
// router sent there: columns cost nothing here, and no row is gathered. gate|up's tile is 128 channels of gate and of up; its CTAs
// quantise silu(gate) * up and leave it as e4m3 for the rows that chose the expert. Down's tile is 128 outputs over all experts in
// use (K runs over expert and input), the router's weight in c, so the sum over a row's experts is taken in registers in
// ascending order of the experts' numbers: no atomics, no third launch.
#include <type_traits>

#include "t3_fp8.cuh"
#include "t3_fp8.h"
#include "t3_internal.h"

namespace t3 {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kTmaWarp = 4, kMmaWarp = 5, kScaleWarp = 6;
constexpr uint32_t kTileBytes = 128u * 128u;
constexpr uint32_t kStagesMax = 12;

constexpr uint32_t acc_slots(uint32_t cap) { return cap <= 32u ? 4u : 2u; }

// Shared memory of a CTA, offsets from a 1024-byte boundary
struct Layout {
    uint32_t ring, rows, part, red, sx, c, mask, list, slots, bars, total;
};
__host__ __device__ __forceinline__ Layout layout_of(int mode, uint32_t cap, bool quantise, uint32_t slice_max, uint32_t split, uint32_t stages,
                                                     uint32_t experts, uint32_t slots) {
    Layout l;
    uint32_t at = 0;
    auto take = [&](uint32_t bytes) {
        const uint32_t o = at;
        at += (bytes + 15u) & ~15u;
        return o;
    };
    const uint32_t own = (cap + split - 1u) / split;  // columns a CTA adds up
    l.ring = take(stages * (kTileBytes + (quantise ? 0u : cap * 128u)));
    l.rows = take(quantise ? slice_max * cap * 128u : 0u);
    l.part = take(mode == kFp8GateUp ? split * own * 2u * 512u : split > 1u ? split * own * 512u : 0u);
    l.red = take(mode == kFp8GateUp ? own * 16u : 0u);
    l.sx = take(quantise ? slice_max * cap * 4u : 0u);
    l.c = take(acc_slots(cap) * cap * 4u);
    l.mask = take(mode == kFp8Linear ? 0u : experts * 4u);
    l.list = take(mode == kFp8Linear ? 0u : (experts < slots ? experts : slots) * 8u);
    l.slots = take(mode == kFp8Down ? slots * 8u : 0u);
    l.bars = take(512u);
    l.total = at;
    return l;
}

// places in Layout::bars
constexpr uint32_t kBarFull = 0, kBarEmpty = 8u * kStagesMax, kBarAccFull = 16u * kStagesMax, kBarAccEmpty = kBarAccFull + 32u,
                   kBarRecvFull = kBarAccEmpty + 32u, kBarRecvEmpty = kBarRecvFull + 8u, kWords = kBarRecvEmpty + 8u;
static_assert(kWords + 16u <= 512u, "barriers and words");

struct Slot {
    uint32_t i = 0, parity = 0;
    __device__ __forceinline__ void next(uint32_t n) {
        if (++i == n) i = 0, parity ^= 1u;
    }
};

// The experts in use, ascending, each with the rows that chose it (a bit a row); ids outside the bank are nobody's. Returns how many.
__device__ __forceinline__ uint32_t list_experts(const Fp8RowsArgs& a, uint32_t* mask, uint2* list, uint32_t* count) {
    for (uint32_t e = threadIdx.x; e < a.experts; e += kThreads) mask[e] = 0u;
    __syncthreads();
    for (uint32_t s = threadIdx.x; s < a.rows * a.topk; s += kThreads) {
        const uint32_t e = a.inds[s];
        if (e < a.experts) atomicOr(&mask[e], 1u << (s / a.topk));
    }
    __syncthreads();
    if (threadIdx.x < 32u) {
        uint32_t at = 0;
        for (uint32_t e0 = 0; e0 < a.experts; e0 += 32u) {
            const uint32_t e = e0 + threadIdx.x, m = e < a.experts ? mask[e] : 0u;
            const uint32_t used = __ballot_sync(0xFFFFFFFFu, m != 0u);
            if (m != 0u) list[at + __popc(used & ((1u << threadIdx.x) - 1u))] = make_uint2(e, m);
            at += __popc(used);
        }
        if (threadIdx.x == 0) *count = at;
    }
    __syncthreads();
    return *count;
}

template <int MODE, uint32_t CAP, bool QUANT>
__global__ void __launch_bounds__(kThreads, CAP <= 64u ? 2 : 1) fp8_rows(const __grid_constant__ Fp8Maps maps, const __grid_constant__ Fp8RowsArgs a) {
    constexpr uint32_t kAcc = acc_slots(CAP), kCols = kAcc * CAP;
    constexpr uint32_t kIdesc = idesc_m128(CAP);
    constexpr uint32_t kStageBytes = kTileBytes + (QUANT ? 0u : CAP * 128u);
    constexpr uint32_t kSums = MODE == kFp8GateUp ? 2u : 1u;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023u) & ~(uintptr_t)1023u);
    const Layout l = layout_of(MODE, CAP, QUANT, a.slice_max, a.split, a.stages, a.experts, a.rows * a.topk);
    const uint32_t base = smem_addr(smem), bars = base + l.bars;
    volatile uint32_t* dead = reinterpret_cast<uint32_t*>(smem + l.bars + kWords);
    uint32_t* words = reinterpret_cast<uint32_t*>(smem + l.bars + kWords);  // dead, tensor memory, experts in use
    float* sx = reinterpret_cast<float*>(smem + l.sx);
    float* cs = reinterpret_cast<float*>(smem + l.c);
    uint2* list = reinterpret_cast<uint2*>(smem + l.list);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const uint32_t rank = a.split > 1u ? cluster_rank() : 0u, cluster = blockIdx.x / a.split, clusters = gridDim.x / a.split;
    const uint32_t kbs = a.in / 128u, tiles = (a.out + 127u) / 128u;
    const uint32_t row0 = blockIdx.y * CAP, live = min(CAP, a.rows - row0);

    if (threadIdx.x == 0) {
        words[0] = 0u;
        auto init = [&](uint32_t at, uint32_t n) { mbar_init(reinterpret_cast<uint64_t*>(smem + l.bars + at), n); };
        for (uint32_t s = 0; s < a.stages; ++s) init(kBarFull + 8u * s, 1), init(kBarEmpty + 8u * s, 1);
        for (uint32_t s = 0; s < kAcc; ++s) init(kBarAccFull + 8u * s, 2), init(kBarAccEmpty + 8u * s, 4);
        init(kBarRecvFull, 4u * a.split), init(kBarRecvEmpty, 4u * a.split);
        mbar_init_fence();
    }
    if (warp == kTmaWarp) {
        if (lane == 0) {
            prefetch_map(&maps.w[0]);
            if (MODE == kFp8GateUp) prefetch_map(&maps.w[1]);
            if (!QUANT) prefetch_map(&maps.rows);
            if (MODE == kFp8Linear)  // into L2 only, which holds whatever the kernels before this one write
                for (uint32_t kb = kbs * rank / a.split, i = 0; kb < kbs * (rank + 1u) / a.split && i < a.stages; ++kb, ++i)
                    tma_prefetch_2d(&maps.w[0], (int)(kb * 128u), (int)(cluster * 128u));
        }
    } else if (warp == kMmaWarp) {
        tmem_alloc(&words[1], kCols);
        tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = words[1];
    if (a.split > 1u) cluster_arrive();  // (waited for ahead of the first store to another CTA)
    pdl_trigger();                       // after the tensor memory is this CTA's: a later kernel's CTAs may hold theirs while they wait
    pdl_wait();

    uint32_t used = 1;
    if (MODE != kFp8Linear) used = list_experts(a, reinterpret_cast<uint32_t*>(smem + l.mask), list, &words[2]);
    if (MODE == kFp8Down) {  // the routing, for the columns' weights
        uint2* slots = reinterpret_cast<uint2*>(smem + l.slots);
        for (uint32_t s = threadIdx.x; s < a.rows * a.topk; s += kThreads) slots[s] = make_uint2(a.inds[s], __float_as_uint(load_act(a.scores, a.score_dt, s)));
        __syncthreads();
    }
    if (a.split > 1u) cluster_wait();

    // this CTA's units: of each task (a tile; gate|up: an expert's tile) `units` blocks
    const uint32_t all = MODE == kFp8Down ? used * kbs : kbs;
    const uint32_t k0 = (uint32_t)((uint64_t)all * rank / a.split), k1 = (uint32_t)((uint64_t)all * (rank + 1u) / a.split);
    const uint32_t units = (k1 - k0) * kSums;
    const uint32_t tasks = MODE == kFp8GateUp ? used * tiles : tiles;
    struct Unit {
        uint32_t op, kb, entry;  // the weight (0, or 1 for up), its 128-block of inputs, the expert's place in the list
    };
    auto unit_of = [&](uint32_t task, uint32_t i) {
        Unit u;
        u.op = MODE == kFp8GateUp ? i & 1u : 0u;
        const uint32_t k = k0 + (MODE == kFp8GateUp ? i >> 1 : i);
        u.entry = MODE == kFp8GateUp ? task / tiles : MODE == kFp8Down ? k / kbs : 0u;
        u.kb = MODE == kFp8Down ? k - u.entry * kbs : k;
        return u;
    };
    auto tile_of = [&](uint32_t task) { return MODE == kFp8GateUp ? task % tiles : task; };

    if (QUANT && warp != kTmaWarp) {
        // the rows' slice to e4m3, a warp a group, four groups under way: lane's four values to their place in the swizzled tile
        const uint32_t me = warp < kTmaWarp ? warp : warp - 1u, nb = k1 - k0, groups = live * nb;
        for (uint32_t g0 = me; g0 < groups; g0 += 7u * 4u) {
            float v[4][4];
            uint32_t most[4];
#pragma unroll
            for (uint32_t j = 0; j < 4u; ++j) {
                const uint32_t g = g0 + 7u * j;
                if (g >= groups) break;
                const uint32_t n = g / nb, kb = g - n * nb;
                load_act4(a.x, a.x_dt, (size_t)(row0 + n) * a.in + (k0 + kb) * 128u + 4u * lane, v[j]);
            }
#pragma unroll
            for (uint32_t j = 0; j < 4u; ++j) {
                const uint32_t g = g0 + 7u * j;
                if (g >= groups) break;
                most[j] = max(max(magnitude(v[j][0]), magnitude(v[j][1])), max(magnitude(v[j][2]), magnitude(v[j][3])));
                most[j] = __reduce_max_sync(0xFFFFFFFFu, most[j]);
                const uint32_t n = g / nb, kb = g - n * nb;
                const float s = fp8_scale(most[j]);
                const uint32_t q = to_e4m3x4(v[j], s);
                asm volatile("st.shared.b32 [%0], %1;" ::"r"(base + l.rows + kb * CAP * 128u + n * 128u + (((lane >> 2) ^ (n & 7u)) << 4) +
                                                             (lane & 3u) * 4u),
                             "r"(q)
                             : "memory");
                if (lane == 0) sx[kb * CAP + n] = s;
            }
        }
        proxy_fence();
        named_sync(1, 7u * 32u);
    }

    if (warp == kTmaWarp) {
        Slot s;
        for (uint32_t task = cluster; task < tasks; task += clusters) {
            for (uint32_t i = 0; i < units; ++i) {
                const Unit u = unit_of(task, i);
                const uint32_t full = bars + kBarFull + 8u * s.i, at = base + l.ring + s.i * kStageBytes;
                fp8_wait(bars + kBarEmpty + 8u * s.i, s.parity ^ 1u, dead, a.err, kErrEmptyWait);
                if (elect_one()) {
                    const uint32_t bank_row = MODE == kFp8Linear ? 0u : list[u.entry].x * a.out;
                    mbar_arrive_expect_tx_addr(full, kStageBytes);
                    tma_load_2d(at, &maps.w[u.op], (int)(u.kb * 128u), (int)(bank_row + tile_of(task) * 128u), full);
                    if (!QUANT)
                        tma_load_2d(at + kTileBytes, &maps.rows, (int)(u.kb * 128u), (int)(MODE == kFp8Down ? u.entry * CAP : row0), full);
                }
                __syncwarp();
                s.next(a.stages);
            }
        }
    } else if (warp == kMmaWarp) {
        Slot s, c;
        for (uint32_t task = cluster; task < tasks; task += clusters) {
            for (uint32_t i = 0; i < units; ++i) {
                const uint32_t at = base + l.ring + s.i * kStageBytes;
                const uint32_t rows_at = QUANT ? base + l.rows + (MODE == kFp8GateUp ? i >> 1 : i) * CAP * 128u : at + kTileBytes;
                const uint64_t ad = umma_desc(at), bd = umma_desc(rows_at);
                fp8_wait(bars + kBarAccEmpty + 8u * c.i, c.parity ^ 1u, dead, a.err, kErrEmptyWait);
                fp8_wait(bars + kBarFull + 8u * s.i, s.parity, dead, a.err, kErrFullWait);
                tc_fence_after();
#pragma unroll
                for (uint32_t k = 0; k < 4u; ++k)  // 32 inputs each
                    if (elect_one()) umma_e4m3(tmem + c.i * CAP, ad + 2u * k, bd + 2u * k, k, kIdesc);
                if (elect_one()) {
                    umma_commit(bars + kBarEmpty + 8u * s.i);
                    umma_commit(bars + kBarAccFull + 8u * c.i);
                }
                __syncwarp();
                s.next(a.stages), c.next(kAcc);
            }
        }
    } else if (warp == kScaleWarp) {
        // the columns' scales of every unit, fetched a unit ahead of their use
        constexpr uint32_t kPer = CAP <= 32u ? 1u : CAP / 32u;
        uint32_t known = 0xFFFFFFFFu;
        float weight = 0.0f;
        auto fetch = [&](uint32_t task, uint32_t i, float (&v)[kPer]) {
            const Unit u = unit_of(task, i);
            const size_t blk = (size_t)(MODE == kFp8Linear ? 0u : list[u.entry].x) * tiles + tile_of(task);
            const float sw = __ldg(a.w_scale[u.op] + blk * kbs + u.kb);
#pragma unroll
            for (uint32_t j = 0; j < kPer; ++j) {
                const uint32_t n = lane + 32u * j;
                if (MODE == kFp8Down) {
                    const uint2 e = list[u.entry];
                    if (u.entry != known) {  // the row's weight of this expert, over all of its slots that name it
                        known = u.entry, weight = 0.0f;
                        const uint2* slots = reinterpret_cast<const uint2*>(smem + l.slots) + lane * a.topk;
                        if (lane < CAP && ((e.y >> lane) & 1u))
                            for (uint32_t k = 0; k < a.topk; ++k)
                                if (slots[k].x == e.x) weight += __uint_as_float(slots[k].y);
                    }
                    v[j] = lane < CAP && ((e.y >> lane) & 1u) ? a.x_scale[((size_t)u.entry * CAP + n) * kbs + u.kb] * sw * weight : 0.0f;
                } else if (QUANT) {
                    v[j] = n < live ? sx[(u.kb - k0) * CAP + n] * sw : 0.0f;
                } else {
                    v[j] = n < live ? __ldg(a.x_scale + (size_t)(row0 + n) * kbs + u.kb) * sw : 0.0f;
                }
            }
        };
        Slot c;
        for (uint32_t task = cluster; task < tasks; task += clusters) {
            float v[kPer];
            if (units) fetch(task, 0, v);
            for (uint32_t i = 0; i < units; ++i) {
                fp8_wait(bars + kBarAccEmpty + 8u * c.i, c.parity ^ 1u, dead, a.err, kErrEmptyWait);
#pragma unroll
                for (uint32_t j = 0; j < kPer; ++j)
                    if (CAP >= 32u || lane < CAP) cs[c.i * CAP + lane + 32u * j] = v[j];
                __syncwarp();
                if (lane == 0) mbar_arrive_addr(bars + kBarAccFull + 8u * c.i);
                c.next(kAcc);
                if (i + 1u < units) fetch(task, i + 1u, v);
            }
        }
    } else if (warp < kTmaWarp) {
        const uint32_t row = warp * 32u + lane;  // of the tile's 128 outputs
        Slot c;
        uint32_t turn = 0;
        for (uint32_t task = cluster; task < tasks; task += clusters, ++turn) {
            float acc[kSums][CAP];
#pragma unroll
            for (uint32_t s = 0; s < kSums; ++s)
#pragma unroll
                for (uint32_t n = 0; n < CAP; ++n) acc[s][n] = 0.0f;
            for (uint32_t i = 0; i < units; i += kSums) {
#pragma unroll
                for (uint32_t s = 0; s < kSums; ++s) {
                    fp8_wait(bars + kBarAccFull + 8u * c.i, c.parity, dead, a.err, kErrMmaWait);
                    tc_fence_after();
                    const uint32_t from = tmem + c.i * CAP + ((warp * 32u) << 16);
                    const float* cc = cs + c.i * CAP;
                    // rows that did not choose the expert have nothing in h: whatever lies there must not reach a sum
                    const uint32_t members = MODE == kFp8Down ? list[unit_of(task, i).entry].y : 0xFFFFFFFFu;
#pragma unroll
                    for (uint32_t b = 0; b < CAP; b += 16u) {
                        uint32_t v[16];
                        tmem_ld_32x16(from + b, v);
                        tmem_ld_wait(v);
#pragma unroll
                        for (uint32_t j = 0; j < 16u; j += 4u) {
                            const float4 f = *reinterpret_cast<const float4*>(cc + b + j);
                            const float g[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
                            for (uint32_t k = 0; k < 4u; ++k)
                                if (MODE != kFp8Down || ((members >> (b + j + k)) & 1u))
                                    acc[s][b + j + k] = fmaf(__uint_as_float(v[j + k]), g[k], acc[s][b + j + k]);
                        }
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_addr(bars + kBarAccEmpty + 8u * c.i);
                    c.next(kAcc);
                }
            }
            if (MODE == kFp8GateUp) {
                // every CTA's sums of column n to the CTA that finishes it (its rank is n mod split), once that has read the last task's
                const uint2 e = list[task / tiles];
                const uint32_t own = (CAP + a.split - 1u) / a.split;
                if (turn) fp8_wait<true>(bars + kBarRecvEmpty, (turn - 1u) & 1u, dead, a.err, kErrEmptyWait);
                uint32_t to = 0, at = base + l.part + rank * own * 1024u + row * 4u;
#pragma unroll
                for (uint32_t n = 0; n < CAP; ++n) {
                    if ((e.y >> n) & 1u) {
                        const uint32_t p = peer_addr(at, to);
                        peer_store(p, acc[0][n]);
                        peer_store(p + 512u, acc[kSums - 1u][n]);
                    }
                    if (++to == a.split) to = 0, at += 1024u;
                }
                __syncwarp();
                if (lane < a.split) peer_arrive(peer_addr(bars + kBarRecvFull, lane));
                fp8_wait<true>(bars + kBarRecvFull, turn & 1u, dead, a.err, kErrFullWait);
                float* part = reinterpret_cast<float*>(smem + l.part);
                uint32_t* red = reinterpret_cast<uint32_t*>(smem + l.red);
                for (uint32_t j = 0, n = rank; n < CAP; ++j, n += a.split) {
                    if (!((e.y >> n) & 1u)) continue;
                    float g = 0.0f, u = 0.0f;
                    for (uint32_t s = 0; s < a.split; ++s) {
                        const float* p = part + (s * own + j) * 256u + row;
                        g += p[0], u += p[128];
                    }
                    const float h = g / (1.0f + expf(-g)) * u;
                    part[j * 256u + row] = h;  // (slice 0's place: this thread alone reads it)
                    const uint32_t most = __reduce_max_sync(0xFFFFFFFFu, magnitude(h));
                    if (lane == 0) red[4u * j + warp] = most;
                }
                named_sync(2, 128);
                const uint32_t tile = task % tiles;
                for (uint32_t j = 0, n = rank; n < CAP; ++j, n += a.split) {
                    if (!((e.y >> n) & 1u)) continue;
                    const uint4 m = *reinterpret_cast<const uint4*>(red + 4u * j);
                    const float s = fp8_scale(max(max(m.x, m.y), max(m.z, m.w)));
                    const float v[4] = {part[j * 256u + row], 0.0f, 0.0f, 0.0f};
                    const size_t r = (size_t)(task / tiles) * CAP + n;
                    a.h[r * a.out + tile * 128u + row] = (uint8_t)to_e4m3x4(v, s);
                    if (row == 0) a.h_scale[r * tiles + tile] = s;
                }
                named_sync(2, 128);  // (red is written again for the next task)
                if (lane < a.split) peer_arrive(peer_addr(bars + kBarRecvEmpty, lane));
            } else if (a.split > 1u) {
                const uint32_t own = (CAP + a.split - 1u) / a.split;
                uint32_t to = 0, at = base + l.part + rank * own * 512u + row * 4u;
#pragma unroll
                for (uint32_t n = 0; n < CAP; ++n) {
                    if (n < live) peer_store(peer_addr(at, to), acc[0][n]);
                    if (++to == a.split) to = 0, at += 512u;
                }
            } else {
                const uint32_t o = task * 128u + row;
                if (o < a.out)
#pragma unroll
                    for (uint32_t n = 0; n < CAP; ++n)
                        if (n < live) {
                            const size_t at = (size_t)(row0 + n) * a.out + o;
                            store_act(a.y, a.y_dt, at, acc[0][n] + (MODE == kFp8Down && a.shared ? load_act(a.shared, a.y_dt, at) : 0.0f));
                        }
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem, kCols);  // ahead of the wait for the other CTAs: they may be waiting for tensor memory themselves
    }
    if (a.split > 1u) {
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        if (MODE != kFp8GateUp) {
            const uint32_t own = (CAP + a.split - 1u) / a.split, row = threadIdx.x & 127u, o = cluster * 128u + row;
            const float* part = reinterpret_cast<const float*>(smem + l.part);
            if (o < a.out)
                for (uint32_t j = threadIdx.x >> 7; rank + j * a.split < live; j += 2u) {
                    float v = 0.0f;
                    for (uint32_t s = 0; s < a.split; ++s) v += part[(s * own + j) * 128u + row];
                    const size_t at = (size_t)(row0 + rank + j * a.split) * a.out + o;
                    store_act(a.y, a.y_dt, at, v + (MODE == kFp8Down && a.shared ? load_act(a.shared, a.y_dt, at) : 0.0f));
                }
        }
    }
}

template <int MODE, uint32_t CAP, bool QUANT>
cudaError_t launch_as(const Fp8Maps& maps, const Fp8RowsArgs& a, uint32_t clusters, uint32_t row_tiles, uint32_t smem, bool overlap,
                      cudaStream_t stream) {
    static std::atomic<uint64_t> ready{0};
    if (cudaError_t rc = allow_smem_once(ready, reinterpret_cast<const void*>(fp8_rows<MODE, CAP, QUANT>), 227u * 1024u)) return rc;
    return launch_overlapped(fp8_rows<MODE, CAP, QUANT>, dim3(clusters * a.split, row_tiles), kThreads, smem, stream, overlap, a.split, maps, a);
}

}  // namespace

uint32_t fp8_rows_smem(int mode, uint32_t cap, bool quantise, uint32_t slice_max, uint32_t split, uint32_t stages, uint32_t experts,
                       uint32_t slots) {
    return layout_of(mode, cap, quantise, slice_max, split, stages, experts, slots).total + 1024u;
}

cudaError_t launch_fp8_rows(int mode, uint32_t cap, const Fp8Maps& maps, const Fp8RowsArgs& a, uint32_t clusters, uint32_t row_tiles,
                            uint32_t smem, bool overlap, cudaStream_t stream) {
    auto as = [&](auto m, auto c, auto q) {
        return launch_as<decltype(m)::value, decltype(c)::value, decltype(q)::value>(maps, a, clusters, row_tiles, smem, overlap, stream);
    };
    using std::integral_constant;
    constexpr auto no = std::false_type{};
    constexpr auto yes = std::true_type{};
    const integral_constant<uint32_t, 16> c16;
    const integral_constant<uint32_t, 32> c32;
    const integral_constant<uint32_t, 64> c64;
    const integral_constant<uint32_t, 128> c128;
    if (mode == kFp8GateUp) return cap == 16u ? as(integral_constant<int, kFp8GateUp>{}, c16, yes) : as(integral_constant<int, kFp8GateUp>{}, c32, yes);
    if (mode == kFp8Down) return cap == 16u ? as(integral_constant<int, kFp8Down>{}, c16, no) : as(integral_constant<int, kFp8Down>{}, c32, no);
    const integral_constant<int, kFp8Linear> lin;
    if (a.x) return cap == 16u ? as(lin, c16, yes) : as(lin, c32, yes);
    switch (cap) {
        case 16: return as(lin, c16, no);
        case 32: return as(lin, c32, no);
        case 64: return as(lin, c64, no);
        default: return as(lin, c128, no);
    }
}

}  // namespace t3
