// Products with e4m3 weights that stream past few rows (up to 32): the linear, and the routed layer's two launches.
//
//   y[n, o] = sum over 128-blocks k of  c[n, k, o / 128] * sum over the block of q[n, i] w[o, i],     c = x scale * w scale
//
// The product is taken transposed: a unit of work is a 128 x 128 block of the weight (the A operand, 128 outputs by 128 inputs,
// K-major as it lies in memory) against the same 128 inputs of the rows (B, 16 or 32 of them), so D [128 outputs x rows] lies in
// tensor memory with an output a lane, and the block's scale and a row's multiply its columns: the epilogue warps add c * D to f32
// sums in registers, since a scale changes every 128 inputs. Bound by the weight's bytes: a block is 16 KB, 700 cycles of a
// multiprocessor's share of memory, against 128 cycles of tensor core and some 60 instructions of epilogue. 29 rows: 16384 -> 7168 in 26.4 us with the
// rows' quantising ahead (117 MB), a layer of 512 experts of 2048 x 512 in 125 us (700 MB).
//
// K is cut into slices, a CTA of a thread-block cluster each; the slices' sums meet in the cluster's shared memory, each CTA
// adding the columns n = rank, rank + split, .. in slice order, so the result does not depend on timing.
//
// Twelve warps: 0-3 and 4-7 epilogue, 32 outputs a warp, the fours taking turns at the blocks (one four was what bounded the kernel: 840 cycles a
// block of 32 columns, most of it the latency of a chain of small steps), 8 TMA, 9 tcgen05.mma, 10 and 11 the columns' scales of each
// four's blocks. With QUANT the CTAs quantise the rows themselves (their own slice of them), ahead of their weights' copies into
// shared memory: loads of rows behind a full queue of those took 21 us instead of 2.
//
// The code is kept short: what is executed once a launch or once a task comes from memory, since the weights have pushed it out of L2 and
// the loops out of the nearer caches. An exchange unrolled over the columns took 6000 cycles a task for one or two stores.
//
// The routed layer (rows <= 32): gate|up's unit of work for an expert is the same block against ALL rows of the call, whichever of them the
// router sent there: columns cost nothing here, and no row is gathered. gate|up's tile is 128 channels of gate (the first four's) and
// of up (the second's); its CTAs quantise silu(gate) * up and leave it as e4m3 for the rows that chose the expert. Down's tile is 128
// outputs over all experts in use (K runs over expert and input), the router's weight in c, so the sum over a row's experts is
// taken in registers in ascending order of the experts' numbers: no atomics, no third launch.
#include "t3_fp8.cuh"
#include "t3_fp8.h"
#include "t3_internal.h"

namespace t3 {
namespace {

constexpr uint32_t kWarps = 12, kThreads = 32u * kWarps;
constexpr uint32_t kEpiWarps = 8, kTmaWarp = 8, kMmaWarp = 9, kScaleWarp = 10;  // and 11
constexpr uint32_t kTileBytes = 128u * 128u;
constexpr uint32_t kStagesMax = 12;
constexpr uint32_t kAcc = 4;      // accumulators in tensor memory; even: one is always the same four's
constexpr uint32_t kAhead = 8;    // units a scale warp's fetches run ahead of their use (a trip to memory is four or five units long)
constexpr uint32_t kFull = 0xFFFFFFFFu;

// down: the most experts one of `split` slices of `used` experts' inputs touches
__host__ __device__ constexpr uint32_t slice_experts(uint32_t used, uint32_t split) { return (used + split - 1u) / split + 1u; }

// places in Fp8RowsLayout::bars
constexpr uint32_t kBarFull = 0, kBarEmpty = 8u * kStagesMax, kBarAccFull = 16u * kStagesMax, kBarAccEmpty = kBarAccFull + 8u * kAcc,
                   kBarRecvFull = kBarAccEmpty + 8u * kAcc, kBarRecvEmpty = kBarRecvFull + 8u, kWords = kBarRecvEmpty + 8u;
static_assert(kWords + 16u <= 512u, "barriers and words");

// a place in a ring and the parity of its round
struct Slot {
    uint32_t i, parity = 0;
    __device__ __forceinline__ explicit Slot(uint32_t first = 0) : i(first) {}
    __device__ __forceinline__ void next(uint32_t n, uint32_t by = 1) {
        i += by;
        if (i >= n) i -= n, parity ^= 1u;
    }
};

// The experts in use, ascending, each with the rows that chose it (a bit a row); ids outside the bank are nobody's. id: the experts of the slots
// threadIdx.x, + kThreads, .. (a number past the bank's where there is none). mask: zeros, before a __syncthreads. Returns how many.
constexpr uint32_t kIds = (32u * 32u + kThreads - 1u) / kThreads;
__device__ __forceinline__ uint32_t list_experts(const Fp8RowsArgs& a, const uint32_t (&id)[kIds], uint32_t* mask, uint2* list, uint32_t* chunks, uint32_t* count) {
    const uint32_t slots = a.rows * a.topk, lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    if (slots <= 32u) {  // one warp, a slot a lane, against every other slot (a token's call: 1.5 us by the general way below)
        if (warp == 0) {
            const uint32_t e = id[0];
            uint32_t rows = 0, smaller = 0;
            bool first = e < a.experts;
#pragma unroll 1
            for (uint32_t t = 0, row = 0, k = 0; t < slots; ++t) {
                const uint32_t other = __shfl_sync(kFull, e, t);
                if (other == e) {
                    rows |= 1u << row;
                    if (t < lane) first = false;
                }
                if (++k == a.topk) k = 0, ++row;
            }
            const uint32_t firsts = __ballot_sync(kFull, first);
#pragma unroll 1
            for (uint32_t t = 0; t < slots; ++t) {
                const uint32_t other = __shfl_sync(kFull, e, t);
                smaller += ((firsts >> t) & 1u) && other < e;
            }
            if (first) list[smaller] = make_uint2(e, rows);
            if (lane == 0) *count = __popc(firsts);
        }
        __syncthreads();
        return *count;
    }
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < kIds; ++i)
        if (id[i] < a.experts) atomicOr(&mask[id[i]], 1u << ((threadIdx.x + i * kThreads) / a.topk));
    __syncthreads();
    const uint32_t runs = (a.experts + 31u) / 32u;  // at most 64
    static_assert(kFp8ExpertsMax <= 64u * 32u, "two words a lane");
#pragma unroll 1
    for (uint32_t r = warp; r < runs; r += kWarps) {
        const uint32_t e = r * 32u + lane, in_use = __ballot_sync(kFull, e < a.experts && mask[e] != 0u);
        if (lane == 0) chunks[r] = __popc(in_use);
    }
    __syncthreads();
    const uint32_t n0 = lane < runs ? chunks[lane] : 0u, n1 = lane + 32u < runs ? chunks[lane + 32u] : 0u;
#pragma unroll 1
    for (uint32_t r = warp; r < runs; r += kWarps) {
        const uint32_t at = __reduce_add_sync(kFull, (lane < r ? n0 : 0u) + (lane + 32u < r ? n1 : 0u));
        const uint32_t e = r * 32u + lane, m = e < a.experts ? mask[e] : 0u, in_use = __ballot_sync(kFull, m != 0u);
        if (m != 0u) list[at + __popc(in_use & ((1u << lane) - 1u))] = make_uint2(e, m);
    }
    if (warp == 0) {
        const uint32_t all = __reduce_add_sync(kFull, n0 + n1);
        if (lane == 0) *count = all;
    }
    __syncthreads();
    return *count;
}

// sum n of a warp's (n the same in all lanes): a select tree, so that the loop around it is short
template <uint32_t CAP>
__device__ __forceinline__ float pick(const float2 (&sums)[CAP / 2u], uint32_t n) {
    float t[CAP / 2u];
#pragma unroll
    for (uint32_t i = 0; i < CAP / 2u; ++i) t[i] = n & 1u ? sums[i].y : sums[i].x;
#pragma unroll
    for (uint32_t w = CAP / 4u, bit = CAP / 2u; w >= 1u; w >>= 1, bit >>= 1)
#pragma unroll
        for (uint32_t i = 0; i < w; ++i) t[i] = n & bit ? t[i + w] : t[i];
    return t[0];
}

template <int MODE, uint32_t CAP, bool QUANT>
__global__ void __launch_bounds__(kThreads, 2) fp8_rows(const __grid_constant__ Fp8Maps maps, const __grid_constant__ Fp8RowsArgs a) {
    constexpr uint32_t kCols = kAcc * CAP, kIdesc = idesc_m128(CAP);
    constexpr uint32_t kStageBytes = kTileBytes + (QUANT ? 0u : CAP * 128u);
    constexpr uint32_t kOps = MODE == kFp8GateUp ? 2u : 1u;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023u) & ~(uintptr_t)1023u);
    const Fp8RowsLayout& l = a.l;
    const uint32_t base = smem_addr(smem), bars = base + l.bars;
    uint32_t* words = reinterpret_cast<uint32_t*>(smem + l.bars + kWords);  // dead, tensor memory, experts in use
    volatile uint32_t* dead = words;
    float* sx = reinterpret_cast<float*>(smem + l.sx);
    uint2* list = reinterpret_cast<uint2*>(smem + l.list);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const uint32_t rank = a.split > 1u ? cluster_rank() : 0u, cluster = blockIdx.x / a.split, clusters = gridDim.x / a.split;
    const uint32_t kbs = a.in / 128u, tiles = (a.out + 127u) / 128u, live = a.rows;

    if (warp == 0) {  // a barrier a lane: one thread for all of them took half a microsecond
        if (lane == 0) words[0] = 0u;
        auto init = [&](uint32_t at, uint32_t n) { mbar_init(reinterpret_cast<uint64_t*>(smem + l.bars + at), n); };
        if (lane < a.stages) init(kBarFull + 8u * lane, 1), init(kBarEmpty + 8u * lane, 1);
        if (lane < kAcc) init(kBarAccFull + 8u * lane, 2), init(kBarAccEmpty + 8u * lane, 4);
        if (lane == 31u) init(kBarRecvFull, 1), init(kBarRecvEmpty, kEpiWarps * a.split);
        mbar_init_fence();
    } else if (warp == kTmaWarp) {
        if (lane == 0) {
            prefetch_map(&maps.w[0]);
            if (MODE == kFp8GateUp) prefetch_map(&maps.w[1]);
            if (!QUANT) prefetch_map(&maps.rows);
            if (MODE == kFp8Linear && !a.early)  // into L2 only, which holds whatever the kernels before this one write
#pragma unroll 1
                for (uint32_t kb = kbs * rank / a.split, i = 0; kb < kbs * (rank + 1u) / a.split && i < a.stages; ++kb, ++i)
                    tma_prefetch_2d(&maps.w[0], (int)(kb * 128u), (int)(cluster * 128u));
        }
    }
    // (Waited for ahead of the first store to another CTA. Ahead of the allocation: no CTA waits, holding tensor memory, for one that waits for some.)
    if (a.split > 1u) {
        __syncwarp();
        cluster_arrive();
    }
    if (warp == kMmaWarp) {
        tmem_alloc(&words[1], kCols);
        tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = words[1];
    // What this kernel reads of the call's earlier launch waits for that one; what was there before the call (`early`: that launch has waited
    // for it ahead of letting this one start) does not. The next kernel may start once this one's tensor memory is allocated, since its
    // CTAs may hold theirs while they wait, and this one's own wait is over.
    const bool early = MODE == kFp8Down || (MODE == kFp8Linear && !QUANT && a.early);
    if (!early) {
        pdl_wait();
        pdl_trigger();
    }

    // The routing, on its way while the rows are quantised. (In down too it was complete before this launch started, since gate|up lets it start only
    // after its own wait. A CTA reads each word once, so past L1, where nothing would be found.)
    uint32_t id[kIds];
    if (MODE != kFp8Linear) {
        const uint32_t slots = a.rows * a.topk;
#pragma unroll
        for (uint32_t i = 0; i < kIds; ++i) {
            const uint32_t s = threadIdx.x + i * kThreads;
            id[i] = s < slots ? __ldcg(a.inds + s) : kFull;
            if (MODE == kFp8Down && s < slots) reinterpret_cast<float*>(smem + l.slots)[2u * s + 1u] = load_act_cg(a.scores, a.score_dt, s);
        }
        uint32_t* mask = reinterpret_cast<uint32_t*>(smem + l.mask);
        if (slots > 32u)
#pragma unroll 1
            for (uint32_t e = threadIdx.x; e < a.experts; e += kThreads) mask[e] = 0u;
    }

    if (QUANT) {
        // The rows' slice to e4m3, a warp a group, a lane's four values to their place in the swizzled tile. The groups come through the ring
        // (which has no weights yet), a share of it a warp: all of a warp's are on their way at once.
        const uint32_t q0 = kbs * rank / a.split, nb = kbs * (rank + 1u) / a.split - q0, groups = live * nb;
        const uint32_t bytes = a.x_dt == kF32 ? 512u : 256u, room = a.stages * kTileBytes / kWarps / bytes, stage = base + warp * room * bytes;
        const uint8_t* x = static_cast<const uint8_t*>(a.x);
        uint32_t g = warp, n = g / nb, kb = g - n * nb;
        const uint32_t dn = kWarps / nb, dk = kWarps - dn * nb;
        auto next = [&](uint32_t& n, uint32_t& kb) {
            n += dn, kb += dk;
            if (kb >= nb) kb -= nb, ++n;
        };
#pragma unroll 1
        while (g < groups) {
            uint32_t m = 0, n2 = n, kb2 = kb;
#pragma unroll 1
            for (; m < room && g < groups; ++m, g += kWarps) {
                if (lane * 16u < bytes) copy_async<16>(stage + m * bytes + lane * 16u, x + ((size_t)n * kbs + q0 + kb) * bytes + lane * 16u);
                next(n, kb);
            }
            copy_commit();
            copy_wait<0>();
            __syncwarp();
#pragma unroll 1
            for (uint32_t j = 0; j < m; ++j) {
                float v[4];
                load_act4(smem + (stage - base) + j * bytes, a.x_dt, 4u * lane, v);
                uint32_t most = max(max(magnitude(v[0]), magnitude(v[1])), max(magnitude(v[2]), magnitude(v[3])));
                most = __reduce_max_sync(kFull, most);
                const float s = fp8_scale(most);
                asm volatile("st.shared.b32 [%0], %1;" ::"r"(base + l.rows + (kb2 * CAP + n2) * 128u + (((lane >> 2) ^ (n2 & 7u)) << 4) + (lane & 3u) * 4u),
                             "r"(to_e4m3x4(v, s))
                             : "memory");
                if (lane == 0) sx[kb2 * CAP + n2] = s;
                next(n2, kb2);
            }
            __syncwarp();
        }
        proxy_fence();
        if (MODE == kFp8Linear) __syncthreads();  // (list_experts is one)
    }
    uint32_t used = 1;
    if (MODE == kFp8Down)
#pragma unroll
        for (uint32_t i = 0; i < kIds; ++i)
            if (threadIdx.x + i * kThreads < a.rows * a.topk) reinterpret_cast<uint32_t*>(smem + l.slots)[2u * (threadIdx.x + i * kThreads)] = id[i];
    if (MODE != kFp8Linear)
        used = list_experts(a, id, reinterpret_cast<uint32_t*>(smem + l.mask), list, reinterpret_cast<uint32_t*>(smem + l.chunks), &words[2]);

    // This CTA's units: of each of its tasks (a tile; gate|up: an expert's tile, of which a cluster takes several) `units` blocks. A unit
    // is (weight, 128-block of inputs, expert's place in the list, tile); they are walked by additions alone, since a division for
    // each cost the lone warps that walk them more than their waits.
    const uint32_t all = MODE == kFp8Down ? used * kbs : kbs;
    const uint32_t k0 = all * rank / a.split, k1 = all * (rank + 1u) / a.split;  // (a bank has at most 2^24 blocks)
    const uint32_t units = (k1 - k0) * kOps;
    const uint32_t tasks = MODE == kFp8GateUp ? used * tiles : tiles;
    const uint32_t mine = MODE == kFp8GateUp ? (tasks > cluster ? (tasks - cluster + clusters - 1u) / clusters : 0u) : 1u;
    const uint32_t blocks = mine * units;
    const uint32_t entry0 = MODE == kFp8Down ? k0 / kbs : MODE == kFp8GateUp ? cluster / tiles : 0u;
    const uint32_t tile0 = MODE == kFp8GateUp ? cluster - entry0 * tiles : cluster;
    const uint32_t d_entry = MODE == kFp8GateUp ? clusters / tiles : 0u, d_tile = MODE == kFp8GateUp ? clusters - d_entry * tiles : 0u;
    struct Walk {
        uint32_t op, kb, entry, tile;
    };
    auto next_task = [&](Walk& u) {
        u.entry += d_entry, u.tile += d_tile;
        if (u.tile >= tiles) u.tile -= tiles, ++u.entry;
    };
    auto step = [&](Walk& u) {
        if (MODE == kFp8GateUp && (u.op ^= 1u) != 0u) return;
        ++u.kb;
        if (MODE == kFp8Down && u.kb == kbs) u.kb = 0, ++u.entry;
        if (MODE == kFp8GateUp && u.kb == k1) u.kb = k0, next_task(u);
    };
    const Walk begin = {0u, MODE == kFp8Down ? k0 - entry0 * kbs : k0, entry0, tile0};

    float* weight = reinterpret_cast<float*>(smem + l.weight);
    if (MODE == kFp8Down && units) {
        // what the router gave each row for each of this slice's experts, over all of the row's slots that name the expert
        const uint2* slots = reinterpret_cast<const uint2*>(smem + l.slots);
        const uint32_t n = (k1 - 1u) / kbs + 1u - entry0;
#pragma unroll 1
        for (uint32_t i = threadIdx.x; i < n * CAP; i += kThreads) {
            const uint2 e = list[entry0 + i / CAP];
            const uint32_t r = i % CAP;
            float v = 0.0f;
            if ((e.y >> r) & 1u)
#pragma unroll 2
                for (uint32_t k = 0; k < a.topk; ++k)
                    if (slots[r * a.topk + k].x == e.x) v += __uint_as_float(slots[r * a.topk + k].y);
            weight[i] = v;
        }
        __syncthreads();
    }
    if (a.split > 1u && warp != kTmaWarp) {  // (the copies need no other CTA)
        __syncwarp();
        cluster_wait();
    }

    if (warp == kTmaWarp) {
        // early: first the ring full of weights, then the rows beside them, once the launch that makes them is over
        const uint32_t ahead = early ? min(a.stages, blocks) : 0u;
        Slot s;
        Walk u = begin, r = begin;
#pragma unroll 1
        for (uint32_t i = 0; i < blocks + ahead; ++i) {
            const bool rows_only = !QUANT && i >= ahead && i < 2u * ahead;
            if (!QUANT && early && i == ahead) {
                pdl_wait();
                pdl_trigger();
            }
            const uint32_t slot = rows_only ? i - ahead : s.i;
            const uint32_t full = bars + kBarFull + 8u * slot, at = base + slot * kStageBytes;
            if (!rows_only) fp8_wait(bars + kBarEmpty + 8u * slot, s.parity ^ 1u, dead, a.err, kErrEmptyWait);
            if (elect_one()) {
                if (!rows_only) {
                    mbar_arrive_expect_tx_addr(full, kStageBytes);
                    const uint32_t row = (MODE == kFp8Linear ? 0u : list[u.entry].x * a.out) + u.tile * 128u;
                    tma_load_2d(at, &maps.w[u.op], (int)(u.kb * 128u), (int)row, full);
                }
                if (!QUANT && i >= ahead)
                    tma_load_2d(at + kTileBytes, &maps.rows, (int)(r.kb * 128u), (int)(MODE == kFp8Down ? r.entry * CAP : 0u), full);
            }
            __syncwarp();
            if (!rows_only) {
                s.next(a.stages);
                step(u);
            }
            if (i >= ahead) step(r);
        }
        if (early && blocks == 0u) pdl_wait();
        if (a.split > 1u) {
            __syncwarp();
            cluster_wait();
        }
#pragma unroll 1
        for (uint32_t i = 0; i < a.stages; ++i) {  // the last products' arrivals are in before the CTA may end
            fp8_wait(bars + kBarEmpty + 8u * s.i, s.parity ^ 1u, dead, a.err, kErrEmptyWait);
            s.next(a.stages);
        }
    } else if (warp == kMmaWarp) {
        Slot s, c;
        uint32_t k = 0;  // gate|up, QUANT: the block's place in the slice, each twice
        uint32_t last = bars + kBarEmpty, last_parity = 1;  // of the last products' arrival
#pragma unroll 1
        for (uint32_t i = 0; i < blocks; ++i) {
            const uint32_t at = base + s.i * kStageBytes;
            const uint64_t ad = umma_desc(at), bd = umma_desc(QUANT ? base + l.rows + k / kOps * CAP * 128u : at + kTileBytes);
            if (++k == units) k = 0;
            fp8_wait(bars + kBarAccEmpty + 8u * c.i, c.parity ^ 1u, dead, a.err, kErrEmptyWait);
            fp8_wait(bars + kBarFull + 8u * s.i, s.parity, dead, a.err, kErrFullWait);
            tc_fence_after();
#pragma unroll
            for (uint32_t j = 0; j < 4u; ++j)  // 32 inputs each
                if (elect_one()) umma_e4m3(tmem + c.i * CAP, ad + 2u * j, bd + 2u * j, j, kIdesc);
            if (elect_one()) {
                umma_commit(bars + kBarEmpty + 8u * s.i);
                umma_commit(bars + kBarAccFull + 8u * c.i);
            }
            __syncwarp();
            last = bars + kBarEmpty + 8u * s.i, last_parity = s.parity;
            s.next(a.stages), c.next(kAcc);
        }
        fp8_wait(last, last_parity, dead, a.err, kErrMmaWait);
    } else if (warp >= kScaleWarp) {
        // The columns' scales of one four's units, a lane a column. What lies in memory (the block's scale; the rows', where they came quantised)
        // is on its way to shared memory kAhead units before its use.
        const uint32_t four = warp - kScaleWarp;
        const uint32_t fetch = l.fetch + four * kAhead * 132u;
        Walk f = begin, u;
        if (four) step(f);
        u = f;
        if (early) pdl_wait();
        auto ask = [&](uint32_t i, uint32_t slot) {
            if (i < blocks) {
                const uint2 e = MODE == kFp8Linear ? make_uint2(0u, (1u << (live - 1u)) * 2u - 1u) : list[f.entry];
                const uint32_t to = base + fetch + slot * 132u;
                if (lane == 0) copy_async<4>(to + 128u, a.w_scale[f.op] + ((size_t)e.x * tiles + f.tile) * kbs + f.kb);
                if (!QUANT && ((e.y >> lane) & 1u)) copy_async<4>(to + 4u * lane, a.x_scale + ((size_t)(MODE == kFp8Down ? f.entry * CAP : 0u) + lane) * kbs + f.kb);
                step(f), step(f);
            }
            copy_commit();
        };
#pragma unroll 1
        for (uint32_t j = 0; j < kAhead; ++j) ask(four + 2u * j, j);
        Slot c(four), q;
#pragma unroll 1
        for (uint32_t i = four; i < blocks; i += 2u) {
            copy_wait<(int)kAhead - 1>();
            __syncwarp();
            const float* got = reinterpret_cast<const float*>(smem + fetch + q.i * 132u);
            float v = 0.0f;
            if (QUANT) {
                if (lane < CAP) v = sx[(u.kb - k0) * CAP + lane] * got[32];
            } else {
                const uint32_t members = MODE == kFp8Down ? list[u.entry].y : (1u << (live - 1u)) * 2u - 1u;
                if ((members >> lane) & 1u) {  // (the others have no scale)
                    v = got[lane] * got[32];
                    if (MODE == kFp8Down) v *= weight[(u.entry - entry0) * CAP + lane];
                }
            }
            __syncwarp();
            ask(i + 2u * kAhead, q.i);
            q.next(kAhead);
            step(u), step(u);
            fp8_wait(bars + kBarAccEmpty + 8u * c.i, c.parity ^ 1u, dead, a.err, kErrEmptyWait);
            if (lane < CAP) reinterpret_cast<float*>(smem + l.c)[c.i * CAP + lane] = v;
            __syncwarp();
            if (lane == 0) mbar_arrive_addr(bars + kBarAccFull + 8u * c.i);
            c.next(kAcc, 2);
        }
    } else {
        const uint32_t four = warp >> 2, quarter = warp & 3u, row = quarter * 32u + lane;  // of the tile's 128 outputs
        const uint32_t own = (CAP + a.split - 1u) / a.split;
        uint32_t columns = 0;  // a bit for each column this CTA finishes
#pragma unroll 1
        for (uint32_t n = rank; n < CAP; n += a.split) columns |= 1u << n;
        Slot c(four);
        Walk t = begin;  // gate|up: the task; down: the expert of the unit
        if (MODE == kFp8Down && four) step(t);
#pragma unroll 1
        for (uint32_t turn = 0; turn < mine; ++turn) {
            float2 sums[CAP / 2u];  // gate|up: of gate (the first four) or of up
#pragma unroll
            for (uint32_t n = 0; n < CAP / 2u; ++n) sums[n] = make_float2(0.0f, 0.0f);
            // Rows that did not choose the expert: their columns are left out by sixteens; in down, where the others' would reach a sum, one by
            // one too (what lies in the place of such a row, nothing having been written there, or its product with a weight that is a NaN)
            uint32_t members = MODE == kFp8GateUp ? list[t.entry].y : (1u << (live - 1u)) * 2u - 1u;
#pragma unroll 1
            for (uint32_t i = four; i < units; i += 2u) {
                if (MODE == kFp8Down) members = list[t.entry].y;
                const uint32_t from = tmem + c.i * CAP + ((quarter * 32u) << 16), cc = base + l.c + c.i * CAP * 4u;
                fp8_wait(bars + kBarAccFull + 8u * c.i, c.parity, dead, a.err, kErrMmaWait);
                tc_fence_after();
#pragma unroll
                for (uint32_t b = 0; b < CAP; b += 16u) {
                    const uint32_t m = members >> b;
                    if ((m & 0xFFFFu) == 0u) continue;
                    uint32_t v[16];
                    float4 f[4];
                    tmem_ld_32x16(from + b, v);
#pragma unroll
                    for (uint32_t j = 0; j < 4u; ++j)
                        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(f[j].x), "=f"(f[j].y), "=f"(f[j].z), "=f"(f[j].w) : "r"(cc + 4u * b + 16u * j));
                    tmem_ld_wait(v);
#pragma unroll
                    for (uint32_t j = 0; j < 4u; ++j) {
                        float2 &lo = sums[b / 2u + 2u * j], &hi = sums[b / 2u + 2u * j + 1u];
                        if (MODE == kFp8Down) {
                            if ((m >> (4u * j)) & 1u) lo.x = fmaf(__uint_as_float(v[4u * j]), f[j].x, lo.x);
                            if ((m >> (4u * j)) & 2u) lo.y = fmaf(__uint_as_float(v[4u * j + 1u]), f[j].y, lo.y);
                            if ((m >> (4u * j)) & 4u) hi.x = fmaf(__uint_as_float(v[4u * j + 2u]), f[j].z, hi.x);
                            if ((m >> (4u * j)) & 8u) hi.y = fmaf(__uint_as_float(v[4u * j + 3u]), f[j].w, hi.y);
                        } else {
                            fma2(lo, v[4u * j], v[4u * j + 1u], f[j].x, f[j].y);
                            fma2(hi, v[4u * j + 2u], v[4u * j + 3u], f[j].z, f[j].w);
                        }
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_addr(bars + kBarAccEmpty + 8u * c.i);
                c.next(kAcc, 2);
                if (MODE == kFp8Down) step(t), step(t);
            }
            if (MODE == kFp8GateUp) {
                // Every CTA's sums of a row that chose the expert to the CTA that finishes it (row n: rank n mod split), in the order of its
                // rows, once that has read the last task's.
                const uint32_t full = bars + kBarRecvFull, mine_of = members & columns, count = __popc(mine_of);
                if (a.split > 1u) {
                    // Only then the arrival of this task's own: a task that sends this CTA nothing ends its phase with it, and a warp that still waited for
                    // the phase before would find the barrier past two of them, which it cannot tell from none.
                    if (turn) fp8_wait<true>(bars + kBarRecvEmpty, (turn - 1u) & 1u, dead, a.err, kErrEmptyWait);
                    if (warp == 0 && lane == 0) mbar_arrive_expect_tx_addr(full, count * a.split * 1024u);
                } else {
                    named_sync(4, kEpiWarps * 32u);  // (both fours have read the last task's)
                }
                const uint32_t from = base + l.part + rank * own * 1024u + four * 512u + row * 4u;
#pragma unroll 1
                for (uint32_t m = members; m; m &= m - 1u) {
                    const uint32_t n = __ffs(m) - 1u, to = n % a.split;
                    uint32_t j = 0;  // its place among the rows of that CTA
#pragma unroll 1
                    for (uint32_t o = to; o < n; o += a.split) j += (members >> o) & 1u;
                    const float v = pick<CAP>(sums, n);
                    if (a.split > 1u)
                        peer_store(peer_addr(from + j * 1024u, to), v, peer_addr(full, to));
                    else
                        *reinterpret_cast<float*>(smem + (from - base) + j * 1024u) = v;
                }
                if (a.split > 1u) fp8_wait<true>(full, turn & 1u, dead, a.err, kErrFullWait);
                else named_sync(4, kEpiWarps * 32u);
                const float* part = reinterpret_cast<const float*>(smem + l.part) + row;
                float* hid = reinterpret_cast<float*>(smem + l.hid) + row;
                uint32_t* red = reinterpret_cast<uint32_t*>(smem + l.red);
#pragma unroll 1
                for (uint32_t j = four; j < count; j += 2u) {  // each four finishes every other of this CTA's rows
                    float g = 0.0f, u = 0.0f;
#pragma unroll 1
                    for (uint32_t s = 0; s < a.split; ++s) g += part[(s * own + j) * 256u], u += part[(s * own + j) * 256u + 128u];
                    const float h = g / (1.0f + expf(-g)) * u;
                    hid[j * 128u] = h;  // (this thread alone reads it)
                    const uint32_t most = __reduce_max_sync(kFull, magnitude(h));
                    if (lane == 0) red[4u * j + quarter] = most;
                }
                named_sync(2u + four, 128);
                // (ahead of the stores below, which a release waits for; after the last task nobody waits, and a late arrival could find its CTA gone)
                if (a.split > 1u && lane < a.split && turn + 1u < mine) peer_arrive(peer_addr(bars + kBarRecvEmpty, lane));
                uint32_t m = mine_of;
#pragma unroll 1
                for (uint32_t j = 0; j < count; ++j, m &= m - 1u) {
                    if ((j & 1u) != four) continue;
                    const uint4 r = *reinterpret_cast<const uint4*>(red + 4u * j);
                    const float s = fp8_scale(max(max(r.x, r.y), max(r.z, r.w)));
                    const float v[4] = {hid[j * 128u], 0.0f, 0.0f, 0.0f};
                    const size_t at = (size_t)t.entry * CAP + (__ffs(m) - 1u);
                    a.h[at * a.out + t.tile * 128u + row] = (uint8_t)to_e4m3x4(v, s);
                    if (row == 0) a.h_scale[at * tiles + t.tile] = s;
                }
                named_sync(2u + four, 128);  // (red is written again for the next task)
                next_task(t);
            } else {
                // Both fours' sums over the ring, once every block has been multiplied, in the order of the CTAs that add the slices up (column
                // n: rank n mod split), and to each by one copy
                float* mid = reinterpret_cast<float*>(smem) + row;
                const uint32_t wrap = (a.split * own - 1u) * 128u;
                auto put = [&](bool add) {
                    uint32_t at = 0, to = 0;
#pragma unroll
                    for (uint32_t n = 0; n < CAP; ++n) {
                        mid[at] = (n & 1u ? sums[n >> 1].y : sums[n >> 1].x) + (add ? mid[at] : 0.0f);
                        at += own * 128u;
                        if (++to == a.split) to = 0, at -= wrap;
                    }
                };
                named_sync(4, kEpiWarps * 32u);
                if (four) put(false);
                named_sync(4, kEpiWarps * 32u);
                if (!four) {
                    put(true);
                    if (a.split > 1u) {
                        proxy_fence();
                        if (threadIdx.x == 0)
                            mbar_arrive_expect_tx_addr(bars + kBarRecvFull, __popc(columns & ((1u << (live - 1u)) * 2u - 1u)) * a.split * 512u);
                        named_sync(2, 128);
                        const uint32_t to = threadIdx.x;
                        if (to < a.split && to < live)
                            peer_copy(peer_addr(base + l.part + rank * own * 512u, to), base + to * own * 512u, (live - to + a.split - 1u) / a.split * 512u,
                                      peer_addr(bars + kBarRecvFull, to));
                    }
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
        __syncwarp();
    }
    // No CTA leaves while another may still write to it, nor while a copy may still read from it: linear's and down's arrive at the cluster's barrier
    // once all that was sent to them is there, so past it every copy is over.
    if (MODE != kFp8GateUp && a.split > 1u) {
        fp8_wait<true>(bars + kBarRecvFull, 0, dead, a.err, kErrFullWait);
        __syncwarp();
    }
    if (a.split > 1u) cluster_arrive_relaxed();
    if (MODE != kFp8GateUp) {
        if (early) pdl_wait();
        // a lane four outputs of a column, a warp a column
        const uint32_t own = (CAP + a.split - 1u) / a.split, o = cluster * 128u + 4u * lane;
        const uint32_t part = base + (a.split > 1u ? l.part : 0u) + 16u * lane;
#pragma unroll 1
        for (uint32_t j = warp; rank + j * a.split < live; j += kWarps) {
            float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 2
            for (uint32_t s = 0; s < a.split; ++s) {
                float4 f;
                asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(f.x), "=f"(f.y), "=f"(f.z), "=f"(f.w) : "r"(part + (s * own + j) * 512u));
                v[0] += f.x, v[1] += f.y, v[2] += f.z, v[3] += f.w;
            }
            const size_t at = (size_t)(rank + j * a.split) * a.out + o;
            if (a.out % 4u == 0u) {
                if (o >= a.out) continue;
                if (MODE == kFp8Down && a.shared) {
                    float f[4];
                    load_act4(a.shared, a.y_dt, at, f);
#pragma unroll
                    for (uint32_t k = 0; k < 4u; ++k) v[k] += f[k];
                }
                store_act4(a.y, a.y_dt, at, v);
            } else {  // (a linear's)
#pragma unroll
                for (uint32_t k = 0; k < 4u; ++k)
                    if (o + k < a.out) store_act(a.y, a.y_dt, at + k, v[k]);
            }
        }
        __syncwarp();
    }
    if (a.split > 1u) cluster_wait();
}

template <int MODE, uint32_t CAP, bool QUANT>
cudaError_t launch_as(const Fp8Maps& maps, const Fp8RowsArgs& a, uint32_t clusters, bool overlap, cudaStream_t stream) {
    static std::atomic<uint64_t> ready{0};
    if (cudaError_t rc = allow_smem_once(ready, reinterpret_cast<const void*>(fp8_rows<MODE, CAP, QUANT>), 227u * 1024u)) return rc;
    return launch_overlapped(fp8_rows<MODE, CAP, QUANT>, dim3(clusters * a.split), kThreads, a.l.total, stream, overlap, a.split, maps, a);
}

}  // namespace

Fp8RowsLayout fp8_rows_layout(int mode, uint32_t cap, bool quantise, uint32_t slice_max, uint32_t split, uint32_t stages, uint32_t experts,
                              uint32_t slots) {
    Fp8RowsLayout l;
    uint32_t at = stages * (kTileBytes + (quantise ? 0u : cap * 128u));
    auto take = [&](uint32_t bytes) {
        const uint32_t o = at;
        at += (bytes + 15u) & ~15u;
        return o;
    };
    const uint32_t own = (cap + split - 1u) / split, used = experts < slots ? experts : slots;  // own: columns a CTA adds up
    const bool gate_up = mode == kFp8GateUp, routed = mode != kFp8Linear, down = mode == kFp8Down;
    l.rows = take(quantise ? slice_max * cap * 128u : 0u);
    l.part = take(split * own * (gate_up ? 1024u : 512u));
    l.hid = take(gate_up ? own * 512u : 0u);
    l.red = take(gate_up ? own * 16u : 0u);
    l.sx = take(quantise ? slice_max * cap * 4u : 0u);
    l.fetch = take(2u * kAhead * 33u * 4u);
    l.c = take(kAcc * cap * 4u);
    l.mask = take(routed ? experts * 4u : 0u);
    l.list = take(routed ? used * 8u : 0u);
    l.chunks = take(routed ? 256u : 0u);  // a word for each 32 experts
    l.slots = take(down ? slots * 8u : 0u);
    l.weight = take(down ? slice_experts(used, split) * cap * 4u : 0u);
    l.bars = take(512u);
    l.total = at + 1024u;  // (and the way to the boundary)
    return l;
}

cudaError_t launch_fp8_rows(int mode, uint32_t cap, const Fp8Maps& maps, const Fp8RowsArgs& a, uint32_t clusters, bool overlap,
                            cudaStream_t stream) {
    if (mode == kFp8GateUp)
        return cap == 16u ? launch_as<kFp8GateUp, 16, true>(maps, a, clusters, overlap, stream)
                          : launch_as<kFp8GateUp, 32, true>(maps, a, clusters, overlap, stream);
    if (mode == kFp8Down)
        return cap == 16u ? launch_as<kFp8Down, 16, false>(maps, a, clusters, overlap, stream)
                          : launch_as<kFp8Down, 32, false>(maps, a, clusters, overlap, stream);
    if (a.x) return launch_as<kFp8Linear, 16, true>(maps, a, clusters, overlap, stream);
    return cap == 16u ? launch_as<kFp8Linear, 16, false>(maps, a, clusters, overlap, stream)
                      : launch_as<kFp8Linear, 32, false>(maps, a, clusters, overlap, stream);
}

}  // namespace t3
