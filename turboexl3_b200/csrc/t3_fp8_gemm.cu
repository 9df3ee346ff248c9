// The 8-bit linear past 32 rows: y = x W^T from e4m3 rows and an e4m3 weight, one f32 scale for each 128 values of a row and each
// 128 x 128 block of the weight.
//
//   y[m, o] = sum over 128-blocks k of  sx[m, k] sw[o / 128, k] * sum over the block of q[m, i] w[o, i]
//
// D [128 rows x N outputs] of one 128-block of K lies in tensor memory with a row a lane, so the block's two scales are one number a thread, and
// the epilogue adds c * D to f32 sums in registers after every block, two values an instruction: tensor memory holds two such
// accumulators, one being multiplied into while the other is read. A block of a 128 x 256 tile is 512 cycles of tensor core at the nominal rate and 256
// of f32 multiply-adds; the products alone take 750 and the epilogue 840, and with two accumulators neither hides all of the other (1130 a
// block with the outputs' share), at 1.7 to 1.8 GHz of the board's power limit. Calls of few tiles are cut along
// K, a CTA of a cluster a slice; each CTA sends the others their share of the columns and adds up its own, in slice order.
//
// One persistent CTA a multiprocessor, twelve warps (two idle, for the registers' sake): 0-7 epilogue (a quarter of the rows, half of the columns each), 8 TMA, 9 tcgen05.mma.
// 8192 rows 2048 -> 6144: 113 us, 1.82 PFLOP/s (115 and more with the next columns' loads not under the multiply-adds).
// The outputs leave through shared memory, a warp 128 bytes of 32 rows at a time, so that a row's bytes are stored together.
#include "t3_fp8.cuh"
#include "t3_fp8.h"
#include "t3_internal.h"

namespace t3 {
namespace {

constexpr uint32_t kEpiWarps = 8, kTmaWarp = 8, kMmaWarp = 9, kThreads = 384;
// A multiprocessor's registers by role: the epilogue's warps hold 128 sums a thread, and at the 168 registers an even split gives they spilled
// (1820 cycles a block against 512 of tensor core)
constexpr uint32_t kRegsEven = 168, kRegsEpi = 216, kRegsOther = 72;
static_assert(256u * kRegsEpi + 128u * kRegsOther <= kThreads * kRegsEven && kThreads * kRegsEven <= 65536u, "what the block is launched with");
constexpr uint32_t kRowBytes = 128u * 128u, kOutBytes = kEpiWarps * 4096u;
// blocks in flight; tiles of 64 outputs serve calls of few tiles, whose slices are short: all of a slice at once
__host__ __device__ constexpr uint32_t stages_of(uint32_t n) { return n == 64u ? 8u : 4u; }

__host__ __device__ constexpr uint32_t stage_bytes(uint32_t n) { return kRowBytes + n * 128u; }
// the slices' sums: [slice][column of this CTA][row], a column's rows padded against bank conflicts of a lane a column
constexpr uint32_t kPartRows = 132;
__host__ __device__ constexpr uint32_t part_bytes(uint32_t n, bool split) { return split ? kPartRows * n * 4u : 0u; }
constexpr uint32_t smem_bytes(uint32_t n, bool split) { return stages_of(n) * stage_bytes(n) + (split ? 0u : kOutBytes) + part_bytes(n, split) + 256u + 1024u; }
static_assert(smem_bytes(256, false) <= 227u * 1024u && smem_bytes(128, true) <= 227u * 1024u && smem_bytes(64, true) <= 227u * 1024u, "shared memory of a CTA");
static_assert(kPartRows * 128u * 4u <= stages_of(128) * stage_bytes(128), "a CTA's sums over its ring");

// 16-bit or f32 outputs of 32 rows x 128 bytes from a warp's buffer: y at (first row, first column); rows and columns past the ends are left out
__device__ __forceinline__ void store_rows(uint32_t buffer, void* y, int dt, size_t row0, uint32_t rows, uint32_t col0, uint32_t out, uint32_t lane) {
    const uint32_t size = dt == kF32 ? 4u : 2u, per = 16u / size;  // values of 16 bytes
    const uint32_t j = lane & 7u, col = col0 + j * per;
    const bool whole = out % per == 0u;  // (y starts on 16 bytes)
#pragma unroll 1
    for (uint32_t r = lane >> 3; r < rows; r += 4u) {
        uint4 w;
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(buffer + r * 128u + ((j ^ (r & 7u)) << 4)));
        uint8_t* at = static_cast<uint8_t*>(y) + ((row0 + r) * out + col) * size;
        if (whole) {
            if (col < out) *reinterpret_cast<uint4*>(at) = w;
        } else {
            const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (uint32_t k = 0; k < 4u; ++k) {
                if (size == 4u) {
                    if (col + k < out) *reinterpret_cast<uint32_t*>(at + 4u * k) = v[k];
                } else {
                    if (col + 2u * k < out) *reinterpret_cast<uint16_t*>(at + 4u * k) = (uint16_t)v[k];
                    if (col + 2u * k + 1u < out) *reinterpret_cast<uint16_t*>(at + 4u * k + 2u) = (uint16_t)(v[k] >> 16);
                }
            }
        }
    }
}

__device__ __forceinline__ uint32_t pack_as(float a, float b, int dt) {
    if (dt == kF16) return pack_half2(a, b);
    const __nv_bfloat162 o = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&o);
}

// a whole warp's wait, in place
__device__ __forceinline__ void whole_wait(uint32_t bar, uint32_t parity, volatile uint32_t* dead, uint32_t* err, uint32_t bit) {
    fp8_wait_here<false, false>(bar, parity, dead, err, bit);
    __syncwarp();
}
// one behind the warp's last issue (see fp8_wait_here): a call in the split kernels, which have registers to spare for it (200 rows 7168 -> 576: 15.0 us
// in place, 14.8 so; in the others it has the epilogue spill, 8192 rows 2048 -> 6144 135 -> 145)
template <bool SPLIT, bool CLUSTER>
__device__ __forceinline__ void last_wait(uint32_t bar, uint32_t parity, volatile uint32_t* dead, uint32_t* err, uint32_t bit) {
    if (SPLIT) {
        fp8_wait<CLUSTER>(bar, parity, dead, err, bit);
    } else {
        fp8_wait_here<CLUSTER, true>(bar, parity, dead, err, bit);
        __syncwarp();
    }
}

template <uint32_t N, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1) fp8_gemm(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap,
                                                         const __grid_constant__ Fp8GemmArgs a) {
    constexpr uint32_t kStages = stages_of(N), kStageBytes = stage_bytes(N), kIdesc = idesc_m128(N), kCols = 2u * N, kMine = N / 2u;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023u) & ~(uintptr_t)1023u);
    const uint32_t base = smem_addr(smem), outs = base + kStages * kStageBytes, part = outs + (SPLIT ? 0u : kOutBytes), bars = part + part_bytes(N, SPLIT);
    uint8_t* bars_at = smem + (bars - base);
    // full[kStages], empty[kStages], accumulator full[2], empty[2], sums received
    const uint32_t full = bars, empty = bars + 8u * kStages, acc_full = bars + 16u * kStages, acc_empty = acc_full + 16u, recv = acc_full + 32u;
    uint32_t* words = reinterpret_cast<uint32_t*>(bars_at + 16u * kStages + 40u);
    volatile uint32_t* dead = words;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const uint32_t split = SPLIT ? a.split : 1u, rank = SPLIT ? cluster_rank() : 0u;
    const uint32_t kbs = a.in / 128u, k0 = kbs * rank / split, k1 = kbs * (rank + 1u) / split;
    const uint32_t row_tiles = (a.rows + 127u) / 128u, tiles = row_tiles * ((a.out + N - 1u) / N);
    const uint32_t first = SPLIT ? blockIdx.x / split : blockIdx.x, stride = SPLIT ? tiles : gridDim.x;

    if (warp == 0) {
        if (lane == 0) words[0] = 0u;
        auto init = [&](uint32_t at, uint32_t n) { mbar_init(reinterpret_cast<uint64_t*>(bars_at + at), n); };
        if (lane < kStages) init(8u * lane, 1), init(8u * (kStages + lane), 1);
        if (lane < 2u) init(16u * kStages + 8u * lane, 1), init(16u * kStages + 16u + 8u * lane, kEpiWarps);
        if (lane == 2u) init(16u * kStages + 32u, 1);
        mbar_init_fence();
    } else if (warp == kTmaWarp) {
        if (lane == 0) prefetch_map(&wmap), prefetch_map(&xmap);
    }
    if (SPLIT) {  // (ahead of the allocation: no CTA waits, holding tensor memory, for one that waits for some)
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
    if (!a.early) {
        pdl_wait();
        pdl_trigger();
    }
    if (SPLIT) {
        __syncwarp();
        cluster_wait();
    }

    if (warp >= kEpiWarps) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
        if (warp == kTmaWarp) {
            // early: the rows are quantised by the launch before this one, which has waited for what was there before the call; a ring of weights comes
            // first, then the rows beside them
            const uint32_t units = tiles > first ? (tiles - first + stride - 1u) / stride * (k1 - k0) : 0u;
            const uint32_t ahead = a.early ? min(kStages, units) : 0u;
            uint32_t slot = 0, parity = 1, t = first, kb = k0, rt = first, rkb = k0;  // the weights' place, and the rows'
    #pragma unroll 1
            for (uint32_t i = 0; i < units + ahead; ++i) {
                const bool rows_only = i >= ahead && i < 2u * ahead;
                if (a.early && i == ahead) {
                    pdl_wait();
                    pdl_trigger();
                }
                const uint32_t s = rows_only ? i - ahead : slot, bar = full + 8u * s, at = base + s * kStageBytes;
                if (!rows_only) whole_wait(empty + 8u * s, parity, dead, a.err, kErrEmptyWait);
                if (elect_one()) {
                    if (!rows_only) {
                        mbar_arrive_expect_tx_addr(bar, kStageBytes);
                        tma_load_2d(at + kRowBytes, &wmap, (int)(kb * 128u), (int)(t / row_tiles * N), bar);
                    }
                    if (i >= ahead) tma_load_2d(at, &xmap, (int)(rkb * 128u), (int)(rt % row_tiles * 128u), bar);
                }
                __syncwarp();
                if (!rows_only) {
                    if (++slot == kStages) slot = 0, parity ^= 1u;
                    if (++kb == k1) kb = k0, t += stride;
                }
                if (i >= ahead && ++rkb == k1) rkb = k0, rt += stride;
            }
            if (a.early && units == 0u) pdl_wait();
#pragma unroll 1
            for (uint32_t i = 0; i < kStages; ++i) {  // the last products' arrivals are in before the CTA may end
                last_wait<SPLIT, false>(empty + 8u * slot, parity, dead, a.err, kErrEmptyWait);
                if (++slot == kStages) slot = 0, parity ^= 1u;
            }
        } else if (warp == kMmaWarp) {
            uint32_t slot = 0, parity = 0, acc = 0, acc_parity = 1;
            uint32_t last = empty, last_parity = 1;  // of the last products' arrival
    #pragma unroll 1
            for (uint32_t t = first; t < tiles; t += stride) {
    #pragma unroll 1
                for (uint32_t kb = k0; kb < k1; ++kb) {
                    const uint32_t at = base + slot * kStageBytes;
                    const uint64_t ad = umma_desc(at), bd = umma_desc(at + kRowBytes);
                    whole_wait(acc_empty + 8u * acc, acc_parity, dead, a.err, kErrEmptyWait);
                    whole_wait(full + 8u * slot, parity, dead, a.err, kErrFullWait);
                    tc_fence_after();
    #pragma unroll
                    for (uint32_t j = 0; j < 4u; ++j)  // 32 inputs each
                        if (elect_one()) umma_e4m3(tmem + acc * N, ad + 2u * j, bd + 2u * j, j, kIdesc);
                    if (elect_one()) {
                        umma_commit(empty + 8u * slot);
                        umma_commit(acc_full + 8u * acc);
                    }
                    __syncwarp();
                    last = empty + 8u * slot, last_parity = parity;
                    if (++slot == kStages) slot = 0, parity ^= 1u;
                    acc ^= 1u;
                    if (acc == 0u) acc_parity ^= 1u;
                }
            }
            last_wait<SPLIT, false>(last, last_parity, dead, a.err, kErrMmaWait);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsEpi));
        const uint32_t quarter = warp & 3u, half = warp >> 2, buffer = outs + warp * 4096u;
        if (a.early) pdl_wait();
        uint32_t acc = 0, parity = 0;
#pragma unroll 1
        for (uint32_t t = first; t < tiles; t += stride) {
            const uint32_t row0 = t % row_tiles * 128u + quarter * 32u, col0 = t / row_tiles * N + half * kMine;
            const float* xs = a.x_scale + (size_t)min(row0 + lane, a.rows - 1u) * kbs;
            const float* ws = a.w_scale + (size_t)(min(col0, a.out - 1u) / 128u) * kbs;
            float2 sums[kMine / 2u];
#pragma unroll
            for (uint32_t n = 0; n < kMine / 2u; ++n) sums[n] = make_float2(0.0f, 0.0f);
            // the scales two blocks ahead of their use, in turns (by plain loads: the rows' may be written by the launch before, after this one has
            // started, and a load through the read-only path is for what no kernel writes while this one is there)
            float sx[2], sw[2];
#pragma unroll
            for (uint32_t p = 0; p < 2u; ++p) sx[p] = k0 + p < k1 ? xs[k0 + p] : 0.0f, sw[p] = k0 + p < k1 ? ws[k0 + p] : 0.0f;
#pragma unroll 1
            for (uint32_t kb = k0; kb < k1; kb += 2u) {
#pragma unroll
                for (uint32_t p = 0; p < 2u; ++p) {
                    if (kb + p >= k1) break;
                    const float c = sx[p] * sw[p];
                    if (kb + p + 2u < k1) sx[p] = xs[kb + p + 2u], sw[p] = ws[kb + p + 2u];
                    whole_wait(acc_full + 8u * acc, parity, dead, a.err, kErrMmaWait);
                    tc_fence_after();
                    const uint32_t from = tmem + acc * N + half * kMine + ((quarter * 32u) << 16);
                    // (the next sixteen columns on their way under the multiply-adds of these: 125 -> 115 us at 8192 rows 2048 -> 6144)
                    uint32_t v[2][16];
                    tmem_ld_32x16(from, v[0]);
#pragma unroll
                    for (uint32_t b = 0; b < kMine; b += 16u) {
                        tmem_ld_wait(v[(b >> 4) & 1u]);
                        if (b + 16u < kMine) tmem_ld_32x16(from + b + 16u, v[((b >> 4) + 1u) & 1u]);
#pragma unroll
                        for (uint32_t j = 0; j < 16u; j += 2u) fma2(sums[(b + j) / 2u], v[(b >> 4) & 1u][j], v[(b >> 4) & 1u][j + 1u], c, c);
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_addr(acc_empty + 8u * acc);
                    acc ^= 1u;
                    if (acc == 0u) parity ^= 1u;
                }
            }
            if (SPLIT) {
                // the sums over the ring, whose every block has been multiplied, and each CTA's columns to it by one copy
                const uint32_t bytes = N / split * kPartRows * 4u;
                const uint32_t at = base + (half * kMine * kPartRows + quarter * 32u + lane) * 4u;
#pragma unroll
                for (uint32_t n = 0; n < kMine; ++n)
                    asm volatile("st.shared.f32 [%0], %1;" ::"r"(at + n * kPartRows * 4u), "f"(n & 1u ? sums[n >> 1].y : sums[n >> 1].x) : "memory");
                if (threadIdx.x == 0) mbar_arrive_expect_tx_addr(recv, split * bytes);
                proxy_fence();
                named_sync(1, kEpiWarps * 32u);
                if (threadIdx.x < split) peer_copy(peer_addr(part + rank * bytes, threadIdx.x), base + threadIdx.x * bytes, bytes, peer_addr(recv, threadIdx.x));
                continue;
            }
            const uint32_t rows = row0 < a.rows ? min(32u, a.rows - row0) : 0u;
            const uint32_t mine = buffer + lane * 128u;
            auto put = [&](uint32_t j, uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3) {
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(mine + ((j ^ (lane & 7u)) << 4)), "r"(w0), "r"(w1), "r"(w2), "r"(w3) : "memory");
            };
            if (a.y_dt == kF32) {
#pragma unroll
                for (uint32_t b = 0; b < kMine; b += 32u) {
#pragma unroll
                    for (uint32_t j = 0; j < 8u; ++j) {
                        const float2 u = sums[b / 2u + 2u * j], v = sums[b / 2u + 2u * j + 1u];
                        put(j, __float_as_uint(u.x), __float_as_uint(u.y), __float_as_uint(v.x), __float_as_uint(v.y));
                    }
                    __syncwarp();
                    store_rows(buffer, a.y, kF32, row0, rows, col0 + b, a.out, lane);
                    __syncwarp();
                }
            } else {
#pragma unroll
                for (uint32_t b = 0; b < kMine; b += 64u) {
#pragma unroll
                    for (uint32_t j = 0; j < 8u; ++j) {
                        const float2* u = &sums[b / 2u + 4u * j];
                        put(j, pack_as(u[0].x, u[0].y, a.y_dt), pack_as(u[1].x, u[1].y, a.y_dt), pack_as(u[2].x, u[2].y, a.y_dt), pack_as(u[3].x, u[3].y, a.y_dt));
                    }
                    __syncwarp();
                    store_rows(buffer, a.y, a.y_dt, row0, rows, col0 + b, a.out, lane);
                    __syncwarp();
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
    if (SPLIT) {
        // (a CTA arrives once all that was sent to it is there: past the barrier no copy reads from a CTA any more, nor writes to one)
        last_wait<true, true>(recv, 0, dead, a.err, kErrFullWait);
        __syncwarp();
        cluster_arrive_relaxed();
        if (a.early) pdl_wait();
        const uint32_t width = N / split, row0 = first % row_tiles * 128u, col0 = first / row_tiles * N + rank * width;
        const float* p = reinterpret_cast<const float*>(smem + (part - base));
        const uint32_t shift = 31u - __clz(width);  // (the slices are a power of two)
#pragma unroll 1
        for (uint32_t i = threadIdx.x; i < 128u * width; i += kThreads) {
            const uint32_t r = i >> shift, n = i & (width - 1u);
            if (row0 + r >= a.rows || col0 + n >= a.out) continue;
            float v = 0.0f;
#pragma unroll 4
            for (uint32_t s = 0; s < split; ++s) v += p[(s * width + n) * kPartRows + r];
            store_act(a.y, a.y_dt, (size_t)(row0 + r) * a.out + col0 + n, v);
        }
        __syncwarp();
        cluster_wait();
    }
}

template <uint32_t N, bool SPLIT>
cudaError_t launch_as(const CUtensorMap& w, const CUtensorMap& x, const Fp8GemmArgs& a, uint32_t grid, bool overlap, cudaStream_t stream) {
    static std::atomic<uint64_t> ready{0};
    constexpr uint32_t smem = smem_bytes(N, SPLIT);
    if (cudaError_t rc = allow_smem_once(ready, reinterpret_cast<const void*>(fp8_gemm<N, SPLIT>), smem)) return rc;
    return launch_overlapped(fp8_gemm<N, SPLIT>, dim3(grid), kThreads, smem, stream, overlap, a.split, w, x, a);
}

uint32_t div_up(uint32_t a, uint32_t b) { return (a + b - 1u) / b; }

}  // namespace

Fp8GemmPlan plan_fp8_gemm(uint32_t rows, uint32_t in, uint32_t out) {
    const uint32_t sms = multiprocessors(), kbs = in / 128u, row_tiles = div_up(rows, 128u);
    const uint32_t wide = row_tiles * div_up(out, 256u), narrow = row_tiles * div_up(out, 128u), slim = row_tiles * div_up(out, 64u);
    // What a tile costs, in hundreds of cycles: its blocks, as they measured in long calls (at the power limit a tile of half the outputs is no twice as
    // quick), the outputs, and a slice's exchange.
    auto cost = [&](uint32_t tiles, uint32_t at_once, uint32_t blocks, uint32_t block, uint32_t fixed) {
        return div_up(tiles, at_once) * (blocks * block + fixed);
    };
    Fp8GemmPlan p = {256u, 1u, 0u};
    uint32_t best = cost(wide, sms, kbs, 7u, 40u);
    uint32_t c = cost(narrow, sms, kbs, 6u, 30u);
    if (c < best) best = c, p.n = 128u;
    // Few tiles may be cut along K, as long as all clusters are resident at once (one CTA a multiprocessor). What the CTAs of a cluster send each
    // other is 64 KB a CTA from narrow tiles, half as much from slim ones.
    static const uint32_t resident[9] = {0, 148, 74, 45, 33, 26, 22, 15, 15};
    for (uint32_t s = 2; s <= 8u && s <= kbs; s *= 2u) {
        const uint32_t at_once = resident[s] * sms / 148u;
        if (narrow <= at_once && (c = cost(narrow, at_once, div_up(kbs, s), 6u, 110u)) < best) best = c, p.n = 128u, p.split = s;
        if (slim <= at_once && (c = cost(slim, at_once, div_up(kbs, s), 5u, 80u)) < best) best = c, p.n = 64u, p.split = s;
    }
    const uint32_t tiles = p.n == 256u ? wide : p.n == 128u ? narrow : slim;
    p.grid = p.split > 1u ? tiles * p.split : tiles < sms ? tiles : sms;
    return p;
}

cudaError_t launch_fp8_gemm(const CUtensorMap& w, const CUtensorMap& x, const Fp8GemmArgs& a, const Fp8GemmPlan& p, bool overlap, cudaStream_t stream) {
    if (p.n == 256u) return launch_as<256, false>(w, x, a, p.grid, overlap, stream);
    if (p.n == 64u) return launch_as<64, true>(w, x, a, p.grid, overlap, stream);
    if (p.split > 1u) return launch_as<128, true>(w, x, a, p.grid, overlap, stream);
    return launch_as<128, false>(w, x, a, p.grid, overlap, stream);
}

}  // namespace t3
