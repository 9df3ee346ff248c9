// Activations to e4m3 with one power-of-two scale for each 128 values of a row (see fp8_scale).
//
// Bound by memory: 2 bytes read and 1 written a value of a 16-bit row. Sixteen lanes hold a group, eight values each (one 16-byte load,
// two of f32), so the largest magnitude takes four shuffles; the magnitudes are compared as bit patterns, where an infinity and a
// NaN are larger than every number and nothing is lost to a comparison with a NaN. 8192 rows of 7168 bf16: 31.2 us, 5.7 TB/s (42.8 with the magnitudes
// compared as f32 one by one).
#include "t3_fp8.cuh"
#include "t3_fp8.h"
#include "t3_internal.h"

namespace t3 {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kUnder = 4;  // groups a half warp has under way

template <int DT>
__global__ void __launch_bounds__(kThreads) fp8_quantize(const void* x, size_t groups, uint8_t* q, float* scale) {
    constexpr uint32_t kWords = DT == kF32 ? 8u : 4u;
    pdl_wait();
    pdl_trigger();
    const uint32_t lane = threadIdx.x & 15u, half = 0xFFFFu << (threadIdx.x & 16u);
    const size_t step = (size_t)gridDim.x * (kThreads / 16u);
    for (size_t g0 = (size_t)blockIdx.x * (kThreads / 16u) + threadIdx.x / 16u; g0 < groups; g0 += step * kUnder) {
        uint32_t w[kUnder][kWords];
#pragma unroll
        for (uint32_t j = 0; j < kUnder; ++j) {
            const size_t g = g0 + j * step;
            if (g >= groups) break;
            const uint4* from = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(x) + (g * 128u + lane * 8u) * (DT == kF32 ? 4u : 2u));
#pragma unroll
            for (uint32_t k = 0; k < kWords / 4u; ++k) {
                const uint4 u = __ldcs(from + k);
                w[j][4u * k] = u.x, w[j][4u * k + 1u] = u.y, w[j][4u * k + 2u] = u.z, w[j][4u * k + 3u] = u.w;
            }
        }
#pragma unroll
        for (uint32_t j = 0; j < kUnder; ++j) {
            const size_t g = g0 + j * step;
            if (g >= groups) break;  // (a half warp's lanes leave together)
            // 16-bit magnitudes order as their bit patterns too, two to a word
            uint32_t most = 0;
#pragma unroll
            for (uint32_t k = 0; k < kWords; ++k)
                most = DT == kF32 ? max(most, w[j][k] & 0x7FFFFFFFu) : __vmaxu2(most, w[j][k] & 0x7FFF7FFFu);
#pragma unroll
            for (uint32_t d = 8; d; d >>= 1) {
                const uint32_t other = __shfl_xor_sync(half, most, d);
                most = DT == kF32 ? max(most, other) : __vmaxu2(most, other);
            }
            if (DT == kBf16) most = max(most << 16, most & 0xFFFF0000u);
            if (DT == kF16) most = __float_as_uint(__half2float(__ushort_as_half((unsigned short)max(most & 0xFFFFu, most >> 16))));
            const float s = fp8_scale(most);
            float v[2][4];
#pragma unroll
            for (uint32_t k = 0; k < 4u; ++k) {
                float2 f;
                if (DT == kF32) f = make_float2(__uint_as_float(w[j][2u * k % kWords]), __uint_as_float(w[j][(2u * k + 1u) % kWords]));
                else if (DT == kF16) f = unpack_half2(w[j][k]);
                else f = make_float2(__uint_as_float(w[j][k] << 16), __uint_as_float(w[j][k] & 0xFFFF0000u));
                v[k >> 1][2u * (k & 1u)] = f.x, v[k >> 1][2u * (k & 1u) + 1u] = f.y;
            }
            *reinterpret_cast<uint2*>(q + g * 128u + lane * 8u) = make_uint2(to_e4m3x4(v[0], s), to_e4m3x4(v[1], s));
            if (lane == 0) scale[g] = s;
        }
    }
}

// A warp waits twice for phases that nothing completes, as the kernels' roles do behind what they have issued: the first wait runs out and says so, the
// second finds `dead` and takes no time.
__global__ void fp8_wait_runs_out(uint32_t* err) {
    __shared__ uint64_t bar[2];
    __shared__ uint32_t dead;
    if (threadIdx.x == 0) {
        mbar_init(&bar[0], 1u), mbar_init(&bar[1], 1u);
        mbar_init_fence();
        dead = 0u;
    }
    __syncthreads();
    fp8_wait(smem_addr(&bar[0]), 0u, &dead, err, kErrMmaWait);
    fp8_wait(smem_addr(&bar[1]), 0u, &dead, err, kErrFullWait);
}

}  // namespace

cudaError_t launch_fp8_wait_runs_out(uint32_t* err, cudaStream_t stream) {
    fp8_wait_runs_out<<<1, 32, 0, stream>>>(err);
    return cudaGetLastError();
}

cudaError_t launch_fp8_quantize(const void* x, int dt, size_t rows, uint32_t in, uint8_t* q, float* scale, bool overlap, cudaStream_t stream) {
    const size_t groups = rows * (in / 128u), per = kThreads / 16u;
    size_t blocks = (groups + per - 1u) / per;
    const size_t most = (size_t)multiprocessors() * 16u;
    if (blocks > most) blocks = most;
    const dim3 grid((unsigned)blocks);
    if (dt == kF32) return launch_overlapped(fp8_quantize<kF32>, grid, kThreads, 0, stream, overlap, 1, x, groups, q, scale);
    if (dt == kF16) return launch_overlapped(fp8_quantize<kF16>, grid, kThreads, 0, stream, overlap, 1, x, groups, q, scale);
    return launch_overlapped(fp8_quantize<kBf16>, grid, kThreads, 0, stream, overlap, 1, x, groups, q, scale);
}

}  // namespace t3
