// Activations to e4m3 with one power-of-two scale for each 128 values of a row (see fp8_scale).
//
// Bound by memory: 2 bytes read and 1 written a value of a 16-bit row. Sixteen lanes hold a group, eight values each (one 16-byte load,
// two of f32), so the largest magnitude takes four shuffles; the magnitudes are compared as bit patterns, where an infinity and a
// NaN are larger than every number and nothing is lost to a comparison with a NaN.
#include "t3_fp8.cuh"
#include "t3_fp8.h"
#include "t3_internal.h"

namespace t3 {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kUnder = 4;  // groups a half warp has under way

template <int DT>
__global__ void __launch_bounds__(kThreads) fp8_quantize(const void* __restrict__ x, size_t groups, uint8_t* __restrict__ q, float* __restrict__ scale) {
    pdl_trigger();
    pdl_wait();
    const uint32_t lane = threadIdx.x & 15u;
    const size_t step = (size_t)gridDim.x * (kThreads / 16u);
    for (size_t g0 = (size_t)blockIdx.x * (kThreads / 16u) + threadIdx.x / 16u; g0 < groups; g0 += step * kUnder) {
        float v[kUnder][8];
#pragma unroll
        for (uint32_t j = 0; j < kUnder; ++j) {
            const size_t g = g0 + j * step;
            if (g >= groups) break;
            const size_t at = g * 128u + lane * 8u;
            if (DT == kF32) {
                load_act4(x, DT, at, reinterpret_cast<float(&)[4]>(v[j][0]));
                load_act4(x, DT, at + 4u, reinterpret_cast<float(&)[4]>(v[j][4]));
            } else {
                const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(x) + at);
                const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if (DT == kF16) {
                        const float2 f = unpack_half2(w[k]);
                        v[j][2 * k] = f.x, v[j][2 * k + 1] = f.y;
                    } else {
                        v[j][2 * k] = __uint_as_float(w[k] << 16), v[j][2 * k + 1] = __uint_as_float(w[k] & 0xFFFF0000u);
                    }
                }
            }
        }
#pragma unroll
        for (uint32_t j = 0; j < kUnder; ++j) {
            const size_t g = g0 + j * step;
            if (g >= groups) break;  // (a half warp's lanes leave together)
            uint32_t most = 0;
#pragma unroll
            for (int k = 0; k < 8; ++k) most = max(most, magnitude(v[j][k]));
            const uint32_t half = 0xFFFFu << (threadIdx.x & 16u);
#pragma unroll
            for (uint32_t d = 8; d; d >>= 1) most = max(most, __shfl_xor_sync(half, most, d));
            const float s = fp8_scale(most);
            *reinterpret_cast<uint2*>(q + g * 128u + lane * 8u) = make_uint2(to_e4m3x4(reinterpret_cast<const float(&)[4]>(v[j][0]), s),
                                                                             to_e4m3x4(reinterpret_cast<const float(&)[4]>(v[j][4]), s));
            if (lane == 0) scale[g] = s;
        }
    }
}

}  // namespace

cudaError_t launch_fp8_quantize(const void* x, int dt, size_t rows, uint32_t in, uint8_t* q, float* scale, bool overlap, cudaStream_t stream) {
    const size_t groups = rows * (in / 128u), per = kThreads / 16u;
    size_t blocks = (groups + per - 1u) / per;
    const size_t most = 148u * 8u;  // eight of 256 threads fill a multiprocessor
    if (blocks > most) blocks = most;
    const dim3 grid((unsigned)blocks);
    if (dt == kF32) return launch_overlapped(fp8_quantize<kF32>, grid, kThreads, 0, stream, overlap, 1, x, groups, q, scale);
    if (dt == kF16) return launch_overlapped(fp8_quantize<kF16>, grid, kThreads, 0, stream, overlap, 1, x, groups, q, scale);
    return launch_overlapped(fp8_quantize<kBf16>, grid, kThreads, 0, stream, overlap, 1, x, groups, q, scale);
}

}  // namespace t3
