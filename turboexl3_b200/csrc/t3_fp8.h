// The 8-bit operators (e4m3 values, one scale for each block of 128): arguments and launches shared by their kernels
// (t3_fp8_rows.cu, t3_fp8_gemm.cu, t3_fp8_quant.cu, t3_route.cu) and the entry points (t3_fp8_api.cu).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace t3 {

constexpr uint32_t kFp8ExpertsMax = 2048; // of a bank: a CTA keeps a word for each
constexpr uint32_t kFp8SplitMax = 8;      // K slices of a tile: the portable cluster size

// What a launch of the streaming kernel does (t3_fp8_rows.cu)
enum Fp8Mode : int { kFp8Linear = 0, kFp8GateUp = 1, kFp8Down = 2 };

// Shared memory of a streaming CTA: offsets from a 1024-byte boundary
struct Fp8RowsLayout {
    uint32_t rows, part, hid, red, sx, fetch, c, mask, list, chunks, slots, weight, bars, total;  // (the ring of weights at 0)
};

struct Fp8RowsArgs {
    Fp8RowsLayout l;
    const void* x;         // [rows, in] in x_dt, quantised by the CTAs; or null: the rows are e4m3 already (the launch's row map)
    int x_dt;
    const float* x_scale;  // without x: [rows, in / 128] (down: the hidden rows', [experts used * cap, in / 128])
    uint32_t rows, in, out;  // a linear's; gate|up: in = hidden, out = inter; down: in = inter, out = hidden
    const float* w_scale[2];  // [out / 128 up, in / 128], of a bank [experts, out / 128, in / 128]; gate|up: the gate's and the up's
    void* y;               // [rows, out] in y_dt
    int y_dt;
    uint32_t split;        // K slices, CTAs of a cluster
    uint32_t stages;       // 128 x 128 weight tiles in flight a CTA
    uint32_t early;        // linear without x: the rows are the output of this call's launch before this one, which has waited for the weights
    // routed
    const uint32_t* inds;  // [rows, topk]
    const void* scores;
    int score_dt;
    uint32_t topk, experts;
    uint8_t* h;            // silu(gate) * up in e4m3, [experts used][cap][inter], and its scales [experts used][cap][inter / 128]
    float* h_scale;
    const void* shared;    // [rows, out] in y_dt added before the one rounding, or null
    uint32_t* err;
};

struct Fp8Maps {
    CUtensorMap w[2];  // e4m3 [rows, in], boxes of 128 values x 128 rows
    CUtensorMap rows;  // the e4m3 rows (without x): boxes of 128 values x the tile's columns
};

// `cap`: columns of a tile (rows of the call it serves): 16 or 32
Fp8RowsLayout fp8_rows_layout(int mode, uint32_t cap, bool quantise, uint32_t slice_max, uint32_t split, uint32_t stages, uint32_t experts,
                              uint32_t slots);
cudaError_t launch_fp8_rows(int mode, uint32_t cap, const Fp8Maps& maps, const Fp8RowsArgs& a, uint32_t clusters, bool overlap,
                            cudaStream_t stream);

// The linear past 32 rows (t3_fp8_gemm.cu)
struct Fp8GemmArgs {
    const float *x_scale, *w_scale;  // [rows, in / 128], [out / 128 up, in / 128]
    void* y;                         // [rows, out] in y_dt
    int y_dt;
    uint32_t rows, in, out;
    uint32_t split;                  // K slices, CTAs of a cluster
    uint32_t early;                  // as Fp8RowsArgs::early
    uint32_t* err;
};
struct Fp8GemmPlan {
    uint32_t n, split, grid;  // outputs of a tile (its map's box is that many rows of the weight), K slices, CTAs
};
Fp8GemmPlan plan_fp8_gemm(uint32_t rows, uint32_t in, uint32_t out);
cudaError_t launch_fp8_gemm(const CUtensorMap& w, const CUtensorMap& x, const Fp8GemmArgs& a, const Fp8GemmPlan& p, bool overlap, cudaStream_t stream);

// x [rows, in] -> e4m3 values and scales [rows, in / 128]
cudaError_t launch_fp8_quantize(const void* x, int dt, size_t rows, uint32_t in, uint8_t* q, float* scale, bool overlap, cudaStream_t stream);

// one warp whose waits nothing ends (test hook)
cudaError_t launch_fp8_wait_runs_out(uint32_t* err, cudaStream_t stream);

struct RouteArgs {
    const void* logits;  // [rows, experts]
    int dt, scoring;
    const float* bias;   // [experts] or null
    size_t rows;
    uint32_t experts, topk, groups, group_topk;
    int renormalise;
    float scale;
    int32_t* inds;       // [rows, topk]
    float* scores;
};
cudaError_t launch_route(const RouteArgs& a, bool overlap, cudaStream_t stream);

}  // namespace t3
