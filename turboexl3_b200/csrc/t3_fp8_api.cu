// The C entry points of the 8-bit layers and the router (include/t3.h): admission and launch planning. Every refusal comes before
// any launch.
#include <algorithm>
#include <cmath>
#include <initializer_list>

#include "../../include/t3.h"
#include "t3_fp8.h"
#include "t3_internal.h"

namespace t3 {
namespace {

bool act_ok(int dt) { return dt == T3_F32 || dt == T3_F16 || dt == T3_BF16; }
bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0u; }
size_t up256(size_t v) { return (v + 255u) & ~(size_t)255u; }
int status_of(cudaError_t rc) { return rc == cudaSuccess ? T3_OK : T3_CUDA_ERROR; }
uint32_t div_up(uint32_t a, uint32_t b) { return (a + b - 1u) / b; }

// Shared memory a CTA may take: where two fit a multiprocessor (228 KB, 1 KB a CTA reserved), and one
constexpr uint32_t kTwo = 113u * 1024u, kOne = 227u * 1024u;
constexpr uint32_t kHalfMore = 115u * 1024u;  // no second CTA that takes as much fits beside it; one of up to 104 KB does beside kBeside
constexpr uint32_t kBeside = 122u * 1024u;
constexpr uint32_t beside(uint32_t total) { return 228u * 1024u - 2048u - total; }  // what a CTA may take beside one of `total`
constexpr uint32_t kStagesMost = 12;

struct RowsPlan {
    uint32_t cap, split, slice_max, stages, per_sm;
    bool quantise;
    Fp8RowsLayout layout;
};

// resident CTAs of two a multiprocessor by cluster size, and of one (clusters lie inside a group of multiprocessors)
uint32_t resident(uint32_t per_sm, uint32_t split) {
    static const uint32_t two[9] = {0, 296, 296, 279, 284, 280, 270, 259, 264}, one[9] = {0, 148, 148, 135, 132, 130, 132, 105, 120};
    return (per_sm == 2u ? two[split] : one[split]) * multiprocessors() / 148u;
}

// the most slices, of at most `most`, whose CTAs all have a multiprocessor to themselves
uint32_t slices_alone(uint32_t tiles, uint32_t most) {
    uint32_t s = 1;
    for (uint32_t t = 2; t <= kFp8SplitMax && t <= most; ++t)
        if (tiles * t <= resident(1, t)) s = t;
    return s;
}

// Weight tiles in flight: what fits beside the rest. pair: two CTAs a multiprocessor where that leaves each three tiles (a stream of 16 KB tiles, 224
// CTAs: 5.0 TB/s with two in flight, 5.6 with three or more). Else up to `room` bytes, and at least what keeps a second one of its kind from the
// multiprocessor: the hardware doubles up CTAs while other multiprocessors are empty, and the late ones set the launch's duration. two: what a
// CTA of a pair may take.
bool fit(int mode, RowsPlan& p, uint32_t units, uint32_t experts, uint32_t slots, bool pair, uint32_t room = kOne, uint32_t two = kTwo) {
    for (uint32_t per = pair ? 2u : 1u; per >= 1u; --per) {
        for (uint32_t stages = kStagesMost < units ? kStagesMost : units < 2u ? 2u : units; stages >= 2u; --stages) {
            if (per == 2u && stages < 3u && stages < units) break;
            const Fp8RowsLayout l = fp8_rows_layout(mode, p.cap, p.quantise, p.slice_max, p.split, stages, experts, slots);
            if (l.total > (per == 2u ? two : room)) continue;
            p.stages = stages, p.per_sm = per, p.layout = l;
            if (!pair && p.layout.total < kHalfMore) p.layout.total = kHalfMore;
            return true;
        }
    }
    return false;
}

constexpr uint32_t kFusedGroups = 128;  // groups of 128 a CTA quantises itself, of up to 16 rows: past that a launch ahead is quicker

// K slices: what leaves the fullest multiprocessor the fewest 128-blocks, counting a CTA's fixed part as three of them
uint32_t pick_slices(uint32_t tiles, uint32_t kbs) {
    const uint32_t sms = multiprocessors();
    uint32_t best = 1, cost = ~0u;
    for (uint32_t s = 1; s <= kFp8SplitMax && s <= kbs; ++s) {
        const uint32_t c = div_up(tiles * s, sms) * (div_up(kbs, s) + 3u);
        if (c < cost) cost = c, best = s;
    }
    return best;
}

// up to T3_DECODE_ROWS_MAX rows
bool plan_linear(size_t rows, uint32_t in, uint32_t out, bool given, RowsPlan& p) {
    p.cap = rows <= 16u ? 16u : 32u;
    const uint32_t kbs = in / 128u, tiles = div_up(out, 128u);
    p.split = tiles >= multiprocessors() ? 1u : pick_slices(tiles, kbs);
    // Long slices, and rows past 16, have their CTAs a multiprocessor each (16384 -> 7168 at one row 33 -> 24 us, at 29 rows 31 -> 27; 2048 -> 6144
    // at 29 rows 11.1 -> 9.9); else two share one (7168 -> 4096 at 8 rows 11.4 -> 10.5).
    bool pair = true;
    if (tiles <= resident(1, 1)) {
        const uint32_t s = slices_alone(tiles, kbs);
        if (p.cap == 32u || div_up(kbs, s) >= 32u) pair = false, p.split = s;
    }
    p.slice_max = div_up(kbs, p.split);
    p.quantise = !given && p.cap == 16u && (uint32_t)rows * p.slice_max <= kFusedGroups;
    if (fit(kFp8Linear, p, p.slice_max, 0, 0, pair)) return true;
    p.quantise = false;  // (the quantised rows of a slice of a hundred blocks leave no room for weights)
    return fit(kFp8Linear, p, p.slice_max, 0, 0, pair);
}

struct LinearWs {
    size_t scale, total;
};
LinearWs linear_ws(size_t rows, uint32_t in) {
    const size_t q = up256(rows * in);
    return {q, q + up256(rows * (in / 128u) * 4u)};
}

bool linear_shape_ok(size_t rows, int in_dim, int out_dim) {
    if (in_dim <= 0 || out_dim <= 0 || in_dim % 128 != 0 || rows < 1 || rows > kPrefillDenseRowsMax) return false;
    const size_t widest = (size_t)(in_dim > out_dim ? in_dim : out_dim);
    return rows <= 0x7FFFFFFFu / widest;
}

struct MoePlan {
    RowsPlan up, down;
    uint32_t used_max, clusters;  // of gate|up
    size_t h_scale, total;
};

bool plan_moe(size_t rows, int topk, const t3_fp8_bank& b, MoePlan& p) {
    const uint32_t cap = rows <= 16u ? 16u : 32u, slots = (uint32_t)rows * (uint32_t)topk;
    const uint32_t hk = (uint32_t)b.hidden / 128u, ik = (uint32_t)b.inter / 128u;
    p.used_max = (uint32_t)b.experts < slots ? (uint32_t)b.experts : slots;
    p.up.cap = p.down.cap = cap;
    p.up.quantise = true, p.down.quantise = false;
    // gate|up. Few tasks: a CTA a multiprocessor, as many slices as that leaves, and room beside it for down's, which start on their weights while
    // these finish (one row of 512 experts of 2048 x 512: 15.8 -> 13.2 us). Else four slices of at least four blocks, two CTAs a multiprocessor. As many slices in
    // any case as leave the quantised rows' slice room for weights.
    const uint32_t tasks = p.used_max * ik;
    auto too_long = [&](uint32_t t) { return div_up(hk, t) * cap * 128u > 32u * 1024u; };
    uint32_t s = tasks <= resident(1, 1) ? slices_alone(tasks, hk) : 1u;
    const bool pair = tasks > resident(1, 1) || too_long(s);
    if (pair)
        for (s = 1; s < kFp8SplitMax && s * 2u <= hk && ((s < 4u && hk >= 8u * s) || too_long(s));) s *= 2u;
    p.up.split = s, p.up.slice_max = div_up(hk, s);
    if (!fit(kFp8GateUp, p.up, 2u * p.up.slice_max, (uint32_t)b.experts, slots, pair, pair ? kOne : kBeside) &&
        !fit(kFp8GateUp, p.up, 2u * p.up.slice_max, (uint32_t)b.experts, slots, true))
        return false;
    const uint32_t most = resident(p.up.per_sm, s) / s;
    p.clusters = tasks < most ? tasks : most < 1u ? 1u : most;
    // down: one tile a cluster, as many slices as are resident at once
    s = 1;
    for (uint32_t t = 2; t <= kFp8SplitMax; ++t)  // (with room to spare: they are placed among gate|up's last CTAs, and a cluster that is left over is 20 us)
        if (hk * t <= resident(2, t) * 7u / 8u) s = t;
    p.down.split = s, p.down.slice_max = 0;
    // Where gate|up leaves room, what it leaves: weights in flight past it would keep down's CTAs waiting for its own to end (one row, four of 8
    // experts of 4096 x 2048, 32 bytes too many: 26.5 -> 26.3 us).
    const bool room = p.up.per_sm == 1u && p.up.layout.total <= kBeside;
    if (!fit(kFp8Down, p.down, kStagesMost, (uint32_t)b.experts, slots, true, kOne, room ? std::min(kTwo, beside(p.up.layout.total)) : kTwo)) return false;
    const size_t h = up256((size_t)p.used_max * cap * (size_t)b.inter);
    p.h_scale = h;
    p.total = h + up256((size_t)p.used_max * cap * ik * 4u);
    return true;
}

bool bank_shape_ok(const t3_fp8_bank& b) {
    return b.hidden > 0 && b.inter > 0 && b.hidden % 128 == 0 && b.inter % 128 == 0 && b.experts > 0 && b.experts <= T3_FP8_EXPERTS_MAX &&
           (size_t)b.experts * (size_t)(b.hidden > b.inter ? b.hidden : b.inter) <= 0x7FFFFFFFu;
}

}  // namespace
}  // namespace t3

using namespace t3;

extern "C" {

int t3_selftest_fp8_wait_runs_out(void* stream) {
    uint32_t* err = device_error_word();
    if (!err) return T3_CUDA_ERROR;
    count_launches(1);
    return status_of(launch_fp8_wait_runs_out(err, static_cast<cudaStream_t>(stream)));
}

int t3_route(const void* logits, int dtype, size_t rows, int experts, int topk, int scoring, const void* bias, int groups, int group_topk,
             int renormalise, float scale, void* inds, void* scores, void* stream) {
    if (!logits || !inds || !scores) return T3_NULL_POINTER;
    if (!act_ok(dtype)) return T3_BAD_EXL3_DTYPE;
    if (scoring != T3_SCORE_SOFTMAX && scoring != T3_SCORE_SIGMOID) return T3_ENGINE_NOT_IMPLEMENTED;
    if (rows < 1 || rows > 0x7FFFFFFFu || experts < 1 || experts > T3_ROUTE_EXPERTS_MAX || topk < 1 || topk > T3_REDUCE_MAX_TOPK ||
        groups < 1 || groups > 32 || experts % groups != 0 || group_topk < 1 || group_topk > groups ||
        topk > experts / groups * group_topk || !std::isfinite(scale))
        return T3_BAD_EXL3_SHAPE;
    RouteArgs a = {};
    a.logits = logits, a.dt = dtype, a.scoring = scoring, a.bias = static_cast<const float*>(bias), a.rows = rows;
    a.experts = (uint32_t)experts, a.topk = (uint32_t)topk, a.groups = (uint32_t)groups, a.group_topk = (uint32_t)group_topk;
    a.renormalise = renormalise != 0, a.scale = scale, a.inds = static_cast<int32_t*>(inds), a.scores = static_cast<float*>(scores);
    count_launches(1);
    return status_of(launch_route(a, launches_overlap(), static_cast<cudaStream_t>(stream)));
}

int t3_quantize_fp8(const void* x, int x_dtype, size_t rows, int in_dim, void* q, void* scale, void* stream) {
    if (!x || !q || !scale) return T3_NULL_POINTER;
    if (!act_ok(x_dtype)) return T3_BAD_EXL3_DTYPE;
    if (in_dim <= 0 || in_dim % 128 != 0 || rows < 1 || rows > (size_t)1 << 40 || !on16(x) || !on16(q)) return T3_BAD_EXL3_SHAPE;
    count_launches(1);
    return status_of(launch_fp8_quantize(x, x_dtype, rows, (uint32_t)in_dim, static_cast<uint8_t*>(q), static_cast<float*>(scale),
                                         launches_overlap(), static_cast<cudaStream_t>(stream)));
}

size_t t3_linear_fp8_workspace_bytes(size_t rows, int in_dim, int out_dim, int x_dtype) {
    if (!act_ok(x_dtype) || !linear_shape_ok(rows, in_dim, out_dim)) return 0;
    RowsPlan p;
    if (rows <= T3_DECODE_ROWS_MAX && plan_linear(rows, (uint32_t)in_dim, (uint32_t)out_dim, false, p) && p.quantise) return 0;
    return linear_ws(rows, (uint32_t)in_dim).total;
}

int t3_linear_fp8(const void* x, int x_dtype, const void* x_scale, size_t rows, const void* w, const void* w_scale, int in_dim, int out_dim,
                  void* y, int y_dtype, void* workspace, size_t workspace_bytes, void* stream_v) {
    const bool given = x_dtype == T3_E4M3, few = rows <= T3_DECODE_ROWS_MAX;
    if (!x || !w || !w_scale || !y || (given && !x_scale)) return T3_NULL_POINTER;
    if ((!given && !act_ok(x_dtype)) || !act_ok(y_dtype)) return T3_BAD_EXL3_DTYPE;
    if (!linear_shape_ok(rows, in_dim, out_dim) || (!given && x_scale) || !on16(x) || !on16(w) || !on16(y)) return T3_BAD_EXL3_SHAPE;
    if (!few && !prefill_served()) return T3_ENGINE_NOT_IMPLEMENTED;
    const uint32_t in = (uint32_t)in_dim, out = (uint32_t)out_dim;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
    RowsPlan p = {};
    Fp8GemmPlan g = {};
    if (!few) g = plan_fp8_gemm((uint32_t)rows, in, out);
    else if (!plan_linear(rows, in, out, given, p)) return T3_ENGINE_NOT_IMPLEMENTED;
    const bool ahead = !given && !p.quantise;  // a launch quantises the rows ahead of the product
    const LinearWs ws = linear_ws(rows, in);
    if (ahead) {
        if (!workspace) return T3_NULL_POINTER;
        if (workspace_bytes < ws.total || (reinterpret_cast<uintptr_t>(workspace) & 255u)) return T3_WORKSPACE_TOO_SMALL;
    }
    float* scale = given ? static_cast<float*>(const_cast<void*>(x_scale)) : reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + ws.scale);
    Fp8Maps maps = {};
    if (!make_byte_map(&maps.w[0], w, out, in, few ? 128u : g.n)) return T3_KERNEL_CREATE_FAILED;
    if (!p.quantise && !make_byte_map(&maps.rows, given ? x : workspace, rows, in, few ? p.cap : 128u)) return T3_KERNEL_CREATE_FAILED;
    const bool overlap = launches_overlap();
    if (ahead) {
        count_launches(1);
        if (cudaError_t rc = launch_fp8_quantize(x, x_dtype, rows, in, static_cast<uint8_t*>(workspace), scale, overlap, stream)) return status_of(rc);
    }
    count_launches(1);
    if (!few) {
        Fp8GemmArgs a = {};
        a.x_scale = scale, a.w_scale = static_cast<const float*>(w_scale), a.y = y, a.y_dt = y_dtype;
        a.rows = (uint32_t)rows, a.in = in, a.out = out, a.split = g.split, a.early = ahead, a.err = device_error_word();
        return status_of(launch_fp8_gemm(maps.w[0], maps.rows, a, g, overlap, stream));
    }
    Fp8RowsArgs a = {};
    if (p.quantise) a.x = x, a.x_dt = x_dtype;
    else a.x_scale = scale;
    a.rows = (uint32_t)rows, a.in = in, a.out = out, a.w_scale[0] = static_cast<const float*>(w_scale);
    a.y = y, a.y_dt = y_dtype, a.split = p.split, a.stages = p.stages, a.early = ahead, a.err = device_error_word();
    a.l = p.layout;
    return status_of(launch_fp8_rows(kFp8Linear, p.cap, maps, a, div_up(out, 128u), overlap, stream));
}

size_t t3_moe_fp8_workspace_bytes(size_t rows, int topk, const t3_fp8_bank* bank) {
    MoePlan p;
    if (!bank || !bank_shape_ok(*bank) || rows < 1 || rows > T3_DECODE_ROWS_MAX || topk < 1 || topk > T3_REDUCE_MAX_TOPK || !plan_moe(rows, topk, *bank, p))
        return 0;
    return p.total;
}

int t3_moe_fp8(const void* x, int x_dtype, size_t rows, const t3_fp8_bank* bank, const void* inds, const void* scores, int scores_dtype,
               int topk, const void* shared, void* y, void* workspace, size_t workspace_bytes, void* stream) {
    if (!x || !bank || !inds || !scores || !y || !workspace) return T3_NULL_POINTER;
    for (const t3_fp8_proj* p : {&bank->gate, &bank->up, &bank->down})
        if (!p->w || !p->scale) return T3_NULL_POINTER;
    if (!act_ok(x_dtype) || !act_ok(scores_dtype)) return T3_BAD_EXL3_DTYPE;
    if (!bank_shape_ok(*bank) || rows < 1 || topk < 1 || topk > T3_REDUCE_MAX_TOPK || !on16(x) || !on16(bank->gate.w) || !on16(bank->up.w) ||
        !on16(bank->down.w) ||
        !on16(y) || !on16(shared))
        return T3_BAD_EXL3_SHAPE;
    MoePlan p;
    if (rows > T3_DECODE_ROWS_MAX || !plan_moe(rows, topk, *bank, p)) return T3_ENGINE_NOT_IMPLEMENTED;
    if (workspace_bytes < p.total || (reinterpret_cast<uintptr_t>(workspace) & 255u)) return T3_WORKSPACE_TOO_SMALL;
    const uint32_t cap = p.up.cap, hidden = (uint32_t)bank->hidden, inter = (uint32_t)bank->inter, experts = (uint32_t)bank->experts;
    Fp8Maps up = {}, down = {};
    if (!make_byte_map(&up.w[0], bank->gate.w, (uint64_t)experts * inter, hidden, 128u) ||
        !make_byte_map(&up.w[1], bank->up.w, (uint64_t)experts * inter, hidden, 128u) ||
        !make_byte_map(&down.w[0], bank->down.w, (uint64_t)experts * hidden, inter, 128u) ||
        !make_byte_map(&down.rows, workspace, (uint64_t)p.used_max * cap, inter, cap))
        return T3_KERNEL_CREATE_FAILED;
    Fp8RowsArgs a = {};
    a.x = x, a.x_dt = x_dtype, a.rows = (uint32_t)rows, a.in = hidden, a.out = inter;
    a.w_scale[0] = static_cast<const float*>(bank->gate.scale), a.w_scale[1] = static_cast<const float*>(bank->up.scale);
    a.split = p.up.split, a.stages = p.up.stages, a.l = p.up.layout;
    a.inds = static_cast<const uint32_t*>(inds), a.scores = scores, a.score_dt = scores_dtype, a.topk = (uint32_t)topk, a.experts = experts;
    a.h = static_cast<uint8_t*>(workspace), a.h_scale = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + p.h_scale);
    a.err = device_error_word();
    const bool overlap = launches_overlap();
    count_launches(1);
    if (cudaError_t rc = launch_fp8_rows(kFp8GateUp, cap, up, a, p.clusters, overlap, static_cast<cudaStream_t>(stream)))
        return status_of(rc);
    Fp8RowsArgs d = a;
    d.x = nullptr, d.x_scale = a.h_scale, d.in = inter, d.out = hidden;
    d.w_scale[0] = static_cast<const float*>(bank->down.scale), d.w_scale[1] = nullptr;
    d.split = p.down.split, d.stages = p.down.stages, d.l = p.down.layout;
    d.shared = shared, d.y = y, d.y_dt = x_dtype;
    count_launches(1);
    return status_of(launch_fp8_rows(kFp8Down, cap, down, d, hidden / 128u, overlap, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
